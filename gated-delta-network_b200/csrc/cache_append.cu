// cache_append.cu -- new key/value rows into a paged cache of 8-bit codes with a scale for each page and head.
//
// For every (page, head) that the call writes to, with m = 127 (int8) or 448 (e4m3):
//   s' = max(s, max |x| / m)     s: the page's scale, or 0 if its first token is among the new ones
//   code = round(x / s') for the new tokens, round(code s / s') for older ones where s' > s
// Quotients are IEEE fp32 and ties go to even, so the codes do not depend on the order of the work.
// max |x| is over finite values; infinities become the largest code, a NaN the code NaN (e4m3) or 0 (int8).
//
// One CTA per (page a sequence touches, head, key or value): its rows stay in registers between the maximum and
// the encoding, so each row is read once and written once.
#include <cuda_fp16.h>

#include "linear.cuh"
#include "prefill_kernels.cuh"

namespace gdn {

// The sequence whose touched pages hold slot u: the last one with cu[b] / P + 2 b <= u.  n tokens touch at most
// floor(n / P) + 2 pages, so these bases need no prefix sum.  32 probes a round, all lanes of every warp together.
__device__ __forceinline__ int find_sequence(const CacheAppendArgs& p, int u) {
    int lo = 0, n = p.c.B;  // candidates lo .. lo + n - 1; lo always qualifies
    const int lane = threadIdx.x & 31;
    while (n > 1) {
        const int step = (n + 31) / 32, at = lo + lane * step;
        bool yes = false;
        if (lane * step < n) {
            int s, e;
            seq_bounds(p.cu, p.cu64, at, p.T, s, e);
            yes = (s >> p.c.page_shift) + 2 * at <= u;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, yes);
        const int last = hit ? 31 - __clz(hit) : 0;
        n = min(step, n - last * step);
        lo += last * step;
    }
    return lo;
}

__device__ __forceinline__ float finite_abs(uint32_t bits) {  // bf16 bits in the high half
    const uint32_t a = bits & 0x7fff0000u;
    return a < 0x7f800000u ? __uint_as_float(a) : 0.f;
}

template <bool kInt8>
__device__ __forceinline__ uint32_t encode4(const float (&x)[4]) {
    uint32_t w = 0;
    if (kInt8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w |= (uint32_t)(max(-127, min(127, __float2int_rn(x[i]))) & 0xff) << (8 * i);
    } else {
        uint16_t a, b;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(a) : "f"(x[1]), "f"(x[0]));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(b) : "f"(x[3]), "f"(x[2]));
        w = (uint32_t)a | ((uint32_t)b << 16);
    }
    return w;
}
template <bool kInt8>
__device__ __forceinline__ void decode4(uint32_t w, float (&x)[4]) {
    if (kInt8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(w >> (8 * i));
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint32_t h;
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)(w >> (16 * i))));
            const __half2 y = *reinterpret_cast<__half2*>(&h);
            x[2 * i] = __low2float(y);
            x[2 * i + 1] = __high2float(y);
        }
    }
}

// R: passes of 8 rows that cover a page.
template <bool kInt8, int R>
__global__ void __launch_bounds__(128) gdn_cache_append_kernel(CacheAppendArgs p) {
    __shared__ float s_max[4];
    pdl_wait();
    pdl_trigger();
    const CacheArgs& c = p.c;
    const int tid = threadIdx.x, head = blockIdx.y;
    const int b = find_sequence(p, blockIdx.x);
    int t0, t1;
    seq_bounds(p.cu, p.cu64, b, p.T, t0, t1);
    // positions of the new tokens; those outside [0, max_pages P) are dropped
    const int end = cache_length(c, b), start = end - (t1 - t0);
    const int i = (int)blockIdx.x - ((t0 >> c.page_shift) + 2 * b) + (max(start, 0) >> c.page_shift);  // page of the sequence
    if (i < 0 || i >= c.max_pages) return;
    const int lo = max(max(start, 0), i << c.page_shift), hi = min(end, (i + 1) << c.page_shift);
    if (lo >= hi) return;
    const int page = c.table[(size_t)b * c.max_pages + i];
    if ((unsigned)page >= (unsigned)c.pages) return;  // no such page: the rows are dropped
    const uint16_t* x = (blockIdx.z ? p.v : p.k) + ((size_t)(t0 + lo - start) * c.Hkv + head) * kD + 8 * (tid & 15);
    uint8_t* codes = static_cast<uint8_t*>(blockIdx.z ? c.v_cache : c.k_cache) + ((((size_t)page * c.Hkv + head) << c.page_shift)) * kD;
    float* scale = (blockIdx.z ? c.v_scale : c.k_scale) + (size_t)page * c.Hkv + head;

    const int rows = hi - lo, row = tid >> 4, held = lo - (i << c.page_shift);
    const float old = held > 0 ? *scale : 0.f;
    uint4 w[R];
    float top = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        w[r] = make_uint4(0, 0, 0, 0);
        if (8 * r + row < rows) w[r] = __ldg(reinterpret_cast<const uint4*>(x + (size_t)(8 * r + row) * c.Hkv * kD));
        const uint32_t u[4] = {w[r].x, w[r].y, w[r].z, w[r].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, fmaxf(finite_abs(u[e] << 16), finite_abs(u[e] & 0xffff0000u)));
    }
#pragma unroll
    for (int off = 16; off; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    if ((tid & 31) == 0) s_max[tid >> 5] = top;
    __syncthreads();
    top = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
    const float s = fmaxf(old, __fdiv_rn(top, kInt8 ? 127.f : 448.f));

    if (held > 0 && s > old) {  // older tokens of the page to the new scale, 16 bytes a thread
        for (int j = tid; j < held * 8; j += 128) {
            uint4* at = reinterpret_cast<uint4*>(codes) + j;
            const uint4 y = *at;
            uint32_t u[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float f[4];
                decode4<kInt8>(u[e], f);
#pragma unroll
                for (int d = 0; d < 4; ++d) f[d] = __fdiv_rn(__fmul_rn(f[d], old), s);
                u[e] = encode4<kInt8>(f);
            }
            *at = make_uint4(u[0], u[1], u[2], u[3]);
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (8 * r + row < rows) {
            const uint32_t u[4] = {w[r].x, w[r].y, w[r].z, w[r].w};
            uint32_t o[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float f[4] = {__uint_as_float(u[2 * e] << 16), __uint_as_float(u[2 * e] & 0xffff0000u),
                              __uint_as_float(u[2 * e + 1] << 16), __uint_as_float(u[2 * e + 1] & 0xffff0000u)};
#pragma unroll
                for (int d = 0; d < 4; ++d) f[d] = s > 0.f ? __fdiv_rn(f[d], s) : 0.f;
                o[e] = encode4<kInt8>(f);
            }
            *reinterpret_cast<uint2*>(codes + (size_t)(held + 8 * r + row) * kD + 8 * (tid & 15)) = make_uint2(o[0], o[1]);
        }
    }
    if (tid == 0) *scale = s;
}

template <bool kInt8>
static cudaError_t launch_rows(const CacheAppendArgs& p, dim3 grid, cudaStream_t stream) {
    switch (p.c.page_shift) {
        case 4: return launch_pdl(gdn_cache_append_kernel<kInt8, 2>, grid, dim3(128), 0, stream, p);
        case 5: return launch_pdl(gdn_cache_append_kernel<kInt8, 4>, grid, dim3(128), 0, stream, p);
        case 6: return launch_pdl(gdn_cache_append_kernel<kInt8, 8>, grid, dim3(128), 0, stream, p);
        default: return launch_pdl(gdn_cache_append_kernel<kInt8, 16>, grid, dim3(128), 0, stream, p);
    }
}

int launch_cache_append(const CacheAppendArgs& p, cudaStream_t stream) {
    const dim3 grid((unsigned)((p.T >> p.c.page_shift) + 2 * p.c.B), (unsigned)p.c.Hkv, 2);
    return (p.c.int8 ? launch_rows<true>(p, grid, stream) : launch_rows<false>(p, grid, stream)) == cudaSuccess ? 0 : -1;
}

}  // namespace gdn
