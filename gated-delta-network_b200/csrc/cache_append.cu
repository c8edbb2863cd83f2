// cache_append.cu -- new key/value rows into a paged cache of 8-bit codes with a scale for each page and head.
//
// For every (page, head) that the call writes to, with m = 127 (int8) or 448 (e4m3):
//   s' = max(s, max |x| / m)     s: the page's scale, or 0 if its first token is among the new ones
//   code = round(x / s') for the new tokens, round(code s / s') for older ones where s' > s
// Quotients are IEEE fp32 and ties go to even, so the codes do not depend on the order of the work.
// max |x| is over finite values; infinities become the largest code, a NaN the code NaN (e4m3) or 0 (int8).
//
// Bound by HBM for prompts (768 bytes a token and head, each row read and written once) and by latency for decode steps.
// Prompts: one CTA per (page a sequence touches, head, key or value), its rows in registers between the maximum and the
// encoding.  Steps of a few tokens: one warp each instead, eight of them a CTA, so that the search for the sequence and
// the loads it leads to are in flight together.
// The quotients would cost more than the traffic: a code is taken from x (1 / s), and from the quotient where the two
// could round to different codes.
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

// Largest magnitude of 8 bf16 values so far, per half; NaN does not count, infinity is dealt with by finite_max.
__device__ __forceinline__ __nv_bfloat162 abs_max(__nv_bfloat162 top, uint4 w) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) top = __hmax2(top, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&u[e])));
    return top;
}
__device__ __forceinline__ float finite_max(uint4 w) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t a = (e & 1 ? u[e >> 1] & 0x7fff0000u : (u[e >> 1] << 16) & 0x7fffffffu);
        if (a < 0x7f800000u) top = fmaxf(top, __uint_as_float(a));
    }
    return top;
}

// Four codes of quotients, to nearest even.  int8: of finite ones up to 127 (kAny: of any); e4m3 saturates.
__device__ __forceinline__ float clamp127(float x) { return x == x ? fminf(fmaxf(x, -127.f), 127.f) : 0.f; }
template <bool kInt8, bool kAny>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    if (kInt8) {
        const float big = 12582912.f;  // + 1.5 2^23 leaves the rounded integer in the low bits
        if (kAny) a = clamp127(a), b = clamp127(b), c = clamp127(c), d = clamp127(d);
        const uint32_t x = __float_as_uint(__fadd_rn(a, big)), y = __float_as_uint(__fadd_rn(b, big));
        const uint32_t z = __float_as_uint(__fadd_rn(c, big)), w = __float_as_uint(__fadd_rn(d, big));
        return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
    }
    uint16_t x, y;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(x) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(y) : "f"(d), "f"(c));
    return (uint32_t)x | ((uint32_t)y << 16);
}
// Eight bf16 values to codes of scale s; r = 1 / s rounded, or 0 to have every code from its quotient.
template <bool kInt8>
__device__ __forceinline__ uint2 encode8(uint4 w, float s, float r) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    bool odd = r == 0.f;  // every code from its quotient
    if (kInt8) {          // infinity or NaN among them
        __nv_bfloat162 top = __habs2(*reinterpret_cast<const __nv_bfloat162*>(&u[0]));
#pragma unroll
        for (int e = 1; e < 4; ++e) top = __hmax2_nan(top, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&u[e])));
        const uint32_t bits = *reinterpret_cast<const uint32_t*>(&top);
        odd |= (bits & 0x7f80u) == 0x7f80u || (bits & 0x7f800000u) == 0x7f800000u;
    }
    uint32_t o[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const float2 x = make_float2(__uint_as_float(u[2 * e] << 16), __uint_as_float(u[2 * e] & 0xffff0000u));
        const float2 y = make_float2(__uint_as_float(u[2 * e + 1] << 16), __uint_as_float(u[2 * e + 1] & 0xffff0000u));
        bool differ;
        if (kInt8) {
            // x (1 / s) is within 127 2^-22 < 2^-15 of x / s: another code only where it is that near to a half
            const float2 r2 = make_float2(r, r), big = make_float2(12582912.f, 12582912.f);  // + 1.5 2^23: the rounded integer in the low bits
            const float2 qx = mul2(x, r2), qy = mul2(y, r2), nx = add2(qx, big), ny = add2(qy, big);
            const float2 dx = sub2(qx, sub2(nx, big)), dy = sub2(qy, sub2(ny, big));
            differ = fmaxf(fmaxf(fabsf(dx.x), fabsf(dx.y)), fmaxf(fabsf(dy.x), fabsf(dy.y))) > 0.5f - 0x1p-14f;
            o[e] = __byte_perm(__byte_perm(__float_as_uint(nx.x), __float_as_uint(nx.y), 0x0040),
                               __byte_perm(__float_as_uint(ny.x), __float_as_uint(ny.y), 0x0040), 0x5410);
        } else {
            // x (1 / s) is within 2^-22 of x / s, whose code lies between those of r (1 -+ 2^-21)
            const float2 lo = make_float2(r * (1.f - 0x1p-21f), r * (1.f - 0x1p-21f)), hi = make_float2(r * (1.f + 0x1p-21f), r * (1.f + 0x1p-21f));
            const float2 a = mul2(x, lo), b = mul2(y, lo), c = mul2(x, hi), d = mul2(y, hi);
            o[e] = encode4<false, false>(a.x, a.y, b.x, b.y);
            differ = o[e] != encode4<false, false>(c.x, c.y, d.x, d.y);
        }
        if (differ || odd)  // (s = 0: zeros, or values whose scale is below fp32)
            o[e] = s > 0.f ? encode4<kInt8, true>(__fdiv_rn(x.x, s), __fdiv_rn(x.y, s), __fdiv_rn(y.x, s), __fdiv_rn(y.y, s)) : 0u;
    }
    return make_uint2(o[0], o[1]);
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
// 16 codes of scale `old` to scale s.
template <bool kInt8>
__device__ __forceinline__ void recode16(uint4* at, float old, float s) {
    const uint4 y = *at;
    uint32_t u[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float f[4];
        decode4<kInt8>(u[e], f);
#pragma unroll
        for (int d = 0; d < 4; ++d) f[d] = __fdiv_rn(__fmul_rn(f[d], old), s);
        u[e] = encode4<kInt8, true>(f[0], f[1], f[2], f[3]);
    }
    *at = make_uint4(u[0], u[1], u[2], u[3]);
}
// 1 / s for encode8, or 0 where it or its products may leave fp32's normal range.
__device__ __forceinline__ float reciprocal(float s) { return s > 0x1p-100f && s < 0x1p100f ? __frcp_rn(s) : 0.f; }

// What one page of one sequence gets from the call.
struct AppendPage {
    int page, rows, held;  // page < 0: nothing; new rows, and older tokens in front of them
    size_t token;          // first new row in k and v
};
__device__ __forceinline__ AppendPage find_page(const CacheAppendArgs& p, int unit) {
    const CacheArgs& c = p.c;
    AppendPage r{-1, 0, 0, 0};
    const int b = find_sequence(p, unit);
    int t0, t1;
    seq_bounds(p.cu, p.cu64, b, p.T, t0, t1);
    // positions of the new tokens; those outside [0, max_pages P) are dropped
    const int end = cache_length(c, b), start = end - (t1 - t0);
    const int i = unit - ((t0 >> c.page_shift) + 2 * b) + (max(start, 0) >> c.page_shift);  // page of the sequence
    if (i < 0 || i >= c.max_pages) return r;
    const int lo = max(max(start, 0), i << c.page_shift), hi = min(end, (i + 1) << c.page_shift);
    if (lo >= hi) return r;
    const int page = c.table[(size_t)b * c.max_pages + i];
    if ((unsigned)page >= (unsigned)c.pages) return r;  // no such page: the rows are dropped
    r.page = page;
    r.rows = hi - lo;
    r.held = lo - (i << c.page_shift);
    r.token = (size_t)(t0 + lo - start);
    return r;
}

// R: passes of 16 rows that cover a page.
template <bool kInt8, int R>
__global__ void __launch_bounds__(256, R <= 4 ? 5 : 3) gdn_cache_append_kernel(CacheAppendArgs p) {
    __shared__ float s_max[8];
    pdl_wait();
    pdl_trigger();
    const CacheArgs& c = p.c;
    const int tid = threadIdx.x, head = blockIdx.y, row = tid >> 4;
    const AppendPage g = find_page(p, blockIdx.x);
    if (g.page < 0) return;
    const uint16_t* x = (blockIdx.z ? p.v : p.k) + (g.token * c.Hkv + head) * kD + 8 * (tid & 15);
    uint8_t* codes = static_cast<uint8_t*>(blockIdx.z ? c.v_cache : c.k_cache) + (((size_t)g.page * c.Hkv + head) << c.page_shift) * kD;
    float* scale = (blockIdx.z ? c.v_scale : c.k_scale) + (size_t)g.page * c.Hkv + head;

    uint4 w[R];
    __nv_bfloat162 top2 = __float2bfloat162_rn(0.f);
#pragma unroll
    for (int r = 0; r < R; ++r) {
        w[r] = make_uint4(0, 0, 0, 0);
        if (16 * r + row < g.rows) w[r] = __ldg(reinterpret_cast<const uint4*>(x + (size_t)(16 * r + row) * c.Hkv * kD));
    }
    const float old = g.held > 0 ? *scale : 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) top2 = abs_max(top2, w[r]);
    float top = fmaxf(__low2float(top2), __high2float(top2));
    if (top == INFINITY) {
        top = 0.f;
#pragma unroll 1
        for (int r = 0; r < R; ++r)
            if (16 * r + row < g.rows) top = fmaxf(top, finite_max(__ldg(reinterpret_cast<const uint4*>(x + (size_t)(16 * r + row) * c.Hkv * kD))));
    }
#pragma unroll
    for (int off = 16; off; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    if ((tid & 31) == 0) s_max[tid >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) top = fmaxf(top, s_max[w]);
    const float s = fmaxf(old, __fdiv_rn(top, kInt8 ? 127.f : 448.f)), inv = reciprocal(s);

    if (g.held > 0 && s > old)  // older tokens of the page to the new scale, 16 bytes a thread
        for (int j = tid; j < g.held * 8; j += 256) recode16<kInt8>(reinterpret_cast<uint4*>(codes) + j, old, s);
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (16 * r + row < g.rows)
            *reinterpret_cast<uint2*>(codes + (size_t)(g.held + 16 * r + row) * kD + 8 * (tid & 15)) = encode8<kInt8>(w[r], s, inv);
    if (tid == 0) *scale = s;
}

// A warp per (page, head, key or value), two rows a pass; the rows are read again for their codes.
template <bool kInt8>
__global__ void __launch_bounds__(256) gdn_cache_append_few_kernel(CacheAppendArgs p) {
    pdl_wait();
    pdl_trigger();
    const CacheArgs& c = p.c;
    const int lane = threadIdx.x & 31, row = lane >> 4, pair = blockIdx.y * 8 + (threadIdx.x >> 5), head = pair >> 1;
    if (head >= c.Hkv) return;
    const AppendPage g = find_page(p, blockIdx.x);
    if (g.page < 0) return;
    const uint16_t* x = (pair & 1 ? p.v : p.k) + (g.token * c.Hkv + head) * kD + 8 * (lane & 15);
    uint8_t* codes = static_cast<uint8_t*>(pair & 1 ? c.v_cache : c.k_cache) + (((size_t)g.page * c.Hkv + head) << c.page_shift) * kD;
    float* scale = (pair & 1 ? c.v_scale : c.k_scale) + (size_t)g.page * c.Hkv + head;
    const float old = g.held > 0 ? *scale : 0.f;
    uint4 w = make_uint4(0, 0, 0, 0);
    float top = 0.f;
#pragma unroll 1
    for (int r = 0; r < g.rows; r += 2) {
        w = make_uint4(0, 0, 0, 0);
        if (r + row < g.rows) w = __ldg(reinterpret_cast<const uint4*>(x + (size_t)(r + row) * c.Hkv * kD));
        top = fmaxf(top, finite_max(w));
    }
#pragma unroll
    for (int off = 16; off; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    const float s = fmaxf(old, __fdiv_rn(top, kInt8 ? 127.f : 448.f));
    if (g.held > 0 && s > old)
        for (int j = lane; j < g.held * 8; j += 32) recode16<kInt8>(reinterpret_cast<uint4*>(codes) + j, old, s);
#pragma unroll 1
    for (int r = 0; r < g.rows; r += 2) {
        if (r + row < g.rows) {
            if (g.rows > 2) w = __ldg(reinterpret_cast<const uint4*>(x + (size_t)(r + row) * c.Hkv * kD));
            *reinterpret_cast<uint2*>(codes + (size_t)(g.held + r + row) * kD + 8 * (lane & 15)) = encode8<kInt8>(w, s, reciprocal(s));
        }
    }
    if (lane == 0) *scale = s;
}

template <bool kInt8>
static cudaError_t launch_rows(const CacheAppendArgs& p, dim3 grid, cudaStream_t stream) {
    switch (p.c.page_shift) {
        case 4: return launch_pdl(gdn_cache_append_kernel<kInt8, 1>, grid, dim3(256), 0, stream, p);
        case 5: return launch_pdl(gdn_cache_append_kernel<kInt8, 2>, grid, dim3(256), 0, stream, p);
        case 6: return launch_pdl(gdn_cache_append_kernel<kInt8, 4>, grid, dim3(256), 0, stream, p);
        default: return launch_pdl(gdn_cache_append_kernel<kInt8, 8>, grid, dim3(256), 0, stream, p);
    }
}

int launch_cache_append(const CacheAppendArgs& p, cudaStream_t stream) {
    const unsigned units = (unsigned)((p.T >> p.c.page_shift) + 2 * p.c.B);
    cudaError_t e;
    if (p.T <= 8 * (long long)p.c.B) {  // at most 8 tokens a sequence on average
        const dim3 grid(units, (unsigned)(2 * p.c.Hkv + 7) / 8);
        e = p.c.int8 ? launch_pdl(gdn_cache_append_few_kernel<true>, grid, dim3(256), 0, stream, p)
                     : launch_pdl(gdn_cache_append_few_kernel<false>, grid, dim3(256), 0, stream, p);
    } else {
        const dim3 grid(units, (unsigned)p.c.Hkv, 2);
        e = p.c.int8 ? launch_rows<true>(p, grid, stream) : launch_rows<false>(p, grid, stream);
    }
    return e == cudaSuccess ? 0 : -1;
}

}  // namespace gdn
