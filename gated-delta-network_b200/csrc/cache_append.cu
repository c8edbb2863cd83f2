// cache_append.cu -- new key/value rows into a paged cache of 8-bit codes with a scale for each page and head.
//
// For every (page, head) that the call writes to, with m = 127 (int8) or 448 (e4m3):
//   s' = max(s, max |x| / m)     s: the page's scale, or 0 if its first token is among the new ones
//   code = round(x / s') for the new tokens, round(code s / s') for older ones where s' > s
// Quotients are IEEE fp32 and ties go to even, so the codes do not depend on the order of the work.
// max |x| is over finite values; infinities become the largest code, a NaN the code NaN (e4m3) or 0 (int8).
//
// Bound by HBM for prompts (768 bytes a token and head, each row read and written once) and by latency for decode steps.
// A warp holds its rows of a (page a sequence touches, head, key or value) in registers between the maximum and the
// encoding.  What a CTA waits for in turn (the lengths, the rows and the table, the page's scale) sets the rate, so many
// bytes have to be in flight: 16 rows a warp, 128 bytes a thread.  12 prompts of 10 to 8192 tokens, 8 heads, pages of 64:
// 22.1 us (5.0 TB/s); 200 x 1 token: 4.8 us.
// Divisions would cost more than the traffic.  With r = 1 / s rounded and q = x r rounded, q + r (x - q s) in two fused
// steps is x / s rounded (Markstein, IBM J. Res. Dev. 34, 1990), as long as nothing underflows.
#include <cuda_fp16.h>

#include "linear.cuh"
#include "prefill_kernels.cuh"

namespace gdn {

struct Sequence {
    int b, t0, t1, len;  // its new tokens, its length behind them
};
// The sequence whose touched pages hold slot u: the last one with cu[b] / P + 2 b <= u.  n tokens touch at most
// floor(n / P) + 2 pages, so these bases need no prefix sum.  32 probes a round, all lanes of every warp together.
__device__ __forceinline__ Sequence find_sequence(const CacheAppendArgs& p, int u) {
    int lo = 0, n = p.c.B;  // candidates lo .. lo + n - 1; lo always qualifies
    const int lane = threadIdx.x & 31;
    while (true) {
        const int step = (n + 31) / 32, at = lo + lane * step;
        const bool any = lane * step < n;
        Sequence x{at, 0, 0, 0};
        if (any) {
            seq_bounds(p.cu, p.cu64, at, p.T, x.t0, x.t1);
            x.len = cache_length(p.c, at);
        }
        const unsigned hit = __ballot_sync(0xffffffffu, any && (x.t0 >> p.c.page_shift) + 2 * at <= u);
        const int last = hit ? 31 - __clz(hit) : 0;
        if (step == 1) {
            x.b = lo + last;
            x.t0 = __shfl_sync(0xffffffffu, x.t0, last);
            x.t1 = __shfl_sync(0xffffffffu, x.t1, last);
            x.len = __shfl_sync(0xffffffffu, x.len, last);
            return x;
        }
        n = min(step, n - last * step);
        lo += last * step;
    }
}

// Largest magnitude of 8 bf16 values so far, per half; a NaN stays.
__device__ __forceinline__ __nv_bfloat162 abs_max(__nv_bfloat162 top, uint4 w) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) top = __hmax2_nan(top, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&u[e])));
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
// x / s rounded, for finite x and r = 1 / s rounded, 2^-60 < s < 2^60.  (Quotients below 2^-30 may be off; their codes are 0.)
// Formed negated, which keeps the sign of a zero.
__device__ __forceinline__ float2 quotients(float2 x, float s, float r) {
    const float2 minus = make_float2(-r, -r), q = mul2(x, minus), y = fma2(fma2(q, make_float2(s, s), x), minus, q);
    return make_float2(-y.x, -y.y);
}
__device__ __forceinline__ float reciprocal(float s) { return s > 0x1p-60f && s < 0x1p60f ? __frcp_rn(s) : 0.f; }
// Eight bf16 values to codes.  r: reciprocal(s), or 0 where there is none or not all values are finite.
// (s = 0: zeros, or values whose scale is below fp32; infinities and NaN among them keep their codes.)
template <bool kInt8>
__device__ __forceinline__ uint2 encode8(uint4 w, float s, float r) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    float2 x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = make_float2(__uint_as_float(u[e] << 16), __uint_as_float(u[e] & 0xffff0000u));
    if (r != 0.f) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = quotients(x[e], s, r);
        return make_uint2(encode4<kInt8, false>(x[0].x, x[0].y, x[1].x, x[1].y), encode4<kInt8, false>(x[2].x, x[2].y, x[3].x, x[3].y));
    }
    if (!(s > 0.f)) {
        s = 1.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = make_float2(fabsf(x[e].x) < INFINITY ? 0.f : x[e].x, fabsf(x[e].y) < INFINITY ? 0.f : x[e].y);
    }
    return make_uint2(encode4<kInt8, true>(__fdiv_rn(x[0].x, s), __fdiv_rn(x[0].y, s), __fdiv_rn(x[1].x, s), __fdiv_rn(x[1].y, s)),
                      encode4<kInt8, true>(__fdiv_rn(x[2].x, s), __fdiv_rn(x[2].y, s), __fdiv_rn(x[3].x, s), __fdiv_rn(x[3].y, s)));
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
// 16 codes of scale `old` to scale s > old.
template <bool kInt8>
__device__ __forceinline__ void recode16(uint4* at, float old, float s, float r) {
    const uint4 y = *at;
    uint32_t u[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float f[4];
        decode4<kInt8>(u[e], f);
        float2 a = mul2(make_float2(f[0], f[1]), make_float2(old, old)), b = mul2(make_float2(f[2], f[3]), make_float2(old, old));
        if (r != 0.f) {
            a = quotients(a, s, r);
            b = quotients(b, s, r);
        } else {
            a = make_float2(__fdiv_rn(a.x, s), __fdiv_rn(a.y, s));
            b = make_float2(__fdiv_rn(b.x, s), __fdiv_rn(b.y, s));
        }
        u[e] = encode4<kInt8, true>(a.x, a.y, b.x, b.y);
    }
    *at = make_uint4(u[0], u[1], u[2], u[3]);
}

// What one page of one sequence gets from the call.
struct AppendPage {
    int page, rows, held;  // the page's number as the table has it; new rows, and older tokens in front of them
    size_t token;          // first new row in k and v
};
__device__ __forceinline__ AppendPage find_page(const CacheAppendArgs& p, int unit) {
    const CacheArgs& c = p.c;
    AppendPage r{-1, 0, 0, 0};
    const Sequence q = find_sequence(p, unit);
    // positions of the new tokens; those outside [0, max_pages P) are dropped
    const int start = q.len - (q.t1 - q.t0);
    const int i = unit - ((q.t0 >> c.page_shift) + 2 * q.b) + (max(start, 0) >> c.page_shift);  // page of the sequence
    if (i < 0 || i >= c.max_pages) return r;
    const int lo = max(max(start, 0), i << c.page_shift), hi = min(q.len, (i + 1) << c.page_shift);
    if (lo >= hi) return r;
    r.page = c.table[(size_t)q.b * c.max_pages + i];
    r.rows = hi - lo;
    r.held = lo - (i << c.page_shift);
    r.token = (size_t)(q.t0 + lo - start);
    return r;
}

// W warps for each (page, head, key or value), 8 / W of these a CTA; a warp takes 16 new rows, two a load (W = 1: 16 at a
// time).
template <bool kInt8, int W>
__global__ void __launch_bounds__(256, 4) gdn_cache_append_kernel(CacheAppendArgs p) {
    __shared__ float s_max[8];
    pdl_wait();
    pdl_trigger();
    const CacheArgs& c = p.c;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp % W;
    const int pair = blockIdx.y * (8 / W) + warp / W, head = pair >> 1;
    const AppendPage g = find_page(p, blockIdx.x);
    if (g.rows == 0) return;  // (the whole CTA, and below)
    const bool here = head < c.Hkv;
    const int rows = here ? g.rows : 0, row = lane >> 4;
    const uint16_t* x = (pair & 1 ? p.v : p.k) + (g.token * c.Hkv + head) * kD + 8 * (lane & 15);
    auto load = [&](int r) { return __ldg(reinterpret_cast<const uint4*>(x + (size_t)r * c.Hkv * kD)); };

    constexpr int L = 8;
    uint4 w[L];
    auto load_block = [&](int r0) {
        const uint16_t* at = x + (size_t)(r0 + row) * c.Hkv * kD;
        const int left = rows - r0 - row;
#pragma unroll
        for (int i = 0; i < L; ++i, at += 2 * c.Hkv * kD)
            w[i] = 2 * i < left ? __ldg(reinterpret_cast<const uint4*>(at)) : make_uint4(0, 0, 0, 0);
    };
    int r0 = 2 * L * part;  // W = 1: the last block afterwards
    load_block(r0);  // with the table's entry still on its way
    if ((unsigned)g.page >= (unsigned)c.pages) return;  // no such page: the rows are dropped
    uint8_t* codes = static_cast<uint8_t*>(pair & 1 ? c.v_cache : c.k_cache) + (((size_t)g.page * c.Hkv + head) << c.page_shift) * kD;
    float* scale = (pair & 1 ? c.v_scale : c.k_scale) + (size_t)g.page * c.Hkv + head;
    const float old = here && g.held > 0 ? *scale : 0.f;
    __nv_bfloat162 top2 = __float2bfloat162_rn(0.f);
    while (true) {
#pragma unroll
        for (int i = 0; i < L; ++i) top2 = abs_max(top2, w[i]);
        if (W > 1 || r0 + 2 * L >= rows) break;
        load_block(r0 += 2 * L);
    }
    float top = fmaxf(__low2float(top2), __high2float(top2));
    const bool odd = !(__low2float(top2) < INFINITY && __high2float(top2) < INFINITY);  // infinities or NaN among them
    if (odd) {
        top = 0.f;
#pragma unroll 1
        for (int r = 2 * L * part + row; r < min(rows, r0 + 2 * L); r += 2) top = fmaxf(top, finite_max(load(r)));
    }
#pragma unroll
    for (int off = 16; off; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    if (W > 1) {
        if (lane == 0) s_max[warp] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < W; ++i) top = fmaxf(top, s_max[warp - part + i]);
    }
    const float s = fmaxf(old, __fdiv_rn(top, kInt8 ? 127.f : 448.f)), inv = odd ? 0.f : reciprocal(s);

    codes += g.held * kD;
    while (true) {
        uint8_t* to = codes + (r0 + row) * kD + 8 * (lane & 15);
        const int left = rows - r0 - row;
        if (inv != 0.f) {
#pragma unroll
            for (int i = 0; i < L; ++i)
                if (2 * i < left) *reinterpret_cast<uint2*>(to + 2 * i * kD) = encode8<kInt8>(w[i], s, inv);
        } else {
#pragma unroll 1
            for (int i = 0; 2 * i < min(left, 2 * L); ++i) *reinterpret_cast<uint2*>(to + 2 * i * kD) = encode8<kInt8>(load(r0 + row + 2 * i), s, 0.f);
        }
        if (W > 1 || r0 == 0) break;
        load_block(r0 -= 2 * L);
    }
    codes -= g.held * kD;
    if (here && g.held > 0 && s > old)  // older tokens of the page to the new scale, 16 bytes a thread
#pragma unroll 1
        for (int j = 32 * part + lane; j < g.held * 8; j += 32 * W) recode16<kInt8>(reinterpret_cast<uint4*>(codes) + j, old, s, reciprocal(s));
    if (here && part == 0 && lane == 0) *scale = s;
}

template <bool kInt8, int W>
static cudaError_t launch_append(const CacheAppendArgs& p, cudaStream_t stream) {
    const dim3 grid((unsigned)((p.T >> p.c.page_shift) + 2 * p.c.B), (unsigned)(2 * p.c.Hkv * W + 7) / 8);
    return launch_pdl(gdn_cache_append_kernel<kInt8, W>, grid, dim3(256), 0, stream, p);
}
// A warp for each 16 rows of a page, or one for all of them where sequences get 32 tokens at most on average.  8 heads,
// pages of 64, us with one warp a page and with four: 200 x 1 token 4.8 and 11.5, 200 x 32 10.4 and 17.9, 64 x 32 8.0 and
// 7.8, 4 x 32 4.3 and 3.0, 64 x 64 12.4 and 9.4.  (CTAs cost as much as rows here, and half of a short call's get none.)
template <bool kInt8>
static cudaError_t launch_append(const CacheAppendArgs& p, cudaStream_t stream) {
    switch (p.T <= 32 * (long long)p.c.B ? 4 : p.c.page_shift) {
        case 4: return launch_append<kInt8, 1>(p, stream);
        case 5: return launch_append<kInt8, 2>(p, stream);
        case 6: return launch_append<kInt8, 4>(p, stream);
        default: return launch_append<kInt8, 8>(p, stream);
    }
}

int launch_cache_append(const CacheAppendArgs& p, cudaStream_t stream) {
    return (p.c.int8 ? launch_append<true>(p, stream) : launch_append<false>(p, stream)) == cudaSuccess ? 0 : -1;
}

}  // namespace gdn
