// cache_attend.cu -- attention of the last Q tokens of every sequence over a paged cache of 8-bit codes.
//
// For q row (i, g) of kv head h (i < Q, g < Hq / Hkv), over the positions j < len - Q + 1 + i:
//   s_j = scale q . k_j,   out = sum_j e^{s_j - m} v_j / sum_j e^{s_j - m},   x = code * scale[page][h]
// A row that sees no position is zero.
//
// Bound by HBM for up to about 16 rows a kv head: 256 bytes a token and head, each read once.
//  * Codes go to the tensor cores as fp16, which holds every int8 and e4m3 value exactly (mma.sync m16n8k16,
//    fp32 accumulation: 16 rows are all there is, a 128-row tcgen05 tile would be 7/8 empty). q is brought to
//    fp16 by a power of two per row (its largest element lands in [1, 2), the others keep an absolute 2^-25 of
//    it), and the page's key scale multiplies the fp32 scores.
//  * The value scale enters the weights: p v_scale / r <= 1 in fp16 with r the largest value scale so far, kept
//    like the running maximum, so the accumulator never sees the scales' range; the sum of p stays fp32 and unrounded.
//  * Both contractions may permute their index, so a thread takes 16 consecutive bytes of a row and no fragment
//    needs a shuffle or a transposing load: key step s of lane l holds dims 16 (l % 4) + 4 s .. and the same of q;
//    value lane l holds dims 16 (l / 4) .. of the four tokens whose weights it owns. Every thread reads back only the
//    shared memory it filled itself (cp.async), so the ring needs no barrier.
//  * Tokens are cut evenly over the CTAs whatever the lengths: all (sequence, head, 16-row tile) segments in 32-token
//    blocks on one line, an equal stretch of it per CTA. A stretch's first and last segment may continue in a
//    neighbour; those pieces go to the workspace, and a second launch joins them.
#include <cuda_fp16.h>

#include "linear.cuh"
#include "prefill_kernels.cuh"

namespace gdn {

namespace att {
constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kBlock = 32;                       // tokens of the unit that is divided over the CTAs
constexpr int kStages = 3;
constexpr int kStageBytes = 4096;                // a warp's 16 tokens of k and v: 8 x 16 bytes a lane
constexpr int kRing = kWarps * kStages * kStageBytes;
constexpr int kOffQ = kRing;                     // q as A fragments: [8 steps][32 lanes][16 bytes]
constexpr int kOffF = kOffQ + 4096;              // f32 [16] row factors
constexpr int kOffM = kOffF + 64;                // f32 [kWarps][16] maxima, then sums
constexpr int kSmem = kOffM + 2 * kWarps * 16 * 4;
constexpr float kLog2e = 1.4426950408889634f;
static_assert(kWarps * 16 * 128 * 4 <= kRing, "the warps' results take the ring's place");
}  // namespace att

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The two codes in the low (kHigh: high) half of w as fp16, exactly.  int8: w holds code + 128.
template <bool kInt8, bool kHigh>
__device__ __forceinline__ uint32_t codes_f16(uint32_t w) {
    uint32_t h;
    if (kInt8) {
        h = __byte_perm(w, 0x64646464u, kHigh ? 0x4342 : 0x4140);  // 1024 + code + 128
        const __half2 y = __hsub2(*reinterpret_cast<__half2*>(&h), __half2half2(__ushort_as_half(0x6480)));
        return *reinterpret_cast<const uint32_t*>(&y);
    }
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)(kHigh ? w >> 16 : w)));
    return h;
}

struct Line {  // segment (b, h, row tile) and the 32-token blocks of it
    int b, seg_in_b, blocks;
    long long begin;  // first block on the line
};

__device__ __forceinline__ int visible_length(const CacheArgs& c, int b) {
    return (int)min((long long)cache_length(c, b), (long long)c.max_pages << c.page_shift);
}
__device__ __forceinline__ int seq_blocks(const CacheArgs& c, int b) {
    return max(1, (visible_length(c, b) + att::kBlock - 1) / att::kBlock);
}

// Total blocks of the line, and the sequence that holds block `at` with the line position of its first block.
// All threads of the CTA take part; two passes over the lengths.
__device__ __forceinline__ long long line_total(const CacheArgs& c, int segs, long long* s_sum) {
    long long sum = 0;
    for (int b = threadIdx.x; b < c.B; b += att::kThreads) sum += seq_blocks(c, b);
#pragma unroll
    for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = sum;
    __syncthreads();
    sum = 0;
#pragma unroll
    for (int w = 0; w < att::kWarps; ++w) sum += s_sum[w];
    __syncthreads();
    return sum * segs;
}
__device__ __forceinline__ void line_find(const CacheArgs& c, int segs, long long at, long long* s_sum, int* s_b, long long* s_begin) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long before = 0;  // blocks of the sequences in front of this pass
    for (int base = 0; base < c.B; base += att::kThreads) {
        const int b = base + threadIdx.x;
        const long long mine = b < c.B ? (long long)seq_blocks(c, b) * segs : 0;
        long long x = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, x, off);
            if (lane >= off) x += y;
        }
        if (lane == 31) s_sum[warp] = x;
        __syncthreads();
        long long total = 0;
#pragma unroll
        for (int w = 0; w < att::kWarps; ++w) {
            if (w < warp) x += s_sum[w];
            total += s_sum[w];
        }
        const long long lo = before + x - mine;
        if (at >= lo && at < lo + mine) {
            *s_b = b;
            *s_begin = lo;
        }
        before += total;
        __syncthreads();
        if (at < before) break;
    }
}

template <bool kInt8>
__global__ void __launch_bounds__(att::kThreads, 2) gdn_cache_attend_kernel(CacheAttendArgs p) {
    using namespace att;
    extern __shared__ __align__(128) unsigned char sm[];
    __shared__ long long s_sum[kWarps], s_begin;
    __shared__ int s_b, s_status;
    const CacheArgs& c = p.c;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    float* s_f = reinterpret_cast<float*>(sm + kOffF);
    float* s_m = reinterpret_cast<float*>(sm + kOffM);
    float* s_l = s_m + kWarps * 16;
    pdl_wait();
    pdl_trigger();
    if (tid == 0) s_status = 0;

    const int G = p.Hq / c.Hkv, R = p.Q * G, tiles = (R + 15) / 16, segs = c.Hkv * tiles;
    const long long total = line_total(c, segs, s_sum);
    // at least a block for each warp, so that short caches are not cut into more pieces than they are worth
    const long long ctas = min((long long)gridDim.x, (total + kWarps - 1) / kWarps);
    const long long first = blockIdx.x * total / ctas, end = min(total, (blockIdx.x + 1) * total / ctas);
    int2 piece = make_int2(-1, 0);  // the segment that begins here and ends elsewhere (thread 0)
    if (blockIdx.x >= ctas) {
        if (tid == 0) p.piece[blockIdx.x] = make_int4(-1, 0, 0, 0);
        return;
    }
    line_find(c, segs, first, s_sum, &s_b, &s_begin);
    __syncthreads();
    int b = s_b;
    long long begin = s_begin;

    for (long long at = first; at < end;) {
        const int nb = seq_blocks(c, b);
        if (at >= begin + (long long)nb * segs) {
            begin += (long long)nb * segs;
            ++b;
            continue;
        }
        const int seg = (int)((at - begin) / nb), h = seg / tiles, row0 = (seg % tiles) * 16;
        const long long seg_begin = begin + (long long)seg * nb, seg_end = seg_begin + nb;
        const long long stop = min(seg_end, end);
        const int len = visible_length(c, b);
        if (tid == 0 && cache_length(c, b) > len) s_status = kErrBadSeqlens;
        const int tok0 = (int)(at - seg_begin) * kBlock, tok1 = min(len, (int)(stop - seg_begin) * kBlock);
        const int steps = tok1 > tok0 ? (tok1 - tok0 + 15) / 16 : 0;

        // q rows as fp16 fragments; 16 threads a row
        {
            const int r = tid >> 4, x = tid & 15, row = row0 + r;
            uint4 w = make_uint4(0, 0, 0, 0);
            if (row < R)
                w = *reinterpret_cast<const uint4*>(p.q + (((size_t)b * p.Q + row / G) * p.Hq + h * G + row % G) * kD + 8 * x);
            const uint32_t u[4] = {w.x, w.y, w.z, w.w};
            float f[8], top = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                f[2 * e] = __uint_as_float(u[e] << 16);
                f[2 * e + 1] = __uint_as_float(u[e] & 0xffff0000u);
                top = fmaxf(top, fmaxf(fabsf(f[2 * e]), fabsf(f[2 * e + 1])));
            }
#pragma unroll
            for (int off = 8; off; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
            // 2^-e with top in [2^e, 2^(e+1)); kept within what 2^e and 2^-e can both hold
            const int ex = min(max((int)(__float_as_uint(top) >> 23), 2), 252);
            const float inv = __uint_as_float((uint32_t)(254 - ex) << 23);
            if (x == 0) s_f[r] = __uint_as_float((uint32_t)ex << 23) * (p.scale * kLog2e);
            // dims 8 x .. 8 x + 7: 16-byte chunk x / 2, steps 2 (x % 2) and the next; the second half of the dims is steps 4-7
            const int xl = (x >> 1) & 3, s0 = 2 * (x & 1) + 4 * (x >> 3);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const __half2 a = __floats2half2_rn(f[4 * e] * inv, f[4 * e + 1] * inv);
                const __half2 d = __floats2half2_rn(f[4 * e + 2] * inv, f[4 * e + 3] * inv);
                uint32_t* dst = reinterpret_cast<uint32_t*>(sm + kOffQ + (s0 + e) * 512 + ((r & 7) * 4 + xl) * 16);
                dst[r >> 3] = *reinterpret_cast<const uint32_t*>(&a);
                dst[2 + (r >> 3)] = *reinterpret_cast<const uint32_t*>(&d);
            }
        }
        __syncthreads();

        float acc[16][4];
#pragma unroll
        for (int j = 0; j < 16; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, vref = 0.f;
        const int ra = row0 + (lane >> 2), rb = ra + 8;
        const int lim[2] = {len - p.Q + 1 + ra / G, len - p.Q + 1 + rb / G};  // positions that the rows see
        const float rf[2] = {s_f[lane >> 2], s_f[(lane >> 2) + 8]};

        unsigned char* ring = sm + warp * kStages * kStageBytes + lane * 16;
        const int mine = steps > warp ? (steps - warp + kWarps - 1) / kWarps : 0;  // steps warp, warp + 8, ..
        const int* trow = c.table + (size_t)b * c.max_pages;
        const size_t head_stride = (size_t)kD << c.page_shift;
        auto page_of = [&](int n) { return n < mine ? trow[(tok0 + 16 * (warp + kWarps * n)) >> c.page_shift] : 0; };
        auto issue = [&](int n, int page) {
            if (n < mine) {
                const int t = tok0 + 16 * (warp + kWarps * n);
                const bool ok = (unsigned)page < (unsigned)c.pages;
                const size_t off = ((size_t)(ok ? page : 0) * c.Hkv + h) * head_stride + (size_t)(t & ((1 << c.page_shift) - 1)) * kD;
                const unsigned char* kp = static_cast<const unsigned char*>(c.k_cache) + off;
                const unsigned char* vp = static_cast<const unsigned char*>(c.v_cache) + off;
                unsigned char* st = ring + (n % kStages) * kStageBytes;
                const int left = ok ? tok1 - t : 0;  // rows behind the end arrive as zeros
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = (lane >> 2) + 8 * (i >> 1), ch = (lane & 3) + 4 * (i & 1);
                    cp_async16(st + i * 512, kp + row * kD + ch * 16, row < left);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = 2 * (lane & 3) + (i & 1) + 8 * (i >> 1);
                    cp_async16(st + 2048 + i * 512, vp + row * kD + (lane >> 2) * 16, row < left);
                }
            }
            cp_async_commit();
        };
        int pg[kStages];  // pages of the steps in the ring, and of the next one to issue
#pragma unroll
        for (int n = 0; n < kStages; ++n) pg[n] = page_of(n);
#pragma unroll
        for (int n = 0; n < kStages - 1; ++n) issue(n, pg[n]);

        for (int n = 0; n < mine; ++n) {
            const int page = pg[0];
            issue(n + kStages - 1, pg[kStages - 1]);
#pragma unroll
            for (int i = 0; i + 1 < kStages; ++i) pg[i] = pg[i + 1];
            pg[kStages - 1] = page_of(n + kStages);
            const bool ok = (unsigned)page < (unsigned)c.pages;
            if (!ok) s_status = kErrBadPage;
            const size_t si = (size_t)(ok ? page : 0) * c.Hkv + h;
            const float ks = c.k_scale[si], vs = ok ? c.v_scale[si] : 0.f;
            cp_async_wait<kStages - 1>();
            const unsigned char* st = ring + (n % kStages) * kStageBytes;
            const int t = tok0 + 16 * (warp + kWarps * n);

            float s[2][4] = {};
#pragma unroll
            for (int half = 0; half < 2; ++half) {  // dims 0-63, 64-127
                uint4 kk[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    kk[i] = *reinterpret_cast<const uint4*>(st + (2 * i + half) * 512);
                    if (kInt8) kk[i] = make_uint4(kk[i].x ^ 0x80808080u, kk[i].y ^ 0x80808080u, kk[i].z ^ 0x80808080u, kk[i].w ^ 0x80808080u);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint4 a = *reinterpret_cast<const uint4*>(sm + kOffQ + (4 * half + e) * 512 + lane * 16);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t w = e == 0 ? kk[i].x : e == 1 ? kk[i].y : e == 2 ? kk[i].z : kk[i].w;
                        mma_f16(s[i], a.x, a.y, a.z, a.w, codes_f16<kInt8, false>(w), codes_f16<kInt8, true>(w));
                    }
                }
            }
            // scores in base 2; hidden ones are -infinity
            float top[2] = {m[0], m[1]};
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int pos = t + 8 * i + 2 * (lane & 3) + (e & 1);
                    s[i][e] = ok && pos < lim[e >> 1] ? s[i][e] * (ks * rf[e >> 1]) : -INFINITY;
                    top[e >> 1] = fmaxf(top[e >> 1], s[i][e]);
                }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
                top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
            }
            const float vnew = fmaxf(vref, vs);
            if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1]) || vnew > vref) {
                const float vr = vnew > 0.f ? vref / vnew : 1.f;
                float f[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    f[r] = m[r] == -INFINITY ? 0.f : ex2(m[r] - top[r]);
                    l[r] *= f[r];
                    f[r] *= vr;
                    m[r] = top[r];
                }
                vref = vnew;
#pragma unroll
                for (int j = 0; j < 16; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[j][e] *= f[e >> 1];
            }
            const float mv = vref > 0.f ? vs / vref : 0.f;
            uint32_t a[4];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float base = m[r] == -INFINITY ? 0.f : m[r];
                    const float x = ex2(s[i][2 * r] - base), y = ex2(s[i][2 * r + 1] - base);
                    l[r] += x + y;
                    const __half2 w = __floats2half2_rn(x * mv, y * mv);
                    a[2 * i + r] = *reinterpret_cast<const uint32_t*>(&w);
                }
            uint4 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = *reinterpret_cast<const uint4*>(st + 2048 + i * 512);
                if (kInt8) v[i] = make_uint4(v[i].x ^ 0x80808080u, v[i].y ^ 0x80808080u, v[i].z ^ 0x80808080u, v[i].w ^ 0x80808080u);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // dims 4 e .. 4 e + 3 of the lane's 16
                uint32_t x[2][2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint4 &v0 = v[2 * i], &v1 = v[2 * i + 1];
                    const uint32_t w0 = e == 0 ? v0.x : e == 1 ? v0.y : e == 2 ? v0.z : v0.w;
                    const uint32_t w1 = e == 0 ? v1.x : e == 1 ? v1.y : e == 2 ? v1.z : v1.w;
                    x[i][0] = __byte_perm(w0, w1, 0x5140);  // tokens t, t + 1 of dims 0 and 1
                    x[i][1] = __byte_perm(w0, w1, 0x7362);
                }
#pragma unroll
                for (int d = 0; d < 2; ++d) {
                    mma_f16(acc[4 * e + 2 * d], a[0], a[1], a[2], a[3], codes_f16<kInt8, false>(x[0][d]), codes_f16<kInt8, false>(x[1][d]));
                    mma_f16(acc[4 * e + 2 * d + 1], a[0], a[1], a[2], a[3], codes_f16<kInt8, true>(x[0][d]), codes_f16<kInt8, true>(x[1][d]));
                }
            }
        }
        cp_async_wait<0>();
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        }

        // join the warps: every warp's result at the common maximum
        if ((lane & 3) == 0) {
            s_m[warp * 16 + (lane >> 2)] = m[0];
            s_m[warp * 16 + (lane >> 2) + 8] = m[1];
            s_l[warp * 16 + (lane >> 2)] = l[0];
            s_l[warp * 16 + (lane >> 2) + 8] = l[1];
        }
        __syncthreads();  // also: every warp is done with its ring
        float* wacc = reinterpret_cast<float*>(sm);  // [kWarps][16][128], 16-byte chunks XORed with the row
        float mall[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            mall[r] = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) mall[r] = fmaxf(mall[r], s_m[w * 16 + (lane >> 2) + 8 * r]);
            const float f = l[r] != 0.f ? ex2(m[r] - mall[r]) * vref : 0.f;
            const int row = (lane >> 2) + 8 * r;
#pragma unroll
            for (int e = 0; e < 2; ++e)  // dims 32 (lane % 4) + 16 e + 0 .. 15
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int ch = 8 * (lane & 3) + 4 * e + j;
                    *reinterpret_cast<float4*>(wacc + (warp * 16 + row) * 128 + (ch ^ (row & 7)) * 4) =
                        make_float4(acc[4 * j][2 * r + e] * f, acc[4 * j + 1][2 * r + e] * f, acc[4 * j + 2][2 * r + e] * f,
                                    acc[4 * j + 3][2 * r + e] * f);
                }
        }
        __syncthreads();
        {
            const int row = tid >> 4;
            float mm = -INFINITY, ll = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, s_m[w * 16 + row]);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float mw = s_m[w * 16 + row];
                const float lw = s_l[w * 16 + row];
                if (lw != 0.f) ll += lw * ex2(mw - mm);  // a NaN stays one
            }
            float o[8] = {};
#pragma unroll
            for (int w = 0; w < kWarps; ++w)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int ch = 2 * (tid & 15) + e;
                    const float4 x = *reinterpret_cast<const float4*>(wacc + (w * 16 + row) * 128 + (ch ^ (row & 7)) * 4);
                    o[4 * e] += x.x;
                    o[4 * e + 1] += x.y;
                    o[4 * e + 2] += x.z;
                    o[4 * e + 3] += x.w;
                }
            const bool whole = at == seg_begin && stop == seg_end;
            const int r = row0 + row;
            if (r < R) {
                if (whole) {
                    const float inv = ll > 0.f || ll != ll ? 1.f / ll : 0.f;
                    uint32_t u[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) u[e] = pack_bf16x2(o[2 * e] * inv, o[2 * e + 1] * inv);
                    *reinterpret_cast<uint4*>(p.out + (((size_t)b * p.Q + r / G) * p.Hq + h * G + r % G) * kD + 8 * (tid & 15)) =
                        make_uint4(u[0], u[1], u[2], u[3]);
                } else {
                    const size_t slot = (2 * (size_t)blockIdx.x + (at == seg_begin ? 1 : 0)) * 16 + row;
                    float4* d = reinterpret_cast<float4*>(p.acc + slot * 128 + 8 * (tid & 15));
                    d[0] = make_float4(o[0], o[1], o[2], o[3]);
                    d[1] = make_float4(o[4], o[5], o[6], o[7]);
                    if ((tid & 15) == 0) {
                        p.ml[slot * 2] = mm;
                        p.ml[slot * 2 + 1] = ll;
                    }
                }
            }
            if (!whole && at == seg_begin && tid == 0) {
                // the CTA that holds the segment's last block
                const long long last = (seg_end * ctas - 1) / total;
                piece = make_int2(b * segs + seg, (int)(last - blockIdx.x));
            }
        }
        at = stop;
        __syncthreads();
    }
    if (tid == 0) p.piece[blockIdx.x] = make_int4(piece.x, piece.y, s_status, 0);
}

// Joins a segment that several CTAs of the line hold: CTA x takes the one that CTA x began, row y of its tile.
__global__ void __launch_bounds__(128) gdn_cache_join_kernel(CacheAttendArgs p) {
    __shared__ float4 s_o[4][32];
    __shared__ float s_l[4];
    pdl_wait();
    pdl_trigger();
    if (blockIdx.x == 0 && blockIdx.y == 0) {  // the call's status: any of the CTAs'
        int st = 0;
        for (int i = threadIdx.x; i < (int)gridDim.x; i += 128) st = max(st, p.piece[i].z);
        const int page = __syncthreads_or(st == kErrBadPage), any = __syncthreads_or(st != 0);
        if (threadIdx.x == 0) *p.status = page ? kErrBadPage : any ? kErrBadSeqlens : 0;
    }
    const int4 pc = p.piece[blockIdx.x];
    if (pc.x < 0) return;
    const int G = p.Hq / p.c.Hkv, R = p.Q * G, tiles = (R + 15) / 16, segs = p.c.Hkv * tiles;
    const int b = pc.x / segs, seg = pc.x % segs, h = seg / tiles, r = (seg % tiles) * 16 + blockIdx.y;
    if (r >= R) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto slot = [&](int i) { return ((size_t)(2 * (blockIdx.x + i) + (i == 0 ? 1 : 0))) * 16 + blockIdx.y; };
    float m = -INFINITY;
    for (int i = lane; i <= pc.y; i += 32) m = fmaxf(m, p.ml[slot(i) * 2]);
#pragma unroll
    for (int off = 16; off; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = warp; i <= pc.y; i += 4) {
        const float li = p.ml[slot(i) * 2 + 1], f = li != 0.f ? ex2(p.ml[slot(i) * 2] - m) : 0.f;
        const float4 x = reinterpret_cast<const float4*>(p.acc + slot(i) * 128)[lane];
        l = fmaf(f, li, l);
        o = make_float4(fmaf(f, x.x, o.x), fmaf(f, x.y, o.y), fmaf(f, x.z, o.z), fmaf(f, x.w, o.w));
    }
    s_o[warp][lane] = o;
    if (lane == 0) s_l[warp] = l;
    __syncthreads();
    if (warp == 0) {
        l = s_l[0] + s_l[1] + s_l[2] + s_l[3];
        const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
        float4 x = s_o[0][lane];
#pragma unroll
        for (int w = 1; w < 4; ++w) {
            x.x += s_o[w][lane].x;
            x.y += s_o[w][lane].y;
            x.z += s_o[w][lane].z;
            x.w += s_o[w][lane].w;
        }
        *reinterpret_cast<uint2*>(p.out + (((size_t)b * p.Q + r / G) * p.Hq + h * G + r % G) * kD + 4 * lane) =
            make_uint2(pack_bf16x2(x.x * inv, x.y * inv), pack_bf16x2(x.z * inv, x.w * inv));
    }
}

template <bool kInt8>
static int launch_attend(const CacheAttendArgs& p, cudaStream_t stream) {
    if (cudaFuncSetAttribute(gdn_cache_attend_kernel<kInt8>, cudaFuncAttributeMaxDynamicSharedMemorySize, att::kSmem) != cudaSuccess)
        return -1;
    if (launch_pdl(gdn_cache_attend_kernel<kInt8>, dim3(kAttendCtas), dim3(att::kThreads), att::kSmem, stream, p) != cudaSuccess)
        return -1;
    const int rows = p.Q * (p.Hq / p.c.Hkv);
    return launch_pdl(gdn_cache_join_kernel, dim3(kAttendCtas, (unsigned)(rows < 16 ? rows : 16)), dim3(128), 0, stream, p) == cudaSuccess ? 0 : -1;
}

int launch_cache_attend(const CacheAttendArgs& p, cudaStream_t stream) {
    return p.c.int8 ? launch_attend<true>(p, stream) : launch_attend<false>(p, stream);
}

}  // namespace gdn
