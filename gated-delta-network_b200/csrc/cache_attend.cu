// cache_attend.cu -- attention of the last Q tokens of every sequence over a paged cache of 8-bit codes.
//
// For q row (i, g) of kv head h (i < Q, g < Hq / Hkv), over the positions j < len - Q + 1 + i:
//   s_j = scale q . k_j,   out = sum_j e^{s_j - m} v_j / sum_j e^{s_j - m},   x = code * scale[page][h]
// A row that sees no position is zero.
//
// Bound by HBM for up to some 16 rows a kv head: 256 bytes a token and head, each read once.
//  * Codes go to the tensor cores as fp16, which holds every int8 and e4m3 value exactly (mma.sync m16n8k16,
//    fp32 accumulation).  The tokens are the 16 rows of S^T = K Q^T, the dims those of O^T = V^T P^T, and the q rows
//    the 8 columns, so a decode step of 4 or 8 rows wastes little; a 128-row tcgen05 tile would.  More rows take
//    several column tiles against the same converted fragments (the conversion costs as much as the products).
//  * q is brought to fp16 by a power of two per row (its largest element lands in [1, 2), the others keep an absolute
//    2^-25 of it), and the page's key scale multiplies the fp32 scores.
//  * The maximum is a reference that moves only when a score exceeds it by 4 (base 2), so most steps need no
//    reduction and no rescaling; weights stay below 2^4 in fp16, their sum is fp32 and of the unrounded ones.
//  * The value scale enters the weights, p v_scale / r, so the accumulator never sees the scales' range.  r is a power of
//    two for each row, at most its largest p v_scale so far and some 9 bits below it at worst, and moves like the maximum.
//    (Of the weights, not of the scales: a page of large values that has no weight must not cost the others their bits.)
//    Weights round to 2^-11, or to 2^-25 r where they are below 2^-14 r.
//  * A row is kept from what it does not see: 0 NaN is NaN, so in the steps that only some rows see all of, values that
//    are not finite (the e4m3 code NaN, or any under such a scale) are left out, and a pass behind the loop, which ordinary
//    data never takes, gives them to the rows that see them.
//  * Both contractions may permute their index, so a thread takes 16 consecutive bytes of a row and no fragment
//    needs a shuffle or a transposing load: key step s of lane l holds dims 32 (l % 4) + 4 s .. and the same of q;
//    value lane l holds dims 16 (l / 4) .. of the four tokens whose weights it owns (after one 8 x 8 transpose).
//  * 16 tokens of k or v of a head are 2 KB in a row, one TMA copy; every warp has a ring of three such pairs of its
//    own.  (16-byte cp.async into the same ring stopped at 4.6 TB/s with nothing saturated; two stages and three CTAs
//    an SM instead of two were slower, 150 us where this takes 95.)
//  * Tokens are cut evenly over the CTAs whatever the lengths: all (sequence, head, row tile) segments in 32-token
//    blocks on one line, an equal stretch of it per CTA. A stretch's first and last segment may continue in a
//    neighbour; those pieces go to the workspace, and a second launch joins them.
// 8 kv heads, e4m3: 64 x 4096 tokens with 4 rows a head 95 us (5.65 TB/s); 16 rows (64 x 2048) 78 us and 32 rows 121 us,
// where the products and conversions bound it; 1 x 1000 tokens 9.8 us, most of it the two launches and what a CTA waits
// for in turn.
#include <cuda_fp16.h>

#include "linear.cuh"
#include "prefill_kernels.cuh"
#include "sm100.cuh"

namespace gdn {

namespace att {
constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kBlock = 32;                       // tokens of the unit that is divided over the CTAs
constexpr int kStages = 3;
constexpr int kStageBytes = 4096;                // a warp's 16 tokens of k and of v, rows of 128 bytes, SWIZZLE_128B
// Places of a segment on the line besides its blocks (40 of 100 to 30000 tokens, 32 rows: 60 us, with 12 places 68, with 24
// 57; 128 of 17 to 4000, 4 rows: 60, with 4 places 86, with 24 67).  The blocks up to which one is not cut (64 of 50 to 2000
// tokens, 16 rows: 42 us, with 16 blocks 44), or if none is longer (8 and 32 x 512 tokens: 11.5 and 15 us, cut 14.5 and 18).
constexpr int kOwn = 16, kKeep = 8, kWhole = 16;
constexpr int kTooLong = 1, kNoPage = 2, kLate = 4;  // what a CTA has met; the gravest of all CTAs' becomes the call's status
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 4.f;                    // scores may exceed the reference by this (base 2)
constexpr float kRoom = 16.f;                    // value scales may exceed a row's r times this much
// Shared memory for tiles of 8 NT rows: the ring, whose place the warps' results take; q as B fragments
// [NT][8 steps][32 lanes][8 bytes]; f32 [8 NT] row factors, int [8 NT] positions that the rows see; f32 [kWarps][8 NT]
// references, then sums; the ring's barriers.
template <int NT>
struct Smem {
    static constexpr int kRing = kWarps * kStages * kStageBytes, kJoin = kWarps * 8 * NT * 128 * 4;
    static constexpr int kOffQ = kRing > kJoin ? kRing : kJoin, kOffF = kOffQ + NT * 2048, kOffM = kOffF + NT * 64;
    static constexpr int kOffBar = kOffM + 2 * kWarps * 8 * NT * 4, kSize = kOffBar + kWarps * kStages * 8;
};
}  // namespace att

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
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
template <bool kInt8>
__device__ __forceinline__ uint4 load_codes(const unsigned char* p) {
    uint4 x = *reinterpret_cast<const uint4*>(p);
    if (kInt8) x = make_uint4(x.x ^ 0x80808080u, x.y ^ 0x80808080u, x.z ^ 0x80808080u, x.w ^ 0x80808080u);
    return x;
}
// 1 / x for a power of two.
__device__ __forceinline__ float power2(float x) { return __uint_as_float(0x7f000000u - __float_as_uint(x)); }
// Bytes of w that are the e4m3 code NaN, as 0xff.
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu); }
__device__ __forceinline__ uint32_t word(const uint4& x, int e) { return e == 0 ? x.x : e == 1 ? x.y : e == 2 ? x.z : x.w; }

__device__ __forceinline__ int visible_length(const CacheArgs& c, int b) {
    return (int)min((long long)cache_length(c, b), (long long)c.max_pages << c.page_shift);
}
__device__ __forceinline__ int seq_blocks(const CacheArgs& c, int b) {
    return max(1, (visible_length(c, b) + att::kBlock - 1) / att::kBlock);
}

// The line of segments: each has its blocks and kOwn places more, for what a piece costs before and after its tokens
// (the q fragments, the first pages, the warps' join).  A CTA's stretch goes from one mark to another.  (Places are
// ints: the entry point refuses more.)
struct AttMark {
    int b, seg, block, before;  // block of segment `seg` of sequence b; places in front of the sequence
};
struct Stretch {
    AttMark at, end;
    int total, ctas;
};
// By one warp, every lane with an equal part of the sequences.
__device__ __forceinline__ void find_stretch(const CacheArgs& c, int segs, Stretch* out) {
    using namespace att;
    const int lane = threadIdx.x & 31, part = (c.B + 31) / 32, b0 = min(c.B, lane * part), b1 = min(c.B, b0 + part);
    int mine = 0, longest = 0;
#pragma unroll 4
    for (int b = b0; b < b1; ++b) {
        const int nb = seq_blocks(c, b);
        mine += nb + kOwn;
        longest = max(longest, nb);
    }
    const int keep = __reduce_max_sync(0xffffffffu, longest) <= kWhole ? kWhole : kKeep;
    int x = mine;
#pragma unroll 1
    for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, off);
        if (lane >= off) x += y;
    }
    const int total = __shfl_sync(0xffffffffu, x, 31) * segs;
    // Stretches of 24 places at least, or of 8 while there are at most 64: 1 x 1000 tokens 9.8 us, with 24 there too 13.0.
    const int ctas = max(1, min((int)gridDim.x, max(total / 24, min(total / 8, 64)))), per = total / ctas, more = total - per * ctas;
    if (lane == 0) {
        out->total = total;
        out->ctas = ctas;
    }
    const int first = (x - mine) * segs;
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
        const int k = blockIdx.x + i, want = min(total, k * per + min(k, more));
        AttMark* m = i ? &out->end : &out->at;
        if (lane == 0 && want == total) *m = AttMark{c.B, 0, 0, total};
        int lo = first;
        if (want < lo || want >= lo + mine * segs) continue;
        int b = b0, w = seq_blocks(c, b) + kOwn;
        while (want >= lo + w * segs) {
            lo += w * segs;
            w = seq_blocks(c, ++b) + kOwn;
        }
        AttMark r{b, (want - lo) / w, 0, lo};
        const int place = want - lo - r.seg * w - kOwn;
        if (w - kOwn > keep) {
            r.block = max(0, place);
        } else if (2 * place >= w - kOwn && ++r.seg == segs) {  // a short segment is not cut: to its nearer end
            r = AttMark{b + 1, 0, 0, lo + w * segs};
        }
        *m = r;
    }
}
// The CTA whose stretch holds place x.
__device__ __forceinline__ int cta_of(int x, int total, int ctas) {
    const int per = total / ctas, more = total - per * ctas, big = more * (per + 1);
    return x < big ? x / (per + 1) : more + (x - big) / per;
}

struct AttendMaps {
    CUtensorMap k, v;  // (128 bytes, rows of all pages) u8, box 128 x 16, SWIZZLE_128B
};

template <bool kInt8, int NT>
__global__ void __launch_bounds__(att::kThreads, NT < 4 ? 2 : 1)
    gdn_cache_attend_kernel(CacheAttendArgs p, const __grid_constant__ AttendMaps maps) {
    using namespace att;
    using S = Smem<NT>;
    constexpr int kRows = 8 * NT;
    extern __shared__ __align__(1024) unsigned char att_sm[];
    __shared__ Stretch s_line;
    __shared__ int s_status;
    const CacheArgs& c = p.c;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    float* s_f = reinterpret_cast<float*>(att_sm + S::kOffF);
    int* s_lim = reinterpret_cast<int*>(s_f + kRows);
    float* s_m = reinterpret_cast<float*>(att_sm + S::kOffM);
    float* s_l = s_m + kWarps * kRows;
    if (tid == 0) s_status = (smem_u32(att_sm) & 1023u) ? kLate : 0;  // (the swizzled tiles need the alignment)
    uint64_t* bars = reinterpret_cast<uint64_t*>(att_sm + S::kOffBar) + warp * kStages;
    if (lane == 0) {
        for (int i = 0; i < kStages; ++i) mbar_init(bars + i, 1);
        mbar_fence_init();
    }
    pdl_wait();
    pdl_trigger();

    const int G = p.Hq / c.Hkv, R = p.Q * G, tiles = (R + kRows - 1) / kRows, segs = c.Hkv * tiles;
    if (warp == 0) find_stretch(c, segs, &s_line);
    __syncthreads();
    const Stretch line = s_line;
    int2 piece = make_int2(-1, 0);  // the segment that begins here and ends elsewhere (thread 0)
    int place = 0;                  // ring place of the next step to read
    uint32_t phases = 0;            // and the phases of the ring's barriers; above them kGaveUp
    constexpr uint32_t kGaveUp = 1u << 31;  // a wait did: the warp takes no more steps

#pragma unroll 1
    for (AttMark at = line.at; at.b < line.end.b || (at.b == line.end.b && (at.seg < line.end.seg || (at.seg == line.end.seg && at.block < line.end.block)));) {
        const int b = at.b, seg = at.seg, h = seg / tiles, row0 = (seg - h * tiles) * kRows;
        const int len = visible_length(c, b), nb = max(1, (len + kBlock - 1) / kBlock);
        const int stop = b == line.end.b && seg == line.end.seg ? line.end.block : nb;
        if (tid == 0 && cache_length(c, b) > len) atomicOr(&s_status, kTooLong);
        const int tok0 = at.block * kBlock, tok1 = min(len, stop * kBlock);
        const int steps = tok1 > tok0 ? (tok1 - tok0 + 15) / 16 : 0;

        unsigned char* ring = att_sm + warp * kStages * kStageBytes;
        const int mine = steps > warp && !(phases & kGaveUp) ? (steps - warp + kWarps - 1) / kWarps : 0;  // steps warp, warp + 8, ..
        const int* trow = c.table + (size_t)b * c.max_pages;
        const int t_first = tok0 + 16 * warp;
        auto page_of = [&](int n) { return n < mine ? trow[(t_first + 16 * kWarps * n) >> c.page_shift] : 0; };
        auto issue = [&](int n, int at_, int page) {
            if (n < mine && lane == 0) {
                uint64_t* bar = bars + at_;
                if ((unsigned)page < (unsigned)c.pages) {
                    const int y = ((page * c.Hkv + h) << c.page_shift) + ((t_first + 16 * kWarps * n) & ((1 << c.page_shift) - 1));
                    mbar_arrive_expect_tx(bar, kStageBytes);
                    tma_load_2d(ring + at_ * kStageBytes, &maps.k, 0, y, bar);
                    tma_load_2d(ring + at_ * kStageBytes + 2048, &maps.v, 0, y, bar);
                } else {
                    mbar_arrive(bar);  // no such page: its tokens are hidden
                }
            }
        };
        auto after = [](int at_) { return at_ + 1 == kStages ? 0 : at_ + 1; };
        int pg0 = page_of(0), pg1 = page_of(1), pg2 = page_of(2);  // pages of the steps in the ring
        issue(0, place, pg0);
        issue(1, after(place), pg1);
        issue(2, after(after(place)), pg2);
        int pg3 = page_of(3);
        auto scale_at = [&](int page) { return (size_t)((unsigned)page < (unsigned)c.pages ? page : 0) * c.Hkv + h; };
        float ks = 0.f, vs = 0.f;
        if (mine > 0) {
            ks = c.k_scale[scale_at(pg0)];
            vs = c.v_scale[scale_at(pg0)];
        }

        // q rows as fp16 fragments; 16 threads a row
#pragma unroll 1
        for (int r = tid >> 4; r < kRows; r += kThreads / 16) {
            const int x = tid & 15, row = row0 + r, i = row / G;
            uint4 w = make_uint4(0, 0, 0, 0);
            if (row < R) w = *reinterpret_cast<const uint4*>(p.q + (((size_t)b * p.Q + i) * p.Hq + h * G + row - i * G) * kD + 8 * x);
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
            if (x == 0) {
                s_f[r] = __uint_as_float((uint32_t)ex << 23) * (p.scale * kLog2e);
                s_lim[r] = len - p.Q + 1 + i;
            }
            // dims 8 x .. 8 x + 7: lane x / 4, whose 32 dims are steps 0-7 four by four
            const int xl = x >> 2, s0 = 2 * (x & 3);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const __half2 lo = __floats2half2_rn(f[4 * e] * inv, f[4 * e + 1] * inv);
                const __half2 hi = __floats2half2_rn(f[4 * e + 2] * inv, f[4 * e + 3] * inv);
                *reinterpret_cast<uint2*>(att_sm + S::kOffQ + (r >> 3) * 2048 + (s0 + e) * 256 + ((r & 7) * 4 + xl) * 8) =
                    make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
            }
        }
        __syncthreads();

        // this thread's q rows of column tile j: row0 + 8 j + 2 (lane % 4) and the next
        float acc[NT][8][4], m[NT][2], l[NT][2], rf[NT][2];
        float inv[NT][2], vmax = 0.f;  // 1 / r; the largest value scale that none of these r has to move for
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int d = 0; d < 8; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[j][d][e] = 0.f;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = 8 * j + 2 * (lane & 3) + r;
                m[j][r] = -INFINITY;
                l[j][r] = 0.f;
                rf[j][r] = s_f[row];
                inv[j][r] = 0x1p120f;
            }
        }
        const int all_see = len - p.Q + 1 + row0 / G;  // positions that every row of the tile sees
        uint2 qf[NT == 1 ? 8 : 1];
        if (NT == 1) {
#pragma unroll
            for (int e = 0; e < 8; ++e) qf[NT == 1 ? e : 0] = *reinterpret_cast<const uint2*>(att_sm + S::kOffQ + e * 256 + lane * 8);
        }

        // scores of a step, still without their factors: tokens lane / 4 and + 8, rows 2 (lane % 4) and the next ([token + 8][row])
        const uint32_t k_off = (lane >> 2) * 128 + (((2 * (lane & 3)) ^ (lane >> 2)) << 4);
        const uint32_t v_off = 2048 + (2 * (lane & 3)) * 128 + (((lane >> 2) ^ (2 * (lane & 3))) << 4);
        auto scores = [&](const unsigned char* st, float (&s)[NT][4]) {
            float s2[NT][4];
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[j][e] = s2[j][e] = 0.f;
#pragma unroll
            for (int half = 0; half < 2; ++half) {  // 16-byte chunk 2 (lane % 4) + half of the tokens lane / 4 and + 8
                const uint4 k0 = load_codes<kInt8>(st + (k_off ^ (half << 4))), k1 = load_codes<kInt8>(st + 1024 + (k_off ^ (half << 4)));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t w0 = word(k0, e), w1 = word(k1, e);
                    const uint32_t a[4] = {codes_f16<kInt8, false>(w0), codes_f16<kInt8, false>(w1), codes_f16<kInt8, true>(w0), codes_f16<kInt8, true>(w1)};
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        const uint2 q = NT == 1 ? qf[NT == 1 ? 4 * half + e : 0]
                                                : *reinterpret_cast<const uint2*>(att_sm + S::kOffQ + j * 2048 + (4 * half + e) * 256 + lane * 8);
                        mma_f16(half ? s2[j] : s[j], a, q.x, q.y);
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[j][e] += s2[j][e];
        };
        // The scores of a step are formed beside the softmax and the second product of the one before: a warp has two
        // chains to work on.  (Those behind the last step are formed from whatever the ring holds, and not used.)
        auto arrived = [&](int at_) {
            if (!mbar_wait(bars + at_, (phases >> at_) & 1u, nullptr, 0)) vmax = -1.f;  // below every scale: seen at the next step
            phases ^= 1u << at_;
        };
        float s[NT][4];
        bool odd = false;  // values that are not finite were left out where not every row sees them
        if (mine > 0) arrived(place);
        scores(ring + place * kStageBytes, s);
#pragma unroll 1
        for (int n = 0; n < mine; ++n) {
            const bool ok = (unsigned)pg0 < (unsigned)c.pages;
            if (!ok) atomicOr(&s_status, kNoPage);
            const int t = t_first + 16 * kWarps * n;
            const bool some = t + 16 > all_see;  // not every row sees all of it
            const float ks0 = ks;
            float vs0 = ok ? vs : 0.f;
            pg0 = pg1;
            pg1 = pg2;
            pg2 = pg3;
            if (n + 1 < mine) {
                ks = c.k_scale[scale_at(pg0)];
                vs = c.v_scale[scale_at(pg0)];
            }
            // scores in base 2; hidden ones are -infinity
            bool over = false;
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[j][e] *= ks0 * rf[j][e & 1];
            if (some || !ok) {
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!ok || t + (lane >> 2) + 8 * (e >> 1) >= s_lim[8 * j + 2 * (lane & 3) + (e & 1)]) s[j][e] = -INFINITY;
                if (!(vs0 < INFINITY)) {
                    vs0 = 0.f;
                    odd = true;
                }
            }
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) over |= s[j][e] > m[j][e & 1] + kSlack;
            if (__any_sync(0xffffffffu, over || vs0 > vmax)) {
                if (__any_sync(0xffffffffu, vmax < 0.f)) {
                    phases |= kGaveUp;
                    atomicOr(&s_status, kLate);
                    for (int i = 1; i < kStages && n + i < mine; ++i) {  // let the other copies land (bounded)
                        const int at_ = (place + i) % kStages;
                        mbar_wait(bars + at_, (phases >> at_) & 1u, nullptr, 0);
                    }
                    break;
                }
                vmax = INFINITY;
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        float here = fmaxf(s[j][r], s[j][2 + r]);  // the step's maximum
                        here = fmaxf(here, __shfl_xor_sync(0xffffffffu, here, 4));
                        here = fmaxf(here, __shfl_xor_sync(0xffffffffu, here, 8));
                        here = fmaxf(here, __shfl_xor_sync(0xffffffffu, here, 16));
                        const float top = fmaxf(here, m[j][r]);
                        const float f = m[j][r] == -INFINITY ? 0.f : ex2(m[j][r] - top);
                        m[j][r] = top;
                        l[j][r] *= f;
                        // r follows the maximum, or the step's largest weight (kept within what r and 1 / r can both hold)
                        const float old = f * power2(inv[j][r]), now = here == -INFINITY ? 0.f : ex2(here - top) * vs0;
                        const int ex = min(max((int)(__float_as_uint(fmaxf(old, now)) >> 23), 7), 247);
                        inv[j][r] = __uint_as_float((uint32_t)(254 - ex) << 23);
                        vmax = fminf(vmax, kRoom * __uint_as_float((uint32_t)ex << 23));
#pragma unroll
                        for (int d = 0; d < 8; ++d) {
                            acc[j][d][r] *= old * inv[j][r];
                            acc[j][d][2 + r] *= old * inv[j][r];
                        }
                    }
            }
            const int next = after(place);
            if (n + 1 < mine) arrived(next);
            float sn[NT][4];
            scores(ring + next * kStageBytes, sn);
            uint32_t w0[NT], w1[NT];  // weights as B fragments: tokens 2 (lane % 4) + {0, 1} (+ 8), row lane / 4
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                float e[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    e[i] = ex2(s[j][i] - (m[j][i & 1] == -INFINITY ? 0.f : m[j][i & 1]));
                    l[j][i & 1] += e[i];
                }
                const float2 in = make_float2(inv[j][0], inv[j][1]), vv = make_float2(vs0, vs0);
                const float2 e0 = mul2(mul2(make_float2(e[0], e[1]), vv), in), e1 = mul2(mul2(make_float2(e[2], e[3]), vv), in);
                const __half2 x = __floats2half2_rn(e0.x, e0.y), y = __floats2half2_rn(e1.x, e1.y);
                w0[j] = transpose_8x8(*reinterpret_cast<const uint32_t*>(&x));
                w1[j] = transpose_8x8(*reinterpret_cast<const uint32_t*>(&y));
            }
            // tokens 2 (lane % 4) + {0, 1} (+ 8), chunk lane / 4
            auto v_at = [&](int i) { return ring + place * kStageBytes + 1024 * (i >> 1) + ((v_off + 128 * (i & 1)) ^ ((i & 1) << 4)); };
            auto v_token = [&](int i) { return t + 2 * (lane & 3) + (i & 1) + 8 * (i >> 1); };
            uint4 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = load_codes<kInt8>(v_at(i));
            if (!ok || t + 16 > tok1) {  // slots behind the sequence's end hold anything: a weight of 0 does not undo a NaN
                const uint32_t none = kInt8 ? 0x80808080u : 0u;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (!ok || v_token(i) >= tok1) v[i] = make_uint4(none, none, none, none);
            }
            if (!kInt8 && some) {  // nor that of a token that some rows do not see: those that do get it after the loop
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint4 x = make_uint4(nan_codes(v[i].x), nan_codes(v[i].y), nan_codes(v[i].z), nan_codes(v[i].w));
                    v[i] = make_uint4(v[i].x & ~x.x, v[i].y & ~x.y, v[i].z & ~x.z, v[i].w & ~x.w);
                    odd |= (x.x | x.y | x.z | x.w) != 0;
                }
            }
            __syncwarp();  // the step's place is read: the next one may land there
            issue(n + 3, place, pg2);
            pg3 = page_of(n + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int d = 0; d < 2; ++d) {  // dims 16 (lane / 4) + 4 e + 2 d and the next: rows lane / 4 and + 8 of the tile
                    const uint32_t x = __byte_perm(word(v[0], e), word(v[1], e), d ? 0x7362 : 0x5140);
                    const uint32_t y = __byte_perm(word(v[2], e), word(v[3], e), d ? 0x7362 : 0x5140);
                    const uint32_t a[4] = {codes_f16<kInt8, false>(x), codes_f16<kInt8, true>(x), codes_f16<kInt8, false>(y), codes_f16<kInt8, true>(y)};
#pragma unroll
                    for (int j = 0; j < NT; ++j) mma_f16(acc[j][2 * e + d], a, w0[j], w1[j]);
                }
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[j][e] = sn[j][e];
            place = next;
        }

        if (__any_sync(0xffffffffu, odd)) {
            // A product of ones, in the places of those values and of the tokens that a row sees, finds the sums that become NaN.
#pragma unroll 1
            for (int n = 0; n < mine; ++n) {
                const int t = t_first + 16 * kWarps * n, page = page_of(n);
                if (t + 16 <= all_see || (unsigned)page >= (unsigned)c.pages) continue;
                const bool all = !(c.v_scale[scale_at(page)] < INFINITY);
                const uint32_t one = kInt8 ? 0x81818181u : 0x38383838u, none = kInt8 ? 0x80808080u : 0u;
                uint4 v[4];  // the value's place, as in the loop above: one
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int tok = t + 2 * (lane & 3) + (i & 1) + 8 * (i >> 1);
                    uint4 x = make_uint4(0, 0, 0, 0);
                    if (!kInt8)
                        x = *reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(c.v_cache) + 16 * (lane >> 2) +
                                                            128 * ((((size_t)page * c.Hkv + h) << c.page_shift) + (tok & ((1 << c.page_shift) - 1))));
                    auto mark = [&](uint32_t w) { return all ? one : kInt8 ? none : one & nan_codes(w); };
                    v[i] = make_uint4(mark(x.x), mark(x.y), mark(x.z), mark(x.w));
                }
                uint32_t w0[NT], w1[NT];
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    float e[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) e[i] = t + (lane >> 2) + 8 * (i >> 1) < s_lim[8 * j + 2 * (lane & 3) + (i & 1)] ? 1.f : 0.f;
                    const __half2 x = __floats2half2_rn(e[0], e[1]), y = __floats2half2_rn(e[2], e[3]);
                    w0[j] = transpose_8x8(*reinterpret_cast<const uint32_t*>(&x));
                    w1[j] = transpose_8x8(*reinterpret_cast<const uint32_t*>(&y));
                }
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int d = 0; d < 2; ++d) {
                        const uint32_t x = __byte_perm(word(v[0], e), word(v[1], e), d ? 0x7362 : 0x5140);
                        const uint32_t y = __byte_perm(word(v[2], e), word(v[3], e), d ? 0x7362 : 0x5140);
                        const uint32_t a[4] = {codes_f16<kInt8, false>(x), codes_f16<kInt8, true>(x), codes_f16<kInt8, false>(y), codes_f16<kInt8, true>(y)};
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            float hit[4] = {0.f, 0.f, 0.f, 0.f};
                            mma_f16(hit, a, w0[j], w1[j]);
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (hit[i] > 0.f) acc[j][2 * e + d][i] = NAN;
                        }
                    }
            }
        }

        // join the warps: every warp's result at the common maximum
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) l[j][r] += __shfl_xor_sync(0xffffffffu, l[j][r], off);
                if (lane < 4) {
                    s_m[warp * kRows + 8 * j + 2 * lane + r] = m[j][r];
                    s_l[warp * kRows + 8 * j + 2 * lane + r] = l[j][r];
                }
            }
        __syncthreads();  // also: every warp is done with its ring
        float* wacc = reinterpret_cast<float*>(att_sm);  // [kWarps][kRows][128], 16-byte chunks XORed with the row
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = 8 * j + 2 * (lane & 3) + r;
                float mall = -INFINITY;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) mall = fmaxf(mall, s_m[w * kRows + row]);
                const float f = l[j][r] != 0.f ? ex2(m[j][r] - mall) * power2(inv[j][r]) : 0.f;  // a NaN stays one
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    *reinterpret_cast<float4*>(wacc + (warp * kRows + row) * 128 + ((4 * (lane >> 2) + e) ^ (row & 7)) * 4) =
                        make_float4(acc[j][2 * e][r] * f, acc[j][2 * e][2 + r] * f, acc[j][2 * e + 1][r] * f, acc[j][2 * e + 1][2 + r] * f);
            }
        __syncthreads();
        const bool begins = at.block == 0, whole = begins && stop == nb;
#pragma unroll 1
        for (int row = tid >> 5; row < min(kRows, R - row0); row += kThreads / 32) {  // a warp a row, four dims a lane
            float mm = -INFINITY, ll = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, s_m[w * kRows + row]);
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float lw = s_l[w * kRows + row];
                if (lw != 0.f) ll += lw * ex2(s_m[w * kRows + row] - mm);
                const float4 x = *reinterpret_cast<const float4*>(wacc + (w * kRows + row) * 128 + (lane ^ (row & 7)) * 4);
                o = make_float4(o.x + x.x, o.y + x.y, o.z + x.z, o.w + x.w);
            }
            if (whole) {
                const int r = row0 + row, i = r / G;
                const float inv = ll > 0.f || ll != ll ? 1.f / ll : 0.f;
                *reinterpret_cast<uint2*>(p.out + (((size_t)b * p.Q + i) * p.Hq + h * G + r - i * G) * kD + 4 * lane) =
                    make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
            } else {
                const size_t slot = (2 * (size_t)blockIdx.x + (begins ? 1 : 0)) * kRows + row;
                *reinterpret_cast<float4*>(p.acc + slot * 128 + 4 * lane) = o;
                if (lane == 0) *reinterpret_cast<float2*>(p.ml + slot * 2) = make_float2(mm, ll);
            }
        }
        if (!whole && begins)  // the pieces that follow
            piece = make_int2(b * segs + seg, cta_of(at.before + seg * (nb + kOwn) + kOwn + nb - 1, line.total, line.ctas) - (int)blockIdx.x);
        fence_async_smem();  // what was written in the ring's place comes before the next copies
        at.block = 0;
        if (++at.seg == segs) {
            at.seg = 0;
            at.before += (nb + kOwn) * segs;
            ++at.b;
        }
        __syncthreads();
    }
    if (tid == 0) p.piece[blockIdx.x] = make_int4(piece.x, piece.y, s_status, 0);
}

// Joins a segment that several CTAs of the line hold: CTA x takes the one that CTA x began, row y of its tile.
__global__ void __launch_bounds__(128) gdn_cache_join_kernel(CacheAttendArgs p, int rows) {
    __shared__ float4 s_o[4][32];
    __shared__ float s_l[4];
    pdl_wait();
    pdl_trigger();
    if (blockIdx.x == 0 && blockIdx.y == 0) {  // the call's status: any of the CTAs'
        int met = 0;
        for (int i = threadIdx.x; i < (int)gridDim.x; i += 128) met |= p.piece[i].z;
        const bool late = __syncthreads_or(met & att::kLate), page = __syncthreads_or(met & att::kNoPage);
        const bool length = __syncthreads_or(met & att::kTooLong);
        if (threadIdx.x == 0) *p.status = late ? kErrScanTmaTimeout : page ? kErrBadPage : length ? kErrBadSeqlens : 0;
    }
    const int4 pc = p.piece[blockIdx.x];
    if (pc.x < 0) return;
    const int G = p.Hq / p.c.Hkv, R = p.Q * G, tiles = (R + rows - 1) / rows, segs = p.c.Hkv * tiles;
    const int b = pc.x / segs, seg = pc.x % segs, h = seg / tiles, r = (seg % tiles) * rows + blockIdx.y;
    if (r >= R) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto slot = [&](int i) { return ((size_t)(2 * (blockIdx.x + i) + (i == 0 ? 1 : 0))) * rows + blockIdx.y; };
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

template <bool kInt8, int NT>
static int launch_attend(const CacheAttendArgs& p, cudaStream_t stream) {
    constexpr int kRows = 8 * NT, kSmem = att::Smem<NT>::kSize;
    const unsigned ctas = NT < 4 ? kAttendCtas : kAttendCtas / 2;  // what fits on the SMs together
    static SmemLimit limit;
    if (!limit.raise(gdn_cache_attend_kernel<kInt8, NT>, kSmem)) return -1;
    AttendMaps maps{};
    if (p.c.max_pages > 0) {
        const uint64_t rows = ((uint64_t)p.c.pages * p.c.Hkv) << p.c.page_shift;
        if (!map_u8_rows(&maps.k, p.c.k_cache, rows) || !map_u8_rows(&maps.v, p.c.v_cache, rows)) return -3;
    }
    if (launch_pdl(gdn_cache_attend_kernel<kInt8, NT>, dim3(ctas), dim3(att::kThreads), kSmem, stream, p, maps) != cudaSuccess) return -1;
    const int rows = p.Q * (p.Hq / p.c.Hkv);
    return launch_pdl(gdn_cache_join_kernel, dim3(ctas, (unsigned)(rows < kRows ? rows : kRows)), dim3(128), 0, stream, p, kRows) == cudaSuccess ? 0 : -1;
}

// Column tiles of 8 rows: as many as a kv head's q rows need, at most 4 (the accumulators fill the registers).  64 x 2048
// tokens with 16 rows: 100 us in tiles of 8, 78 of 16, 112 of 32; with 32 rows 182 of 8, 121 of 32; 64 x 4096 with 4 rows
// 95 of 8, 185 of 32.
int attend_tiles(int rows) { return rows <= 8 ? 1 : rows <= 16 ? 2 : 4; }

int launch_cache_attend(const CacheAttendArgs& p, cudaStream_t stream) {
    const int nt = attend_tiles(p.Q * (p.Hq / p.c.Hkv));
    if (p.c.int8) return nt == 1 ? launch_attend<true, 1>(p, stream) : nt == 2 ? launch_attend<true, 2>(p, stream) : launch_attend<true, 4>(p, stream);
    return nt == 1 ? launch_attend<false, 1>(p, stream) : nt == 2 ? launch_attend<false, 2>(p, stream) : launch_attend<false, 4>(p, stream);
}

}  // namespace gdn
