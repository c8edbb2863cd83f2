// linear_prefill.cu -- linear attention with a decay for each head over packed sequences, chunked.
//
// Recurrence per token: S <- e^{a_t} S + v_t k_t^T (S is [V][K], fp32), o_t = scale S q_t.  Over a chunk of
// C = 64 tokens with G_i = a_1 + .. + a_i and the state S_0 at its start:
//   o_i = scale (e^{G_i} S_0 q_i + sum_{j <= i} e^{G_i - G_j} (q_i . k_j) v_j)
//   S_C = e^{G_C} S_0 + sum_j (e^{G_C - G_j} v_j) k_j^T
// All products run on tcgen05 with the V dimension as the M = 128 rows, so no accumulator row is wasted on
// a 64-token chunk:
//   QK  [Q; K] (128 x 128, K-major) x K (64 tokens)            -> rows 0-63: q_i . k_j
//   OI  S_0 (128 V x 128 K, bf16)   x Q (64 tokens)            -> S_0 q_i, scaled by e^{G_i} in the epilogue
//   OA  V^T (128 V x 64 tokens, MN-major from the v tile) x P  -> P = decayed, causal QK in bf16
//   U   Vd^T (128 V x 64 tokens) x K (128 K)                   -> Vd = decayed v as bf16 hi + lo
// The state stays in fp32 registers; hi + lo keeps what a chunk adds to it at 2^-17 relative.
//
// The update does not read the state, so a long sequence is cut into segments of m chunks: a first launch
// builds what every segment but the last adds to the state (U alone), a second one chains the segments, and
// the output launch runs all segments side by side.
#include <algorithm>

#include "linear.cuh"
#include "prefill_kernels.cuh"
#include "sm100.cuh"

namespace gdn {

namespace lin {
constexpr int C = 64;
constexpr int kThreads = 288;  // 8 math warps + 1 TMA warp
constexpr int kMath = 256;
constexpr int kStages = 2;
// stage: [Q0 | K0 | Q1 | K1 | V0 | V1], each 64 tokens x 64 columns bf16, SWIZZLE_128B
constexpr uint32_t kOffQ = 0, kOffK = 8192, kAtom = 16384, kOffV = 32768;
constexpr uint32_t kStage = 49152;
constexpr uint32_t kOffS = kStages * kStage;     // bf16 state [128 V][128 K]: two 64-column atoms of 16 KB
constexpr uint32_t kOffVh = kOffS + 32768;       // decayed v, hi then lo: two atoms of 64 tokens x 128 B each
constexpr uint32_t kOffVl = kOffVh + 16384;
constexpr uint32_t kOffP = kOffVl + 16384;       // P [64 i][64 j] bf16
constexpr uint32_t kOffO = kOffP + 8192;         // output staging [64 tokens][128 V] bf16, 16-byte chunks swizzled
constexpr uint32_t kOffG = kOffO + 16384;        // f32 [64] G log2(e) | [64] e^G | [64] e^{G_C - G} | e^{G_C}
constexpr uint32_t kOffBar = kOffG + 1024;
constexpr uint32_t kSmem = kOffBar + 128 + 1024;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColP = 0, kColI = 64, kColA = 128, kColU = 192;
static_assert(kSmem <= 227 * 1024, "shared memory");

constexpr float kLog2e = 1.4426950408889634f;
// Log decays are clamped here: e^-110 is below every fp32 number, and -infinity would turn the differences
// of prefix sums into NaN.
constexpr float kMinDecay = -110.f;
}  // namespace lin

struct LinearMaps {
    CUtensorMap q, k, v;  // (128, heads, T) bf16, box 64 x 1 x 64, SWIZZLE_128B
};

// Work items: sequence n owns the slots from cu[n] / len + n on (len = 64 m tokens), at least as many as it has
// segments, and one if it is empty.  What its segments add to the state lies in the state slots from
// 2 (cu[n] / len) on: a sequence of more than one segment has at most 2 floor(tokens / len) of them.  Neither needs
// a prefix sum over the sequences, only a search for the owner.
__device__ __forceinline__ int seq_start(const LinearPrefillArgs& p, int n) {
    int s, e;
    seq_bounds(p.cu, p.cu64, n, p.T, s, e);
    return s;
}
struct SegItem {
    int n, seg, nsegs, t0, t1, state0;  // tokens [t0, t1) of segment `seg` of sequence n (n < 0: none); its first state slot
};
__device__ __forceinline__ SegItem find_segment(const LinearPrefillArgs& p, int slot, int per_seq, int per_len) {
    const int len = lin::C * p.m;
    int lo = 0, hi = p.N - 1;  // the last sequence whose first slot, per_len (cu[n] / len) + per_seq n, is <= slot
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (per_len * (seq_start(p, mid) / len) + per_seq * mid <= slot) lo = mid;
        else hi = mid - 1;
    }
    SegItem it;
    int s, e;
    seq_bounds(p.cu, p.cu64, lo, p.T, s, e);
    it.nsegs = max(1, (e - s + len - 1) / len);
    it.seg = slot - (per_len * (s / len) + per_seq * lo);
    it.n = (it.seg >= 0 && it.seg < it.nsegs) ? lo : -1;  // also where cu_seqlens is not non-decreasing
    it.t0 = s + it.seg * len;
    it.t1 = min(e, it.t0 + len);
    it.state0 = 2 * (s / len);
    return it;
}

__device__ __forceinline__ void zero_rows(const LinearPrefillArgs& p, int tid, int nthreads) {
    int lo, tmp, hi;
    seq_bounds(p.cu, p.cu64, 0, p.T, lo, tmp);
    seq_bounds(p.cu, p.cu64, p.N - 1, p.T, tmp, hi);
    hi = max(hi, lo);
    const size_t row_words = (size_t)p.HV * kD / 8;
    uint4* o4 = reinterpret_cast<uint4*>(p.out);
    for (size_t i = tid; i < (size_t)lo * row_words; i += nthreads) o4[i] = make_uint4(0, 0, 0, 0);
    for (size_t i = (size_t)hi * row_words + tid; i < (size_t)p.T * row_words; i += nthreads) o4[i] = make_uint4(0, 0, 0, 0);
}

// kOut: the output launch.  Otherwise the segment launch: what each segment but a sequence's last adds to the state.
template <bool kOut>
__global__ void __launch_bounds__(lin::kThreads, 1)
    gdn_linear_prefill_kernel(LinearPrefillArgs p, const __grid_constant__ LinearMaps maps) {
    using namespace lin;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t sbase = smem_u32(sm);
    uint64_t* full = reinterpret_cast<uint64_t*>(sm + kOffBar);
    uint64_t* empty = full + kStages;
    uint64_t* bar_p = empty + kStages;
    uint64_t* bar_u = bar_p + 1;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(bar_u + 1);
    uint32_t* tslot = reinterpret_cast<uint32_t*>(bar_u + 1) + 1;
    float* sG2 = reinterpret_cast<float*>(sm + kOffG);
    float* sEG = sG2 + 64;
    float* sER = sEG + 64;
    float* sEL = sER + 64;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_wait();
    pdl_trigger();
    if (blockIdx.x == 0) {
        if (tid == 0 && (!kOut || !p.cut)) *p.status = 0;  // the call's first launch
        if (kOut && p.zero_unowned) zero_rows(p, tid, kThreads);
    }
    const int hv = blockIdx.x % p.HV, slot = blockIdx.x / p.HV, hq = hv / (p.HV / p.H);
    const SegItem it = kOut ? find_segment(p, slot, 1, 1) : find_segment(p, slot, 0, 2);
    const bool last = it.seg == it.nsegs - 1;
    if (it.n < 0 || (!kOut && last)) return;

    if (tid == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full + s, 1);
            mbar_init(empty + s, kMath / 32);
        }
        mbar_init(bar_p, 1);
        mbar_init(bar_u, 1);
        *abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 0) tmem_alloc(tslot, kTmemCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tslot;
    const int nchunks = max(0, (it.t1 - it.t0 + C - 1) / C);

    if (warp == kMath / 32) {
        if (lane == 0) {
            for (int c = 0; c < nchunks; ++c) {
                const int s = c % kStages;
                if (c >= kStages && !mbar_wait(empty + s, (uint32_t)((c / kStages - 1) & 1), p.status, kErrScanTmaTimeout)) break;
                unsigned char* st = sm + s * kStage;
                const int t = it.t0 + c * C;
                mbar_arrive_expect_tx(full + s, kOut ? 49152 : 32768);
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    if (kOut) tma_load_3d(st + kOffQ + a * kAtom, &maps.q, 64 * a, hq, t, full + s);
                    tma_load_3d(st + kOffK + a * kAtom, &maps.k, 64 * a, hq, t, full + s);
                    tma_load_3d(st + kOffV + a * 8192, &maps.v, 64 * a, hv, t, full + s);
                }
            }
        }
    } else {
        const int quarter = warp & 3, half = warp >> 2;
        const int r = lane + 32 * quarter;  // TMEM lane: V row of the state, or token of the chunk
        const uint32_t tl = tmem + ((uint32_t)(32 * quarter) << 16);
        float h[64];  // state row r, columns 64 half ..
        {
            const float* src = nullptr;
            if (kOut) {
                if (it.nsegs == 1)
                    src = p.state ? p.state + ((size_t)it.n * p.HV + hv) * kD * kD : nullptr;
                else  // the chain left the states at the segments' ends, and the initial state behind them
                    src = p.seg + ((size_t)(it.state0 + (it.seg == 0 ? it.nsegs - 1 : it.seg - 1)) * p.HV + hv) * kD * kD;
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const float4 x = src ? *reinterpret_cast<const float4*>(src + (size_t)r * kD + 64 * half + 4 * j)
                                     : make_float4(0.f, 0.f, 0.f, 0.f);
                h[4 * j] = x.x;
                h[4 * j + 1] = x.y;
                h[4 * j + 2] = x.z;
                h[4 * j + 3] = x.w;
            }
        }
        // bf16 copy of the state: row r, atom `half`, eight 16-byte chunks XOR-swizzled by the row
        auto write_s = [&]() {
            unsigned char* row = sm + kOffS + half * 16384 + r * 128;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                *reinterpret_cast<uint4*>(row + ((j ^ (r & 7)) << 4)) =
                    make_uint4(pack_bf16x2(h[8 * j], h[8 * j + 1]), pack_bf16x2(h[8 * j + 2], h[8 * j + 3]),
                               pack_bf16x2(h[8 * j + 4], h[8 * j + 5]), pack_bf16x2(h[8 * j + 6], h[8 * j + 7]));
        };
        if (kOut && nchunks > 0) write_s();
        constexpr uint32_t idesc_qk = umma_idesc_bf16(128, 64, false, false);
        constexpr uint32_t idesc_oi = umma_idesc_bf16(128, 64, false, false);
        constexpr uint32_t idesc_oa = umma_idesc_bf16(128, 64, true, false);
        constexpr uint32_t idesc_u = umma_idesc_bf16(128, 128, true, true);
        float gamma = 1.f;  // product of the segment's decays (thread 0 of the segment launch)
        int c = 0;
        for (; c < nchunks; ++c) {
            const int s = c % kStages, t0 = it.t0 + c * C, L = min(C, it.t1 - t0);
            unsigned char* st = sm + s * kStage;
            const uint32_t sst = sbase + (uint32_t)s * kStage;
            if (warp == 0) {
                // prefix and suffix sums of the chunk's log decays, two tokens a lane
                float a0 = 0.f, a1 = 0.f;
                if (2 * lane < L) a0 = p.decay[p.per_token ? (size_t)(t0 + 2 * lane) * p.HV + hv : hv];
                if (2 * lane + 1 < L) a1 = p.decay[p.per_token ? (size_t)(t0 + 2 * lane + 1) * p.HV + hv : hv];
                a0 = a0 < kMinDecay ? kMinDecay : a0;
                a1 = a1 < kMinDecay ? kMinDecay : a1;
                float pre = a0 + a1, suf = a0 + a1;
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) {
                    const float x = __shfl_up_sync(0xffffffffu, pre, off), y = __shfl_down_sync(0xffffffffu, suf, off);
                    if (lane >= off) pre += x;
                    if (lane + off < 32) suf += y;
                }
                float before = __shfl_up_sync(0xffffffffu, pre, 1), after = __shfl_down_sync(0xffffffffu, suf, 1);
                if (lane == 0) before = 0.f;
                if (lane == 31) after = 0.f;
                const float g0 = before + a0, g1 = pre;
                sG2[2 * lane] = g0 * kLog2e;
                sG2[2 * lane + 1] = g1 * kLog2e;
                sEG[2 * lane] = expf(g0);
                sEG[2 * lane + 1] = expf(g1);
                // e^{G_C - G_j} from the sum of the later decays: exact where it matters, near the chunk's end
                sER[2 * lane] = 2 * lane < L ? expf(after + a1) : 0.f;
                sER[2 * lane + 1] = 2 * lane + 1 < L ? expf(after) : 0.f;
                if (lane == 31) *sEL = expf(pre);
            }
            if (!mbar_wait(full + s, (uint32_t)((c / kStages) & 1), p.status, kErrScanTmaTimeout)) *abort_flag = 1;
            fence_async_smem();  // the state copy (generic stores) -> the tensor core
            tc_fence_before();
            named_bar_sync(1, kMath);
            if (*abort_flag) break;
            tc_fence_after();
            const float eL = *sEL;
            if (kOut && tid == 0) {
#pragma unroll
                for (int kk = 0; kk < 8; ++kk)
                    umma_bf16(tmem + kColP, umma_desc_sw128(sst + kOffQ + (uint32_t)(kk >> 2) * kAtom + (uint32_t)(kk & 3) * 32u, 16, 1024),
                              umma_desc_sw128(sst + kOffK + (uint32_t)(kk >> 2) * kAtom + (uint32_t)(kk & 3) * 32u, 16, 1024), idesc_qk, kk > 0);
                umma_commit(bar_p);
#pragma unroll
                for (int kk = 0; kk < 8; ++kk)
                    umma_bf16(tmem + kColI, umma_desc_sw128(sbase + kOffS + (uint32_t)(kk >> 2) * 16384u + (uint32_t)(kk & 3) * 32u, 16, 1024),
                              umma_desc_sw128(sst + kOffQ + (uint32_t)(kk >> 2) * kAtom + (uint32_t)(kk & 3) * 32u, 16, 1024), idesc_oi, kk > 0);
            }
            bool ok = true;
            if (kOut && L < C) ok = mbar_wait(bar_p, (uint32_t)(c & 1), p.status, kErrScanMmaTimeout);
            // Decayed v: thread (token i, 32 columns).  Rows behind the segment's end (another sequence's
            // tokens, or zeros) become zero in v and k too, so whatever they hold cannot reach a product.
            {
                const int i = tid & 63, q4 = tid >> 6;  // columns 32 q4 ..
                const float er = sER[i];
                unsigned char* vt = st + kOffV + (q4 >> 1) * 8192 + i * 128;
                unsigned char* vh = sm + kOffVh + (q4 >> 1) * 8192 + i * 128;
                unsigned char* vl = sm + kOffVl + (q4 >> 1) * 8192 + i * 128;
#pragma unroll
                for (int jj = 0; jj < 4; ++jj) {
                    const uint32_t off = (uint32_t)(((4 * (q4 & 1) + jj) ^ (i & 7)) << 4);
                    uint4 x = *reinterpret_cast<const uint4*>(vt + off);
                    if (i >= L) {
                        x = make_uint4(0, 0, 0, 0);
                        *reinterpret_cast<uint4*>(vt + off) = x;
                        *reinterpret_cast<uint4*>(st + kOffK + (q4 >> 1) * kAtom + i * 128 + off) = x;
                    }
                    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 y = mul2(make_float2(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xffff0000u)), make_float2(er, er));
                        hi[e] = pack_bf16x2(y.x, y.y);
                        const float2 z = sub2(y, make_float2(__uint_as_float(hi[e] << 16), __uint_as_float(hi[e] & 0xffff0000u)));
                        lo[e] = pack_bf16x2(z.x, z.y);
                    }
                    *reinterpret_cast<uint4*>(vh + off) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    *reinterpret_cast<uint4*>(vl + off) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
            }
            if (kOut) {
                if (L == C) ok = mbar_wait(bar_p, (uint32_t)(c & 1), p.status, kErrScanMmaTimeout);
                tc_fence_after();
                if (quarter < 2) {  // P row i = r, columns 32 half ..
                    uint32_t d[32];
                    tmem_ld32_async(tl + kColP + 32 * half, d);
                    tmem_ld_wait();
                    tmem_regs_ready(d);
                    const float gi = sG2[r];
                    unsigned char* row = sm + kOffP + r * 128;
#pragma unroll
                    for (int jj = 0; jj < 4; ++jj) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int j = 32 * half + 8 * jj + 2 * e;
                            const float x = j <= r && j < L ? __uint_as_float(d[8 * jj + 2 * e]) * exp2f(gi - sG2[j]) : 0.f;
                            const float y = j + 1 <= r && j + 1 < L ? __uint_as_float(d[8 * jj + 2 * e + 1]) * exp2f(gi - sG2[j + 1]) : 0.f;
                            w[e] = pack_bf16x2(x, y);
                        }
                        *reinterpret_cast<uint4*>(row + (((4 * half + jj) ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
            fence_async_smem();
            tc_fence_before();
            if (!ok) *abort_flag = 1;
            named_bar_sync(1, kMath);
            tc_fence_after();
            if (*abort_flag) break;
            if (tid == 0) {
                if (kOut) {
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                        umma_bf16(tmem + kColA, umma_desc_sw128(sst + kOffV + 2048u * kk, 8192, 1024),
                                  umma_desc_sw128(sbase + kOffP + 32u * kk, 16, 1024), idesc_oa, kk > 0);
                }
#pragma unroll
                for (int kk = 0; kk < 8; ++kk)
                    umma_bf16(tmem + kColU, umma_desc_sw128(sbase + (kk < 4 ? kOffVh : kOffVl) + 2048u * (kk & 3), 8192, 1024),
                              umma_desc_sw128(sst + kOffK + 2048u * (kk & 3), kAtom, 1024), idesc_u, kk > 0);
                umma_commit(bar_u);
            }
            ok = mbar_wait(bar_u, (uint32_t)(c & 1), p.status, kErrScanMmaTimeout);
            tc_fence_after();
            if (lane == 0) mbar_arrive(empty + s);  // the products of this stage are done
            if (kOut) {
                // output column r, tokens 32 half ..: o = scale (e^{G_i} OI + OA), staged so that rows leave whole
                uint32_t x[32], y[32];
                tmem_ld32_async(tl + kColI + 32 * half, x);
                tmem_ld32_async(tl + kColA + 32 * half, y);
                tmem_ld_wait();
                tmem_regs_ready(x);
                tmem_regs_ready(y);
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    const int i = 32 * half + j;
                    const float o = p.scale * fmaf(sEG[i], __uint_as_float(x[j]), __uint_as_float(y[j]));
                    *reinterpret_cast<uint16_t*>(sm + kOffO + i * 256 + (((r >> 3) ^ (i & 7)) << 4) + (r & 7) * 2) = f2bf(o);
                }
            }
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                uint32_t d[32];
                tmem_ld32_async(tl + kColU + 64 * half + 32 * b, d);
                tmem_ld_wait();
                tmem_regs_ready(d);
#pragma unroll
                for (int j = 0; j < 32; ++j) h[32 * b + j] = fmaf(eL, h[32 * b + j], __uint_as_float(d[j]));
            }
            gamma *= eL;
            if (!ok) *abort_flag = 1;
            if (kOut) {
                write_s();
                named_bar_sync(1, kMath);  // the staged output rows
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int i = 16 * q + (tid >> 4), ch = tid & 15;
                    if (i < L)
                        *reinterpret_cast<uint4*>(p.out + ((size_t)(t0 + i) * p.HV + hv) * kD + 8 * ch) =
                            *reinterpret_cast<const uint4*>(sm + kOffO + i * 256 + ((ch ^ (i & 7)) << 4));
                }
            } else {
                named_bar_sync(1, kMath);  // the chunk's decays are consumed
            }
        }
        if (c < nchunks) {
            // gave up: let copies already in flight land (bounded) before the CTA exits
            if (tid == 0)
                for (int cc = c; cc < min(nchunks, c + kStages); ++cc)
                    mbar_wait(full + cc % kStages, (uint32_t)((cc / kStages) & 1), nullptr, 0);
        } else if (!kOut || last) {
            float* dst = kOut ? p.new_state + ((size_t)it.n * p.HV + hv) * kD * kD : p.seg + ((size_t)slot * p.HV + hv) * kD * kD;
#pragma unroll
            for (int j = 0; j < 16; ++j)
                *reinterpret_cast<float4*>(dst + (size_t)r * kD + 64 * half + 4 * j) =
                    make_float4(h[4 * j], h[4 * j + 1], h[4 * j + 2], h[4 * j + 3]);
            if (!kOut && tid == 0) p.gamma[(size_t)slot * p.HV + hv] = gamma;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem, kTmemCols);
}

// State at the end of every segment but a sequence's last, in place of what the segment adds, and the initial state
// in the slot behind them: new_state may be state itself, and a last segment may end before a first one begins.
// One CTA per (1024 state elements, v-head, start of a possible sequence of several segments).
__global__ void __launch_bounds__(256) gdn_linear_chain_kernel(LinearPrefillArgs p) {
    pdl_wait();
    pdl_trigger();
    const int hv = blockIdx.x % p.HV;
    const SegItem it = find_segment(p, 2 * (blockIdx.x / p.HV), 0, 2);
    if (it.n < 0 || it.seg != 0 || it.nsegs == 1) return;
    const size_t el = blockIdx.y * 1024 + threadIdx.x * 4;
    float4 h = make_float4(0.f, 0.f, 0.f, 0.f);
    if (p.state) h = *reinterpret_cast<const float4*>(p.state + ((size_t)it.n * p.HV + hv) * kD * kD + el);
    *reinterpret_cast<float4*>(p.seg + ((size_t)(it.state0 + it.nsegs - 1) * p.HV + hv) * kD * kD + el) = h;
#pragma unroll 4
    for (int g = 0; g < it.nsegs - 1; ++g) {
        const size_t at = (size_t)(it.state0 + g) * p.HV + hv;
        const float gm = p.gamma[at];
        float4* d = reinterpret_cast<float4*>(p.seg + at * kD * kD + el);
        const float4 x = *d;
        h = make_float4(fmaf(gm, h.x, x.x), fmaf(gm, h.y, x.y), fmaf(gm, h.z, x.z), fmaf(gm, h.w, x.w));
        *d = h;
    }
}

LinearPrefillLayout linear_prefill_layout(int N, int T, int HV) {
    LinearPrefillLayout L{};
    // Chunks per segment: as many as one of 148 SMs has to do, but at least 8 (below, the two more launches of a cut
    // sequence cost more than its chunks).
    const long long chunks = (long long)T / lin::C + N;
    const long long m = std::min<long long>(std::max<long long>(8, (chunks * HV + 147) / 148), 1 << 20);
    const long long len = lin::C * m;
    L.m = (int)m;
    L.cut = T > len ? 1 : 0;
    L.slots = (int)(T / len) + N;
    L.states = L.cut ? 2 * (int)(T / len) : 0;
    auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    L.off_status = 0;
    L.off_gamma = 256;
    L.off_seg = up(L.off_gamma + (size_t)L.states * HV * sizeof(float));
    L.total = L.off_seg + (size_t)L.states * HV * kD * kD * sizeof(float);
    return L;
}

int launch_linear_prefill(const LinearPrefillArgs& p, cudaStream_t stream) {
    using namespace lin;
    LinearMaps maps{};
    if (p.T > 0 && !(map_bf16_rows(&maps.q, p.q, p.H, p.T) && map_bf16_rows(&maps.k, p.k, p.H, p.T) &&
                     map_bf16_rows(&maps.v, p.v, p.HV, p.T)))
        return -3;
    if (cudaFuncSetAttribute(gdn_linear_prefill_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess ||
        cudaFuncSetAttribute(gdn_linear_prefill_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess)
        return -1;
    const dim3 grid((unsigned)p.slots * (unsigned)p.HV), seg_grid((unsigned)p.states * (unsigned)p.HV);
    if (p.cut) {
        if (launch_pdl(gdn_linear_prefill_kernel<false>, seg_grid, dim3(kThreads), kSmem, stream, p, maps) != cudaSuccess) return -1;
        if (launch_pdl(gdn_linear_chain_kernel, dim3(seg_grid.x / 2, 16), dim3(256), 0, stream, p) != cudaSuccess) return -1;
    }
    return launch_pdl(gdn_linear_prefill_kernel<true>, grid, dim3(kThreads), kSmem, stream, p, maps) == cudaSuccess ? 0 : -1;
}

}  // namespace gdn
