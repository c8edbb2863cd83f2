// linear_prefill.cu -- linear attention with a decay for each head over packed sequences, chunked.
//
// Recurrence per token: S <- e^{a_t} S + v_t k_t^T (S is [V][K], fp32), o_t = scale S q_t.  Over a chunk of
// C = 64 tokens with G_i = a_1 + .. + a_i and the state S_0 at its start:
//   o_i = scale (e^{G_i} S_0 q_i + sum_{j <= i} e^{G_i - G_j} (q_i . k_j) v_j)
//   S_C = e^{G_C} S_0 + sum_j (e^{G_C - G_j} v_j) k_j^T
// Four tcgen05 products a chunk:
//   QK  Q (64 tokens) x K (64 tokens)                          -> q_i . k_j
//   U   Vd^T (128 V x 64 tokens, A from TMEM) x K (128 K)      -> added to the state where it lies in TMEM
//   OA  V^T (128 V x 64 tokens, MN-major from the v tile) x P  -> P = decayed, causal QK in bf16
//   OI  S_0 (128 V x 128 K, A from TMEM) x Q (64 tokens)       -> S_0 q_i, scaled by e^{G_i} in the epilogue
// The state stays in TMEM in fp32, in a unit 2^X that takes the decays, so that it is multiplied only where X would leave
// [-8, 8] or a segment ends: mostly, U adds to it and a bf16 copy for OI is all that is read.  That copy and P round to
// 2^-8, as the output does (the q, k and v they meet are bf16 too).  The decayed v is cut into three bf16 parts that keep
// all 24 bits: the state is off by 4e-7 after 2 chunks and 1e-6 in the long run (the tensor core's sums drop bits that an
// fp32 sum would round; two parts gave 3e-6).
//
// Bound by HBM for many sequences (1 KB a token and head), but not reached: S -> OI and U -> S form a chain over the
// chunks, some 2750 clocks each for one CTA an SM.  Operands that a thread forms anyway (S_0, Vd) go to TMEM, which takes
// 128 KB a chunk off the shared-memory bandwidth.  Every product and every group of warps works on a chunk of its own: TMA
// and gates run ahead, the P and V warps prepare chunk c + 1 while the tensor core works on c and the output warps write
// c - 1.  Loops stay rolled: unrolled, the roles together missed the instruction cache and warps waited 2.9 clocks an
// instruction for it, 0.5 now.  4 q/k and 8 v heads: 64 x 4096 tokens 440 to 465 us (3.6 to 3.8 TB/s, 0.30 PFLOP/s; 520
// to 545 at the power cap, called for a second on end), 16 of 6 to 8192 93, 1 x 8192 46, 1 x 100 10.9.  Not better: 1024
// threads with a second group of warps for P; OI in tf32 from the fp32 state without the bf16 copy (64 x 4096 443 -> 485).
//
// Tokens are cut evenly over the CTAs whatever the lengths: all (sequence, v-head) segments lie on one line in
// chunks, and a CTA takes an equal stretch of it.  The state at a stretch's start comes from two launches before:
// what every unfinished segment adds to the state in its CTA (U alone; it does not read the state), and a chain over
// those sums.  Where no segment is long, stretches end at segment ends and one launch does it all.
#include <algorithm>

#include "linear.cuh"
#include "prefill_kernels.cuh"
#include "sm100.cuh"

namespace gdn {

namespace lin {
constexpr int C = 64;
constexpr int kThreads = 768;  // 6 warpgroups: {TMA, U, gates, QK + OI + OA}, P, V, V, O, S
constexpr int kStages = 3;
constexpr int kGates = 8;
// stage: [Q0 | K0 | Q1 | K1 | V0 | V1], each 64 tokens x 64 columns bf16, SWIZZLE_128B
constexpr uint32_t kOffQ = 0, kOffK = 8192, kAtom = 16384, kOffV = 32768;
constexpr uint32_t kStage = 49152;
constexpr uint32_t kOffP = kStages * kStage;     // P [2][64 i][64 j] bf16
constexpr uint32_t kOffO = kOffP + 2 * 8192;     // output staging [2][2 atoms][64 tokens][64 V] bf16, SWIZZLE_128B
constexpr uint32_t kOffG = kOffO + 2 * 16384;    // gates, kGates slots of f32: [64] G | [64] factors of OI | [64] of v | [64] e^{G_b - G}, b the
                                                 // last of the token's block of 16 | state: factor, unit at the end, log of the decay, whether to multiply;
                                                 // of v: int [8] whether 16 V have a value that is not finite | int [128] its first token
constexpr uint32_t kGateFloats = 400, kOdd = 264, kOddFrom = 272;
constexpr uint32_t kOffBar = kOffG + kGates * kGateFloats * 4;
constexpr uint32_t kOffRange = kOffBar + 512;
constexpr uint32_t kSmem = kOffRange + 256;
constexpr uint32_t kTmemCols = 512;
// accumulators QK, OI, OA and the state S in fp32, then its bf16 copy and the three parts of the decayed v
constexpr uint32_t kColQK = 0, kColI = 64, kColA = 128, kColS = 192, kColB = 320, kColV = 384;
static_assert(kSmem <= 227 * 1024, "shared memory");

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718f;
// Log decays are clamped here: e^-110 is below every fp32 number, and -infinity would turn the differences
// of prefix sums into NaN.
constexpr float kMinDecay = -110.f;

// A wait tells a phase from the one before it only, so whoever waits on a barrier must be needed for its next phase
// but one: hence the pairs p_full and p_empty, whose sides run up to two chunks apart.  v_full goes by the gates' slots:
// the V warps of chunk g + 8 start when the gates of g + 8 are there, so after the outputs of g + 1 and the OA of g.
struct Bars {
    uint64_t full[kStages], empty[kStages], g_full[kGates], g_empty[kGates], v_full[kGates];
    uint64_t qk_full, qk_empty, u_ready, u_full, b_ready, i_full, p_full[2], p_empty[2], o_empty, o_full, done[2];
    uint32_t tmem;
};
static_assert(sizeof(Bars) <= 512, "barriers");
}  // namespace lin

struct LinearMaps {
    CUtensorMap q, k, v, o;  // (128, heads, T) bf16, box 64 x 1 x 64, SWIZZLE_128B
};

// ---- the line of chunks ---------------------------------------------------------------------
struct Mark {  // a place on the line: chunk `chunk` of (sequence n, v-head hv)
    int n, hv, chunk;
};

// cu_seqlens[n], clamped to [0, T]; a sequence that ends before it begins is empty.
__device__ __forceinline__ int cu_at(const LinearPrefillArgs& p, int n) {
    const long long x = p.cu64 ? reinterpret_cast<const long long*>(p.cu)[n] : reinterpret_cast<const int*>(p.cu)[n];
    return (int)max(0ll, min((long long)p.T, x));
}
__device__ __forceinline__ int lin_chunks(int s, int e) { return max(0, (e - s + lin::C - 1) / lin::C); }

// The ends of the stretch of CTA blockIdx.x, by one warp: every lane sums up an equal part of the sequences.  A segment
// takes its chunks and 2 more places for its state, which is 128 KB to the 48 of a chunk.  (Places are ints: the entry
// point refuses calls that could have 2^31.  Overlapping sequences may claim more than it counted; then every stretch is
// empty, and the status says so.)
__device__ __forceinline__ void find_range(const LinearPrefillArgs& p, Mark* at) {
    const int lane = threadIdx.x & 31, part = (p.N + 31) / 32, n0 = min(p.N, lane * part), n1 = min(p.N, n0 + part);
    long long x = 0;
    int lo = 0, total = 0, per = 0, more = 0, keep = 0;
#pragma unroll 1
    for (int round = 0; round < 2; ++round) {  // the sum of the lane's lengths, then the marks among them
        int s = n0 < n1 ? cu_at(p, n0) : 0;
#pragma unroll 1
        for (int n = n0; n < n1; ++n) {
            const int e = cu_at(p, n + 1), nc = lin_chunks(s, e), w = nc + 2;
            s = e;
            x += w;
            if (round == 0) {
                keep = max(keep, nc);
                continue;
            }
#pragma unroll 1
            for (int i = 0; i < 2; ++i) {
                const int c = blockIdx.x + i, off = min(total, c * per + min(c, more)) - lo;
                if (off < 0 || off >= w * p.HV) continue;
                Mark m{n, off / w, 0};
                const int place = off - m.hv * w - 2;
                if (nc > keep) {
                    m.chunk = max(0, place);
                } else if (2 * place >= nc) {  // a short segment is not cut: to its nearer end
                    if (++m.hv == p.HV) m = Mark{n + 1, 0, 0};
                }
                at[i] = m;
            }
            lo += w * p.HV;
        }
        if (round == 0) {
            const long long mine = x;
#pragma unroll 1
            for (int off = 1; off < 32; off <<= 1) {
                const long long y = __shfl_up_sync(0xffffffffu, x, off);
                if (lane >= off) x += y;
            }
            const long long places = __shfl_sync(0xffffffffu, x, 31);
            if (places > p.T / lin::C + 3ll * p.N) {
                if (lane < 2) at[lane] = Mark{p.N, 0, 0};
                if (blockIdx.x == 0 && lane == 0) atomicCAS(p.status, 0, kErrBadSeqlens);
                return;
            }
            keep = __reduce_max_sync(0xffffffffu, keep);
            if (keep > p.whole) keep = p.keep;
            lo = (int)(x - mine) * p.HV;
            total = (int)places * p.HV;
            const int ctas = max(1, min(p.ctas, total / p.min_share)), c = blockIdx.x + lane;
            per = total / ctas;
            more = total - per * ctas;
            if (lane < 2 && min(total, c * per + min(c, more)) == total) at[lane] = Mark{p.N, 0, 0};
        }
    }
}

struct Piece {
    int n, hv, s, e, ca, cb, nc;  // chunks [ca, cb) of the nc of segment (n, hv), tokens [s, e)
};
struct Walk {  // from a mark to another one
    Mark at, end;
    __device__ __forceinline__ bool next(const LinearPrefillArgs& p, Piece& x) {
        if (at.n > end.n || (at.n == end.n && (at.hv > end.hv || (at.hv == end.hv && at.chunk >= end.chunk)))) return false;
        x.n = at.n;
        x.hv = at.hv;
        x.s = cu_at(p, x.n);
        x.e = max(x.s, cu_at(p, x.n + 1));
        x.nc = lin_chunks(x.s, x.e);
        x.ca = at.chunk;
        x.cb = x.n == end.n && x.hv == end.hv ? end.chunk : x.nc;
        at.chunk = 0;
        if (++at.hv == p.HV) {
            at.hv = 0;
            ++at.n;
        }
        return true;
    }
    __device__ __forceinline__ bool empty() const {
        return at.n > end.n || (at.n == end.n && (at.hv > end.hv || (at.hv == end.hv && at.chunk >= end.chunk)));
    }
};

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

// ---- small pieces ---------------------------------------------------------------------------
__device__ __forceinline__ float lin_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The MMA warp stays convergent and one elected lane issues by predicate: descriptors then live in uniform
// registers, where a branch to one lane had each of them moved there per instruction (280 cycles a product step).
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t r;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
    return r;
}
// Shared-memory descriptors as (low, high) words: the high one (stride 1024, SWIZZLE_128B) is the same for all.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_low(uint32_t saddr, uint32_t lbo_bytes) { return ((saddr >> 4) & 0x3fffu) | ((lbo_bytes >> 4) << 16); }
template <bool kAccumulate>
__device__ __forceinline__ void mma_ss(uint32_t one, uint32_t dtmem, uint32_t adesc, uint32_t bdesc, uint32_t idesc) {
    asm volatile(
        "{\n.reg .pred p, e;\n.reg .b64 a, b;\nmov.b64 a, {%1, %6};\nmov.b64 b, {%2, %6};\nsetp.ne.b32 e, %5, 0;\n"
        "setp.ne.b32 p, %4, 0;\n@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n}\n" ::"r"(dtmem),
        "r"(adesc), "r"(bdesc), "r"(idesc), "n"(kAccumulate ? 1 : 0), "r"(one), "n"(kDescHigh)
        : "memory");
}
// A from TMEM (K-major, two bf16 a column)
template <bool kAccumulate>
__device__ __forceinline__ void mma_ts(uint32_t one, uint32_t dtmem, uint32_t atmem, uint32_t bdesc, uint32_t idesc) {
    asm volatile(
        "{\n.reg .pred p, e;\n.reg .b64 b;\nmov.b64 b, {%2, %6};\nsetp.ne.b32 e, %5, 0;\n"
        "setp.ne.b32 p, %4, 0;\n@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n}\n" ::"r"(dtmem),
        "r"(atmem), "r"(bdesc), "r"(idesc), "n"(kAccumulate ? 1 : 0), "r"(one), "n"(kDescHigh)
        : "memory");
}
__device__ __forceinline__ void commit_one(uint32_t one, uint64_t* bar) {
    asm volatile(
        "{\n.reg .pred e;\nsetp.ne.b32 e, %1, 0;\n@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(
            smem_u32(bar)),
        "r"(one)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
// 16 lanes x 8 columns: register 2 i (2 i + 1) of thread t is lane t / 4 (+ 8), column 4 i + t % 4.
__device__ __forceinline__ void tmem_st_16x128b_x2(uint32_t taddr, const uint32_t (&r)[4]) {
    asm volatile("tcgen05.st.sync.aligned.16x128b.x2.b32 [%0], {%1,%2,%3,%4};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
                 : "memory");
}
// 16 lanes x 32 columns: registers 4 i + {0, 1} ({2, 3}) of thread t are lane t / 4 (+ 8), columns 8 i + 2 (t % 4) + {0, 1}.
__device__ __forceinline__ void tmem_ld_16x256b_x4(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_16x256b_x8(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_st_16x256b_x8(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.16x256b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_st_16x128b_x8(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_ld_16x256b_x2(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
}
// Four 8 x 8 blocks: register i of thread t holds (row t / 4, columns 2 (t % 4) + {0, 1}) of block i, lane 8 i + r gives
// the address of its row r.
__device__ __forceinline__ void stsm_x4(uint32_t addr, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(r0), "r"(r1), "r"(r2), "r"(r3) : "memory");
}
// Four 8 x 8 blocks, each stored transposed: register i of thread t holds (row t / 4, columns 2 (t % 4) + {0, 1}) of
// block i, lane 8 i + c gives the address of its column c.
__device__ __forceinline__ void stsm_x4_t(uint32_t addr, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(r0), "r"(r1), "r"(r2), "r"(r3)
                 : "memory");
}
__device__ __forceinline__ float2 bf2_to_f2(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }

// Bounded wait (about a second); false when it gave up.  Kept short and free of branches of its own, for it is there 30
// times and the roles' loops share the instruction cache: a role looks at the results once a chunk.
__device__ __forceinline__ uint32_t lin_wait(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n.reg .pred p;\n.reg .u32 t, t0;\n"
        "mov.u32 t0, %%clock;\n"
        "LOOP:\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n@p bra DONE;\n"
        "mov.u32 t, %%clock;\nsub.u32 t, t, t0;\nsetp.lt.u32 p, t, 0x78000000;\n@p bra LOOP;\n"  // falls through with p false
        "DONE:\n"
        "selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok;
}

// The kernel's shared memory.  Named directly everywhere, so that every access is a shared-memory one with a
// constant offset; the kernel checks the alignment that the swizzled tiles need.
extern __shared__ __align__(1024) unsigned char lin_sm[];
__device__ __forceinline__ lin::Bars* lin_bars() { return reinterpret_cast<lin::Bars*>(lin_sm + lin::kOffBar); }
__device__ __forceinline__ float* lin_gates(uint32_t g) {
    return reinterpret_cast<float*>(lin_sm + lin::kOffG + (g % lin::kGates) * (lin::kGateFloats * 4));
}

struct LinCtx {
    uint32_t sbase;
    static constexpr uint32_t tmem = 0;  // a CTA that holds all 512 columns holds them from column 0
    Walk walk;
    int prev;  // the CTA's slot of segment states is blockIdx.x; a stretch that begins inside a segment starts from `prev`
};

// ---- roles ----------------------------------------------------------------------------------
// Every wait is bounded; on expiry the role ends at the end of its chunk, and the others' waits expire in turn.
#define LIN_WAIT(bar, parity) ok &= lin_wait(&(bar), (uint32_t)(parity) & 1u)
#define LIN_CHECK() \
    if (!__all_sync(0xffffffffu, ok)) return false

// Warp 0: the TMA copies.
template <bool kOut>
__device__ __forceinline__ bool role_load(const LinearPrefillArgs& p, const LinearMaps& maps, const LinCtx& x, uint32_t one, int* issued) {
    using namespace lin;
    Walk w = x.walk;
    Piece pc;
    uint32_t s = 0, s_ph = 1, ok = 1;
#pragma unroll 1
    while (w.next(p, pc)) {
        if (pc.e <= pc.s) continue;
        const int hq = pc.hv / (p.HV / p.H);
#pragma unroll 1
        for (int c = pc.ca; c < pc.cb; ++c) {
            const int t0 = pc.s + c * C;
            LIN_WAIT(lin_bars()->empty[s], s_ph);  // (the first round passes: the barriers are new)
            LIN_CHECK();
            if (one) {
                unsigned char* st = lin_sm + s * kStage;
                mbar_arrive_expect_tx(&lin_bars()->full[s], kOut ? 49152 : 32768);
#pragma unroll 1
                for (int a = 0; a < 2; ++a) {
                    if (kOut) tma_load_3d(st + kOffQ + a * kAtom, &maps.q, 64 * a, hq, t0, &lin_bars()->full[s]);
                    tma_load_3d(st + kOffK + a * kAtom, &maps.k, 64 * a, hq, t0, &lin_bars()->full[s]);
                    tma_load_3d(st + kOffV + a * 8192, &maps.v, 64 * a, pc.hv, t0, &lin_bars()->full[s]);
                }
            }
            __syncwarp();
            ++*issued;
            if (++s == kStages) {
                s = 0;
                s_ph ^= 1;
            }
        }
    }
    return true;
}

// Warp 2: prefix and suffix sums of every chunk's log decays (base 2 from here on), two tokens a lane.  The state in TMEM
// is S 2^-X: as long as -8 <= X <= 8 a chunk's decay only moves X (its own tokens enter times 2^-(G_j + X)), so the state
// is not touched; beyond that it is multiplied by 2^(X + G_C) and X is 0 again.  The exponents stay small, so fp32 holds
// them to 2^-21; what the sums X drop is carried along, since it would add up over the chunks.
__device__ __forceinline__ bool role_gates(const LinearPrefillArgs& p, const LinCtx& x) {
    using namespace lin;
    const int lane = threadIdx.x & 31;
    Walk w = x.walk;
    Piece pc;
    uint32_t g = 0, ok = 1;
#pragma unroll 1
    while (w.next(p, pc)) {
        if (pc.e <= pc.s) continue;
        float X = 0.f, rest = 0.f;  // X, and what its sum has rounded away
#pragma unroll 1
        for (int c = pc.ca; c < pc.cb; ++c, ++g) {
            const int t0 = pc.s + c * C, L = min(C, pc.e - t0);
            float a0 = 0.f, a1 = 0.f;
            if (2 * lane < L) a0 = p.decay[p.per_token ? (size_t)(t0 + 2 * lane) * p.HV + pc.hv : pc.hv];
            if (2 * lane + 1 < L) a1 = p.decay[p.per_token ? (size_t)(t0 + 2 * lane + 1) * p.HV + pc.hv : pc.hv];
            a0 = (a0 < kMinDecay ? kMinDecay : a0) * kLog2e;
            a1 = (a1 < kMinDecay ? kMinDecay : a1) * kLog2e;
            float pre = a0 + a1, suf = a0 + a1;
#pragma unroll 1
            for (int off = 1; off < 32; off <<= 1) {
                const float y = __shfl_up_sync(0xffffffffu, pre, off), z = __shfl_down_sync(0xffffffffu, suf, off);
                if (lane >= off) pre += y;
                if (lane + off < 32) suf += z;
            }
            float before = __shfl_up_sync(0xffffffffu, pre, 1), after = __shfl_down_sync(0xffffffffu, suf, 1);
            if (lane == 0) before = 0.f;
            if (lane == 31) after = 0.f;
            const float total = __shfl_sync(0xffffffffu, pre, 31), g0 = before + a0, gb = __shfl_sync(0xffffffffu, pre, lane | 7);
            const bool scale = fabsf(X + total) > 8.f;
            // the last group to finish chunk g - 7 has finished g - 8 for all the others: the slot is free
            if (g >= kGates) LIN_WAIT(lin_bars()->g_empty[(g + 1) % kGates], (g + 1) / kGates - 1);
            float* gt = lin_gates(g);
            *reinterpret_cast<float2*>(gt + 2 * lane) = make_float2(g0, pre);
            *reinterpret_cast<float2*>(gt + 64 + 2 * lane) = make_float2(p.scale * lin_ex2(g0 + X), p.scale * lin_ex2(pre + X));
            // 2^(G_C - G_j) from the sum of the later decays: exact where it matters, near the chunk's end
            *reinterpret_cast<float2*>(gt + 128 + 2 * lane) =
                scale ? make_float2(lin_ex2(after + a1), lin_ex2(after))
                      : make_float2(lin_ex2(-(g0 + X)) * (1.f - kLn2 * rest), lin_ex2(-(pre + X)) * (1.f - kLn2 * rest));
            *reinterpret_cast<float2*>(gt + 192 + 2 * lane) = make_float2(lin_ex2(gb - g0), lin_ex2(gb - pre));
            const float sum = X + total, added = sum - X;
            rest += (X - (sum - added)) + (total - added);
            const float unit = exp2f(sum) * (1.f + kLn2 * rest);
            X = scale ? 0.f : sum;
            if (scale) rest = 0.f;
            if (lane == 0) {
                gt[256] = scale ? unit : 1.f;  // what the state is multiplied by
                gt[257] = scale ? 1.f : unit;  // of the state at the chunk's end
                gt[258] = total;               // the chunk's decay, as its logarithm
                gt[259] = scale ? 1.f : 0.f;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&lin_bars()->g_full[g % kGates]);
            LIN_CHECK();
        }
    }
    return true;
}

__device__ __forceinline__ int count_chunks(const LinearPrefillArgs& p, Walk w) {
    Piece pc;
    int total = 0;
#pragma unroll 1
    while (w.next(p, pc))
        if (pc.e > pc.s) total += pc.cb - pc.ca;
    return __shfl_sync(0xffffffffu, total, 0);
}

// Warp 1: the products U, which the chain over chunks goes through.
__device__ __forceinline__ bool role_u(const LinearPrefillArgs& p, const LinCtx& x, uint32_t one) {
    using namespace lin;
    const int total = count_chunks(p, x.walk);
    constexpr uint32_t idesc = umma_idesc_bf16(128, 128, false, true);
    const uint32_t d_k = desc_low(x.sbase + kOffK, kAtom);  // at stage 0; an offset adds its sixteenth
    uint32_t s = 0, ok = 1;
#pragma unroll 1
    for (int g = 0; g < total; ++g) {
        const uint32_t st = (uint32_t)s * (kStage >> 4);
        LIN_WAIT(lin_bars()->u_ready, g);
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < 12; ++kk) mma_ts<true>(one, x.tmem + kColS, x.tmem + kColV + 8 * kk, d_k + st + 128 * (kk & 3), idesc);
        commit_one(one, &lin_bars()->u_full);
        commit_one(one, &lin_bars()->empty[s]);
        if (++s == kStages) s = 0;
        LIN_CHECK();
    }
    return true;
}

// Warp 3: the products of the output.
__device__ __forceinline__ bool role_mma(const LinearPrefillArgs& p, const LinCtx& x, uint32_t one) {
    using namespace lin;
    const int total = count_chunks(p, x.walk);
    constexpr uint32_t idesc_qk = umma_idesc_bf16(64, 64, false, false), idesc_oi = umma_idesc_bf16(128, 64, false, false);
    constexpr uint32_t idesc_oa = umma_idesc_bf16(128, 64, true, false);
    // descriptors at stage 0; an offset adds its sixteenth
    const uint32_t d_q = desc_low(x.sbase + kOffQ, 16), d_k = desc_low(x.sbase + kOffK, 16);
    const uint32_t d_v = desc_low(x.sbase + kOffV, 8192), d_p = desc_low(x.sbase + kOffP, 16);
    auto step = [](int kk) { return (uint32_t)(((kk >> 2) * kAtom + (kk & 3) * 32) >> 4); };  // 16 of 128 columns
    uint32_t s = 0, sn = 0, sn_ph = 0, ok = 1;  // stages of chunk g and of the next QK, and the latter's phase
#pragma unroll 1
    for (int g = -1; g < total; ++g) {
        const uint32_t st = (uint32_t)s * (kStage >> 4), pb = d_p + (uint32_t)(g & 1) * 512u;
        if (g >= 0) {
            LIN_WAIT(lin_bars()->b_ready, g);  // the state's bf16 copy
            if (g > 0) LIN_WAIT(lin_bars()->o_empty, g - 1);
            tc_fence_after();
            mma_ts<false>(one, x.tmem + kColI, x.tmem + kColB, d_q + st, idesc_oi);
#pragma unroll
            for (int kk = 1; kk < 8; ++kk) mma_ts<true>(one, x.tmem + kColI, x.tmem + kColB + 8 * kk, d_q + st + step(kk), idesc_oi);
            commit_one(one, &lin_bars()->i_full);
        }
        if (g + 1 < total) {  // QK of the next chunk, so that the P warps are ahead
            LIN_WAIT(lin_bars()->full[sn], sn_ph);
            if (g >= 0) LIN_WAIT(lin_bars()->qk_empty, g);
            tc_fence_after();
            const uint32_t st1 = (uint32_t)sn * (kStage >> 4);
            mma_ss<false>(one, x.tmem + kColQK, d_q + st1, d_k + st1, idesc_qk);
#pragma unroll
            for (int kk = 1; kk < 8; ++kk) mma_ss<true>(one, x.tmem + kColQK, d_q + st1 + step(kk), d_k + st1 + step(kk), idesc_qk);
            commit_one(one, &lin_bars()->qk_full);
            if (++sn == kStages) {
                sn = 0;
                sn_ph ^= 1;
            }
        }
        if (g >= 0) {
            LIN_WAIT(lin_bars()->p_full[g & 1], g >> 1);
            LIN_WAIT(lin_bars()->v_full[g % kGates], g / kGates);  // no foreign rows in v: P is 0 there, but 0 NaN is NaN
            tc_fence_after();
            mma_ss<false>(one, x.tmem + kColA, d_v + st, pb, idesc_oa);
#pragma unroll
            for (int kk = 1; kk < 4; ++kk) mma_ss<true>(one, x.tmem + kColA, d_v + st + 128 * kk, pb + 2 * kk, idesc_oa);
            commit_one(one, &lin_bars()->o_full);
            commit_one(one, &lin_bars()->p_empty[g & 1]);
            commit_one(one, &lin_bars()->empty[s]);
            if (++s == kStages) s = 0;
        }
        LIN_CHECK();
    }
    return true;
}

// Warps 4-7: P, 16 rows a warp (a 64-row accumulator has its rows in the first 16 lanes of every quarter).  Blocks above
// the diagonal stay the zeros that the kernel starts with.
__device__ __forceinline__ bool role_p(const LinearPrefillArgs& p, const LinCtx& x) {
    using namespace lin;
    const int lane = threadIdx.x & 31, quarter = __shfl_sync(0xffffffffu, (threadIdx.x >> 5) & 3, 0);
    const uint32_t tl = x.tmem + kColQK + ((uint32_t)(32 * quarter) << 16);
    const int r = 16 * quarter + (lane >> 2);  // and r + 8
    // stmatrix rows: P row (lane % 16), 16-byte chunk lane / 16 of a block of 16 columns
    const uint32_t row = x.sbase + kOffP + (uint32_t)(16 * quarter + (lane & 15)) * 128, sw = lane & 7;
    Walk w = x.walk;
    Piece pc;
    uint32_t g = 0, ok = 1;
#pragma unroll 1
    while (w.next(p, pc)) {
        if (pc.e <= pc.s) continue;
#pragma unroll 1
        for (int c = pc.ca; c < pc.cb; ++c, ++g) {
            const int L = min(C, pc.e - pc.s - c * C);
            const float* g2 = lin_gates(g);
            LIN_WAIT(lin_bars()->g_full[g % kGates], g / kGates);
            const float2 gi = make_float2(g2[r], g2[r + 8]);
            LIN_WAIT(lin_bars()->qk_full, g);
            tc_fence_after();
            if (g >= 2) LIN_WAIT(lin_bars()->p_empty[g & 1], (g >> 1) - 1);
#pragma unroll 1
            for (int b = 0; b <= quarter; ++b) {  // 16 columns
                uint32_t d[8], o[4];
                tmem_ld_16x256b_x2(tl + 16 * b, d);
                // e^{G_i - G_j} = e^{G_i - G_b} e^{G_b - G_j} below the diagonal (both factors <= 1), directly on it
                const bool diag = b == quarter;
                const float gb = g2[16 * b + 15];
                const float2 rf = diag ? gi : make_float2(lin_ex2(gi.x - gb), lin_ex2(gi.y - gb));
                const int j0 = 16 * b + 2 * (lane & 3);
                const float2 c0 = *reinterpret_cast<const float2*>(g2 + (diag ? 0 : 192) + j0);
                const float2 c1 = *reinterpret_cast<const float2*>(g2 + (diag ? 0 : 192) + j0 + 8);
                float2 f[4] = {mul2(make_float2(rf.x, rf.x), c0), mul2(make_float2(rf.y, rf.y), c0),
                               mul2(make_float2(rf.x, rf.x), c1), mul2(make_float2(rf.y, rf.y), c1)};
                if (diag) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {  // columns j0 (+ 8), rows r (+ 8)
                        const float2 c = i < 2 ? c0 : c1;
                        const float fr = i & 1 ? rf.y : rf.x;
                        f[i] = make_float2(lin_ex2(fr - c.x), lin_ex2(fr - c.y));
                    }
                }
                tmem_ld_wait();
                tmem_regs_ready_n(d);
                // kept: columns on or below the diagonal, and not behind the segment's end (k rows of another sequence)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int j = j0 + 8 * (i >> 1), lim = min(r + 8 * (i & 1), L - 1);
                    const float2 y = mul2(f[i], make_float2(__uint_as_float(d[2 * i]), __uint_as_float(d[2 * i + 1])));
                    o[i] = pack_bf16x2(j <= lim ? y.x : 0.f, j + 1 <= lim ? y.y : 0.f);
                }
                stsm_x4(row + (uint32_t)(g & 1) * 8192 + ((((uint32_t)(2 * b) + (lane >> 4)) ^ sw) << 4), o[0], o[1], o[2], o[3]);
            }
            tc_fence_before();
            mbar_arrive(&lin_bars()->qk_empty);
            fence_async_smem();
            mbar_arrive(&lin_bars()->p_full[g & 1]);
            LIN_CHECK();
        }
    }
    return true;
}

// Column v of a staged [2 atoms][64 tokens][64 V] bf16 tile becomes NaN from token `from` on.
__device__ __noinline__ void void_odd_v(unsigned char* tile, int v, int from) {
    for (int t = from; t < 64; ++t)
        *reinterpret_cast<uint16_t*>(tile + (v >> 6) * 8192 + t * 128 + ((((v >> 3) & 7) ^ (t & 7)) << 4) + (v & 7) * 2) = 0x7fff;
}
// By a warp: of the 64 tokens and the V columns v0 .. v0 + 15 of a v tile, values that are not finite become 0, and `from`
// gets the first token of one for each V (64: there is none).
__device__ __noinline__ void hide_odd_v(unsigned char* tile, int* from, int v0) {
    const int lane = threadIdx.x & 31, v = v0 + (lane & 15);
    int first = 64;
    for (int t = lane >> 4; t < 64; t += 2) {
        uint16_t* at = reinterpret_cast<uint16_t*>(tile + (v >> 6) * 8192 + t * 128 + ((((v >> 3) & 7) ^ (t & 7)) << 4) + (v & 7) * 2);
        if ((*at & 0x7f80u) == 0x7f80u) {
            *at = 0;
            first = min(first, t);
        }
    }
    first = min(first, __shfl_xor_sync(0xffffffffu, first, 16));
    from[v] = first;
}

// Warps 8-15: the decayed v, transposed, as three bf16 parts in TMEM (lane = V index, two tokens a column); 16 V a warp.
template <bool kOut>
__device__ __forceinline__ bool role_v(const LinearPrefillArgs& p, const LinCtx& x) {
    using namespace lin;
    const int lane = threadIdx.x & 31, quarter = (threadIdx.x >> 5) & 3, hf = (threadIdx.x >> 7) - 2, tid = threadIdx.x - 256;
    const uint32_t tl = x.tmem + kColV + ((uint32_t)(32 * quarter + 16 * hf) << 16);
    // ldmatrix rows: token (lane % 8) + 8 (lane / 16), 16-byte chunk of 8 V
    const int tok = (lane & 7) + 8 * (lane >> 4), ch = 4 * quarter + 2 * hf + ((lane >> 3) & 1);
    const uint32_t from = kOffV + (uint32_t)(ch >> 3) * 8192 + (uint32_t)tok * 128 + (uint32_t)(((ch & 7) ^ (tok & 7)) << 4);
    Walk w = x.walk;
    Piece pc;
    uint32_t g = 0, s = 0, s_ph = 0, ok = 1;
#pragma unroll 1
    while (w.next(p, pc)) {
        if (pc.e <= pc.s) continue;
#pragma unroll 1
        for (int c = pc.ca; c < pc.cb; ++c, ++g) {
            const int L = min(C, pc.e - pc.s - c * C);
            const float* er = lin_gates(g) + 128 + 2 * (lane & 3);
            LIN_WAIT(lin_bars()->g_full[g % kGates], g / kGates);
            LIN_WAIT(lin_bars()->full[s], s_ph);
            unsigned char* st = lin_sm + s * kStage;
            if (L < C) {
                // Rows behind the segment's end hold another sequence's tokens, or zeros.  They become zero in v and
                // k before OA (v_full) and U (u_ready) read them; QK may read either, its columns there are dropped.
                for (int i = tid; i < (C - L) * 16; i += 256) {
                    const uint32_t off = (uint32_t)(L + (i >> 4)) * 128 + (i & 7) * 16;
                    *reinterpret_cast<uint4*>(st + kOffV + ((i >> 3) & 1) * 8192 + off) = make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint4*>(st + kOffK + ((i >> 3) & 1) * kAtom + off) = make_uint4(0, 0, 0, 0);
                }
                fence_async_smem();
                named_bar_sync(1, 256);
            }
            uint32_t part[3][16];
            float2 zero = make_float2(0.f, 0.f);  // NaN if one of the values is not finite
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // 16 V x 16 tokens, transposed
                uint32_t raw[4];
                ldsm_x4_t(raw[0], raw[1], raw[2], raw[3], st + from + 2048 * i);
#pragma unroll
                for (int j = 0; j < 4; ++j) {  // {0, 1}: tokens 16 i + .., {2, 3}: 8 later; odd ones are 8 V further
                    float2 y = mul2(bf2_to_f2(raw[j]), *reinterpret_cast<const float2*>(er + 16 * i + 8 * (j >> 1)));
                    if (kOut) zero = fma2(y, make_float2(0.f, 0.f), zero);
#pragma unroll
                    for (int k = 0; k < 3; ++k) {
                        part[k][4 * i + j] = pack_bf16x2(y.x, y.y);
                        if (k < 2) y = sub2(y, bf2_to_f2(part[k][4 * i + j]));
                    }
                }
            }
            if (g > 0) LIN_WAIT(lin_bars()->u_full, g - 1);  // the parts of the chunk before are consumed
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < 3; ++k) tmem_st_16x128b_x8(tl + 32 * k, part[k]);
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(&lin_bars()->u_ready);
            if (kOut) {
                const bool odd = __any_sync(0xffffffffu, !(zero.x + zero.y == 0.f));
                int* note = reinterpret_cast<int*>(lin_gates(g) + kOdd);
                if (lane == 0) note[2 * quarter + hf] = odd;
                if (odd) {
                    // P is 0 for a later token, but 0 NaN is NaN: OA gets 0 in place of such values, and the outputs of that
                    // V become NaN from its token on (the state does by U).
                    hide_odd_v(st + kOffV, note + (kOddFrom - kOdd), 32 * quarter + 16 * hf);
                    fence_async_smem();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&lin_bars()->v_full[g % kGates]);
            }
            if (++s == kStages) {
                s = 0;
                s_ph ^= 1;
            }
            LIN_CHECK();
        }
    }
    return true;
}

// Warps 16-19: o = scale (e^{G_i} OI + OA), transposed into shared memory; whole chunks leave by TMA.
__device__ __forceinline__ bool role_o(const LinearPrefillArgs& p, const LinearMaps& maps, const LinCtx& x) {
    using namespace lin;
    const int lane = threadIdx.x & 31, quarter = (threadIdx.x >> 5) & 3, r = threadIdx.x & 127;
    const uint32_t tl = x.tmem + ((uint32_t)(32 * quarter) << 16);
    // stmatrix rows: token (lane % 8) + 8 (lane / 16), 16-byte chunk of 8 V
    const uint32_t to = x.sbase + kOffO + (uint32_t)(quarter >> 1) * 8192 + (uint32_t)((lane & 7) + 8 * (lane >> 4)) * 128;
    const uint32_t ch = 4 * (quarter & 1) + ((lane >> 3) & 1), sw = lane & 7;
    Walk w = x.walk;
    Piece pc;
    uint32_t g = 0, ok = 1;
#pragma unroll 1
    while (w.next(p, pc)) {
        if (pc.e <= pc.s) continue;
#pragma unroll 1
        for (int c = pc.ca; c < pc.cb; ++c, ++g) {
            const int t0 = pc.s + c * C, L = min(C, pc.e - t0);
            const float* eg = lin_gates(g) + 64;
            const uint32_t buf = (uint32_t)(g & 1) * 16384;
            LIN_WAIT(lin_bars()->g_full[g % kGates], g / kGates);
            LIN_WAIT(lin_bars()->o_full, g);
            tc_fence_after();
#pragma unroll 1
            for (int th = 0; th < 2; ++th) {  // 32 tokens
                float2 e2[4];  // tokens 8 i + 2 (lane % 4) and the next
#pragma unroll
                for (int i = 0; i < 4; ++i) e2[i] = *reinterpret_cast<const float2*>(eg + 32 * th + 8 * i + 2 * (lane & 3));
#pragma unroll 1
                for (int hf = 0; hf < 2; ++hf) {  // 16 V
                    uint32_t y[16], z[16];
                    const uint32_t ta = tl + ((uint32_t)(16 * hf) << 16) + 32 * th;
                    tmem_ld_16x256b_x4(ta + kColI, y);
                    tmem_ld_16x256b_x4(ta + kColA, z);
                    tmem_ld_wait();
                    tmem_regs_ready_n(y);
                    tmem_regs_ready_n(z);
                    uint32_t o[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {  // even: V row lane / 4, odd: 8 further
                        const float2 v2 = fma2(e2[i >> 1], make_float2(__uint_as_float(y[2 * i]), __uint_as_float(y[2 * i + 1])),
                                               mul2(make_float2(p.scale, p.scale), make_float2(__uint_as_float(z[2 * i]), __uint_as_float(z[2 * i + 1]))));
                        o[i] = pack_bf16x2(v2.x, v2.y);
                    }
                    const uint32_t at = to + buf + (32 * th) * 128 + (((ch + 2 * hf) ^ sw) << 4);
                    stsm_x4_t(at, o[0], o[1], o[2], o[3]);
                    stsm_x4_t(at + 16 * 128, o[4], o[5], o[6], o[7]);
                }
            }
            tc_fence_before();
            mbar_arrive(&lin_bars()->o_empty);
            LIN_WAIT(lin_bars()->v_full[g % kGates], g / kGates);
            const int* note = reinterpret_cast<const int*>(eg - 64);
            const int2 odd = *reinterpret_cast<const int2*>(note + kOdd + 2 * quarter);
            if ((odd.x | odd.y) && __all_sync(0xffffffffu, ok)) {  // (the notes are there)
                if (lane < 16 ? odd.x : odd.y) void_odd_v(lin_sm + kOffO + buf, 32 * quarter + lane, note[kOddFrom + 32 * quarter + lane]);
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&lin_bars()->g_empty[g % kGates]);
            if (r == 0) tma_store_wait_read();  // the chunk before has left its buffer, which the next one writes
            named_bar_sync(2, 128);
            if (L == C) {
                if (r == 0) {
                    tma_store_3d(&maps.o, 0, pc.hv, t0, lin_sm + kOffO + buf);
                    tma_store_3d(&maps.o, 64, pc.hv, t0, lin_sm + kOffO + buf + 8192);
                    tma_store_commit();
                }
            } else {  // rows behind the segment's end are not its own
#pragma unroll 1
                for (int q = r; q < L * 16; q += 128) {
                    const int i = q >> 4, k = q & 15;
                    *reinterpret_cast<uint4*>(p.out + ((size_t)(t0 + i) * p.HV + pc.hv) * kD + 8 * k) =
                        *reinterpret_cast<const uint4*>(lin_sm + kOffO + buf + (k >> 3) * 8192 + i * 128 + (((k & 7) ^ (i & 7)) << 4));
                }
                named_bar_sync(2, 128);  // nobody writes the other buffer, then this one, before it is read
            }
            LIN_CHECK();
        }
    }
    return true;
}

// Warps 20-23: the state, V row r a thread.  It lives in TMEM, where U adds to it: before U of chunk g the warps read
// it and leave its bf16 copy for OI; now and then (see the gates) they write it back in another unit.
template <bool kOut>
__device__ __forceinline__ bool role_s(const LinearPrefillArgs& p, const LinCtx& x) {
    using namespace lin;
    const int lane = threadIdx.x & 31, quarter = (threadIdx.x >> 5) & 3, r = threadIdx.x & 127;
    const uint32_t tl = x.tmem + ((uint32_t)(32 * quarter) << 16);
    Walk w = x.walk;
    Piece pc;
    uint32_t g = 0, ok = 1;
#pragma unroll 1
    while (w.next(p, pc)) {
        const size_t at = ((size_t)pc.n * p.HV + pc.hv) * kD * kD;
        const float* src = nullptr;
        if (kOut) {
            if (pc.ca > 0)
                src = p.seg + (size_t)x.prev * kD * kD;
            else if (p.state)
                src = pc.cb < pc.nc ? p.seg + (size_t)(p.ctas + blockIdx.x) * kD * kD : p.state + at;
        }
        float* dst = kOut ? p.new_state + at : p.seg + (size_t)blockIdx.x * kD * kD;
        const bool ends = !kOut || pc.cb == pc.nc;
        if (src && pc.e > pc.s)  // on its way to L2 while the gates and the first tiles are
            for (int j = r; j < kD * kD / 32; j += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(src + 32 * j));
        if (pc.e <= pc.s) {  // an empty sequence keeps its state
#pragma unroll 4
            for (int j = r; j < kD * kD / 4; j += 128)
                reinterpret_cast<float4*>(dst)[j] = src ? reinterpret_cast<const float4*>(src)[j] : make_float4(0.f, 0.f, 0.f, 0.f);
            continue;
        }
        float gamma = 0.f, unit = 1.f;  // gamma: logarithm of the piece's decay, so that its rounding is not a product's
#pragma unroll 1
        for (int c = pc.ca; c < pc.cb; ++c, ++g) {
            const float* gt = lin_gates(g);
            LIN_WAIT(lin_bars()->g_full[g % kGates], g / kGates);
            const float factor = gt[256];
            unit = gt[257];
            gamma += gt[258];
            const bool begins = c == pc.ca, write = gt[259] != 0.f;
            if (g > 0) {
                // the state is complete (or, at a segment's start, was read) and OI has read its copy
                LIN_WAIT(lin_bars()->u_full, g - 1);
                if (kOut) LIN_WAIT(lin_bars()->i_full, g - 1);
            }
            tc_fence_after();
            if (begins) {
                // 16 V x 64 K a round, as fragments: a load of the warp covers eight whole 32-byte sectors
#pragma unroll 1
                for (int b = 0; b < 4; ++b) {
                    uint32_t d[32];
                    const float* row = src + (size_t)(32 * quarter + 16 * (b & 1) + (lane >> 2)) * kD + 64 * (b >> 1) + 2 * (lane & 3);
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float2 y = src ? *reinterpret_cast<const float2*>(row + 8 * (j >> 1) + 8 * kD * (j & 1)) : make_float2(0.f, 0.f);
                        d[2 * j] = __float_as_uint(y.x);
                        d[2 * j + 1] = __float_as_uint(y.y);
                    }
                    const uint32_t ta = tl + ((uint32_t)(16 * (b & 1)) << 16);
                    if (kOut) {
                        uint32_t o[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) o[j] = pack_bf16x2(__uint_as_float(d[2 * j]), __uint_as_float(d[2 * j + 1]));
                        tmem_st_16x128b_x8(ta + kColB + 32 * (b >> 1), o);
                    }
#pragma unroll
                    for (int j = 0; j < 32; ++j) d[j] = __float_as_uint(factor * __uint_as_float(d[j]));
                    tmem_st_16x256b_x8(ta + kColS + 64 * (b >> 1), d);
                }
                tmem_st_wait();
            } else if (kOut || write) {
#pragma unroll 1
                for (int b = 0; b < 4; ++b) {  // 32 K
                    uint32_t d[32];
                    tmem_ld32_async(tl + kColS + 32 * b, d);
                    tmem_ld_wait();
                    tmem_regs_ready(d);
                    if (kOut) {
                        uint32_t o[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) o[j] = pack_bf16x2(__uint_as_float(d[2 * j]), __uint_as_float(d[2 * j + 1]));
                        tmem_st16(tl + kColB + 16 * b, o);
                    }
                    if (write) {
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            const float2 z = mul2(make_float2(__uint_as_float(d[j]), __uint_as_float(d[j + 1])), make_float2(factor, factor));
                            d[j] = __float_as_uint(z.x);
                            d[j + 1] = __float_as_uint(z.y);
                        }
                        tmem_st32(tl + kColS + 32 * b, d);
                    }
                }
                if (write) tmem_st_wait();
            }
            tc_fence_before();
            mbar_arrive(&lin_bars()->u_ready);  // U may add to the state
            if (kOut) {
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive(&lin_bars()->b_ready);
            } else {
                __syncwarp();
                if (lane == 0) mbar_arrive(&lin_bars()->g_empty[g % kGates]);
            }
            LIN_CHECK();
        }
        if (ends) {
            LIN_WAIT(lin_bars()->u_full, g - 1);
            LIN_CHECK();
            tc_fence_after();
#pragma unroll 1
            for (int b = 0; b < 4; ++b) {
                uint32_t d[32];
                tmem_ld_16x256b_x8(tl + ((uint32_t)(16 * (b & 1)) << 16) + kColS + 64 * (b >> 1), d);
                tmem_ld_wait();
                tmem_regs_ready(d);
                float* row = dst + (size_t)(32 * quarter + 16 * (b & 1) + (lane >> 2)) * kD + 64 * (b >> 1) + 2 * (lane & 3);
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    *reinterpret_cast<float2*>(row + 8 * (j >> 1) + 8 * kD * (j & 1)) =
                        make_float2(unit * __uint_as_float(d[2 * j]), unit * __uint_as_float(d[2 * j + 1]));
            }
            if (!kOut && r == 0) p.gamma[blockIdx.x] = exp2f(gamma);
        }
    }
    return true;
}
#undef LIN_WAIT

// kOut: the output launch.  Otherwise the segment launch: what the unfinished segment at the end of every stretch
// adds to the state there.
template <bool kOut>
__global__ void __launch_bounds__(lin::kThreads, 1)
    gdn_linear_prefill_kernel(LinearPrefillArgs p, const __grid_constant__ LinearMaps maps) {
    using namespace lin;
    Bars* b = lin_bars();
    Mark* range = reinterpret_cast<Mark*>(lin_sm + kOffRange);
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // known to be uniform, and with it all role code
    if (smem_u32(lin_sm) & 1023u) {
        if (tid == 0) atomicCAS(p.status, 0, kErrPrepTmaTimeout);
        return;
    }
    if (tid == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&b->full[s], 1);
            mbar_init(&b->empty[s], kOut ? 2 : 1);
        }
        for (int s = 0; s < kGates; ++s) {
            mbar_init(&b->g_full[s], 1);
            mbar_init(&b->g_empty[s], 4);
            mbar_init(&b->v_full[s], 8);
        }
        mbar_init(&b->qk_full, 1);
        mbar_init(&b->qk_empty, 128);
        mbar_init(&b->u_ready, 256 + 128);  // V and S warps
        mbar_init(&b->u_full, 1);
        mbar_init(&b->p_full[0], 128);
        mbar_init(&b->p_full[1], 128);
        mbar_init(&b->p_empty[0], 1);
        mbar_init(&b->p_empty[1], 1);
        mbar_init(&b->b_ready, 128);
        mbar_init(&b->i_full, 1);
        mbar_init(&b->o_empty, 128);
        mbar_init(&b->o_full, 1);
        mbar_init(&b->done[0], 1);
        mbar_init(&b->done[1], 1);
        mbar_fence_init();
    }
    pdl_wait();
    pdl_trigger();
    if (blockIdx.x == 0 && tid == 0 && (!kOut || !p.cut)) *p.status = 0;  // the call's first launch
    if (kOut && p.zero_unowned && warp >= 2)  // beside find_range
        zero_rows(p, blockIdx.x * (kThreads - 64) + tid - 64, gridDim.x * (kThreads - 64));
    if (warp == 0) find_range(p, range);
    if (warp == 1) tmem_alloc(&b->tmem, kTmemCols);
    if (kOut) {  // P above its diagonal
        for (int i = tid; i < 1024; i += kThreads) reinterpret_cast<uint4*>(lin_sm + kOffP)[i] = make_uint4(0, 0, 0, 0);
        fence_async_smem();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const Mark m0 = range[0], m1 = range[1];
    LinCtx x;
    x.sbase = smem_u32(lin_sm);
    x.prev = (int)blockIdx.x - 1;
    if (kOut) {
        x.walk = Walk{m0, m1};
    } else {
        const int from = m0.n == m1.n && m0.hv == m1.hv ? m0.chunk : 0;
        x.walk = Walk{Mark{m1.n, m1.hv, from}, m1};
        // 1: a segment begins here and goes on, 2: one goes through, 0: neither
        if (tid == 0) p.kind[blockIdx.x] = make_int4(x.walk.empty() ? 0 : from > 0 ? 2 : 1, m1.n, m1.hv, 0);
    }
    bool ok = true;
    if (warp == 0) {
        int issued = 0;
        if (!(ok = role_load<kOut>(p, maps, x, elect_one(), &issued)))
            // gave up: let copies already in flight land (bounded) before the CTA exits
            for (int g = max(0, issued - kStages); g < issued; ++g) lin_wait(&b->full[g % kStages], (uint32_t)((g / kStages) & 1));
    } else if (warp == 1 || (kOut && warp == 3)) {
        const uint32_t one = elect_one();
        ok = warp == 1 ? role_u(p, x, one) : role_mma(p, x, one);
        // products still in flight end before the TMEM is given back
        commit_one(one, &b->done[warp >> 1]);
        ok = lin_wait(&b->done[warp >> 1], 0) && ok;
    } else if (warp == 2) {
        ok = role_gates(p, x);
    } else if (warp < 4) {
    } else if (warp < 8) {
        if (kOut) ok = role_p(p, x);
    } else if (warp < 16) {
        ok = role_v<kOut>(p, x);
    } else if (warp < 20) {
        if (kOut) ok = role_o(p, maps, x);
        if (kOut && warp == 16) tma_store_wait_all();  // its first lane's stores, if a wait gave up too
    } else {
        ok = role_s<kOut>(p, x);
    }
    if (!ok && lane == 0) atomicCAS(p.status, 0, kErrScanMmaTimeout);
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_dealloc(b->tmem, kTmemCols);
}

// The state at the end of every stretch that ends inside a segment, in place of what its last segment adds there, and
// the segment's initial state in the slot p.ctas further: new_state may be state itself, and a segment may end in
// one CTA before it begins in another.  One CTA per (stretch in which such a segment begins, 1024 state elements).
__global__ void __launch_bounds__(256) gdn_linear_chain_kernel(LinearPrefillArgs p) {
    pdl_wait();
    pdl_trigger();
    // the stretches that the segment goes through from here: a run of 2s, of which the first 31 come with the 1
    const int lane = threadIdx.x & 31;
    const int4 mine = p.kind[min((int)blockIdx.x + lane, p.ctas - 1)];
    if (__shfl_sync(0xffffffffu, mine.x, 0) != 1) return;
    const int n = __shfl_sync(0xffffffffu, mine.y, 0), hv = __shfl_sync(0xffffffffu, mine.z, 0);
    unsigned stops = __ballot_sync(0xffffffffu, lane > 0 && ((int)blockIdx.x + lane >= p.ctas || mine.x != 2));
    int end = blockIdx.x + 32;
    while (!stops) {
        stops = __ballot_sync(0xffffffffu, end + lane >= p.ctas || p.kind[min(end + lane, p.ctas - 1)].x != 2);
        end += 32;
    }
    end += __ffs(stops) - 1 - 32;
    const size_t el = blockIdx.y * 1024 + threadIdx.x * 4;
    float4 h = make_float4(0.f, 0.f, 0.f, 0.f);
    if (p.state) h = *reinterpret_cast<const float4*>(p.state + ((size_t)n * p.HV + hv) * kD * kD + el);
    // twelve stretches at a time: their loads do not wait for one another, nor for the stores before them
    constexpr int kBatch = 12;
#pragma unroll 1
    for (int c = blockIdx.x; c < end; c += kBatch) {
        float4 y[kBatch];
        float gm[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int k = min(c + i, end - 1);
            y[i] = __ldcg(reinterpret_cast<const float4*>(p.seg + (size_t)k * kD * kD + el));
            gm[i] = __ldcg(p.gamma + k);
        }
        if (c == (int)blockIdx.x && p.state) *reinterpret_cast<float4*>(p.seg + (size_t)(p.ctas + c) * kD * kD + el) = h;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (c + i < end) {
                h = make_float4(fmaf(gm[i], h.x, y[i].x), fmaf(gm[i], h.y, y[i].y), fmaf(gm[i], h.z, y[i].z), fmaf(gm[i], h.w, y[i].w));
                *reinterpret_cast<float4*>(p.seg + (size_t)(c + i) * kD * kD + el) = h;
            }
        }
    }
}

// A segment that is cut costs its chunks twice, in part, and the call three launches instead of one; one that is not may
// make a CTA's stretch that much longer.  So none is cut while the longest is shorter than an equal share and 16 chunks
// (us without and with cuts, 8 heads: 12 x 2048 tokens 66 and 101, 20 x 2048 119 and 138, 1 x 1000 31 and 30, 60 of 100 to
// 4000 184 and 203; 30 of 200 to 6000 205 and 180).  Beyond that, short ones stay whole: with 16 or 0.3 shares instead of
// 8 or 0.3 shares 8 of 64 to 4096 54 instead of 57, with 16 and half a share 64.  A stretch is at least 4 chunks long
// where there are cuts: 1 x 2500 31 us, with 1 chunk 32.5, with 8 40.
LinearPrefillLayout linear_prefill_layout(int N, int T, int HV) {
    LinearPrefillLayout L{};
    const long long share = ((long long)T / lin::C + 3ll * N) * HV / kLinearCtas;  // places of a CTA
    L.whole = (int)std::min<long long>(16 + share, 1 << 24);
    L.keep = (int)std::max<long long>(16, std::min<long long>(3 * share / 10, 1 << 24));
    L.cut = T > (long long)lin::C * L.whole ? 1 : 0;
    L.min_share = L.cut ? 4 : 1;
    auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    const size_t slots = L.cut ? kLinearCtas : 0;
    L.off_status = 0;
    L.off_kind = 256;
    L.off_gamma = up(L.off_kind + slots * sizeof(int4));
    L.off_seg = up(L.off_gamma + slots * sizeof(float));
    L.total = L.off_seg + 2 * slots * kD * kD * sizeof(float);
    return L;
}

int launch_linear_prefill(const LinearPrefillArgs& p, cudaStream_t stream) {
    using namespace lin;
    LinearMaps maps{};
    if (p.T > 0 && !(map_bf16_rows(&maps.q, p.q, p.H, p.T) && map_bf16_rows(&maps.k, p.k, p.H, p.T) &&
                     map_bf16_rows(&maps.v, p.v, p.HV, p.T) && map_bf16_rows(&maps.o, p.out, p.HV, p.T)))
        return -3;
    static SmemLimit out, seg;
    if (!out.raise(gdn_linear_prefill_kernel<true>, kSmem) || !seg.raise(gdn_linear_prefill_kernel<false>, kSmem)) return -1;
    const dim3 grid((unsigned)p.ctas);
    if (p.cut) {
        if (launch_pdl(gdn_linear_prefill_kernel<false>, grid, dim3(kThreads), kSmem, stream, p, maps) != cudaSuccess) return -1;
        if (launch_pdl(gdn_linear_chain_kernel, dim3((unsigned)p.ctas, 16), dim3(256), 0, stream, p) != cudaSuccess) return -1;
    }
    return launch_pdl(gdn_linear_prefill_kernel<true>, grid, dim3(kThreads), kSmem, stream, p, maps) == cudaSuccess ? 0 : -1;
}

}  // namespace gdn
