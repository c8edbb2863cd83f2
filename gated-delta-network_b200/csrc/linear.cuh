// linear.cuh -- argument blocks and launch helpers of the linear-attention and 8-bit-cache operators.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace gdn {

struct LinearDecodeArgs {
    const uint16_t* q;     // [B, H, 128] bf16
    const uint16_t* k;     // [B, H, 128] bf16
    const uint16_t* v;     // [B, HV, 128] bf16
    const float* state;    // [B, HV, 128, 128] f32 or nullptr (zeros)
    const float* decay;    // [HV] or [B, HV] log decay
    int per_token;         // decay has a row for each sequence
    float scale;
    uint16_t* out;         // [B, HV, 128] bf16
    float* new_state;      // [B, HV, 128, 128] f32 (may alias state)
    int B, H, HV;
};

struct LinearPrefillArgs {
    const uint16_t* q;     // [T, H, 128]
    const uint16_t* k;     // [T, H, 128]
    const uint16_t* v;     // [T, HV, 128]
    const float* state;    // [N, HV, 128, 128] or nullptr
    const float* decay;    // [HV] or [T, HV]
    int per_token;
    const void* cu;        // [N+1]
    int cu64;
    int N, T, H, HV;
    int zero_unowned;      // write zeros to the rows outside every sequence
    float scale;
    uint16_t* out;         // [T, HV, 128]
    float* new_state;      // [N, HV, 128, 128] (may alias state)
    int ctas;              // stretches of the line of chunks, one per SM
    int min_share;         // chunks of a stretch, at least
    int whole;             // no segment is cut if the longest one has at most this many chunks,
    int keep;              // else those of at most this many are not
    int cut;               // a sequence can be longer than that: build and chain segment states
    int* status;           // workspace: first error code of a bounded wait
    int4* kind;            // workspace: [ctas] what the stretch's last segment does, its sequence and v-head
    float* gamma;          // workspace: [ctas] product of its decays there
    float* seg;            // workspace: [2 ctas][128 V][128 K] what it adds to the state, then (after the chain) the state
                           //            at the stretch's end; behind them the initial states
};
constexpr int kLinearCtas = 148;

struct LinearPrefillLayout {
    int min_share, whole, keep, cut;
    size_t off_status, off_kind, off_gamma, off_seg, total;
};
LinearPrefillLayout linear_prefill_layout(int N, int T, int HV);

// Paged key/value cache of 8-bit codes: x = code * scale[page][head].
struct CacheArgs {
    void* k_cache;         // [pages][Hkv][P][128] int8 or e4m3
    void* v_cache;
    float* k_scale;        // [pages][Hkv]
    float* v_scale;
    int int8;              // int8 codes, else e4m3
    int pages, Hkv;
    int page_shift;        // log2(P), 4 .. 7
    const int* table;      // [B][max_pages] page of each P tokens of a sequence
    int max_pages;
    const void* seq_lens;  // [B] tokens of each sequence, the call's new ones included
    int len64;
    int B;
};

// Tokens of sequence b; a length that is not an int counts as 0.
__device__ __forceinline__ int cache_length(const CacheArgs& c, int b) {
    const long long n = c.len64 ? reinterpret_cast<const long long*>(c.seq_lens)[b] : reinterpret_cast<const int*>(c.seq_lens)[b];
    return n < 0 || n > 0x7fffffffll ? 0 : (int)n;
}

struct CacheAppendArgs {
    CacheArgs c;
    const uint16_t* k;     // [T, Hkv, 128] bf16
    const uint16_t* v;
    const void* cu;        // [B+1]
    int cu64;
    int T;
};

struct CacheAttendArgs {
    CacheArgs c;
    const uint16_t* q;     // [B, Q, Hq, 128] bf16
    int Q, Hq;
    float scale;
    uint16_t* out;         // [B, Q, Hq, 128] bf16
    int* status;           // workspace
    int4* piece;           // workspace: [kAttendCtas] {segment that CTA c begins and others end, pieces that follow, what it met}
    float* ml;             // workspace: [CTAs][2][rows of a tile][2] reference (base 2) and sum of a piece
    float* acc;            // workspace: [CTAs][2][rows of a tile][128]
};
constexpr int kAttendCtas = 296;  // 2 per SM with tiles of up to 16 rows; half as many with tiles of 32
int attend_tiles(int rows);

// Raise a kernel's shared-memory limit, once per device and kernel: `done` is that kernel's.  (Two threads may both set
// it; they set the same.)
struct SmemLimit {
    bool done[64] = {};
    template <typename K>
    bool raise(K* kernel, int bytes) {
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
        if (done[dev]) return true;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
        return done[dev] = true;
    }
};

int launch_cache_append(const CacheAppendArgs& p, cudaStream_t stream);
int launch_cache_attend(const CacheAttendArgs& p, cudaStream_t stream);
int launch_linear_decode(const LinearDecodeArgs& p, cudaStream_t stream);
int launch_linear_prefill(const LinearPrefillArgs& p, cudaStream_t stream);

}  // namespace gdn
