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
    int m;                 // chunks per segment
    int slots;             // work items per v-head: T / (64 m) + N
    int states;            // state slots: 2 (T / (64 m))
    int cut;               // a sequence can be longer than one segment: build and chain segment states
    int* status;           // workspace: first error code of a bounded wait
    float* gamma;          // workspace: [states][HV] product of a segment's decays
    float* seg;            // workspace: [states][HV][128 V][128 K] what a segment adds to the state, then
                           //            (after the chain) the state at its end
};

struct LinearPrefillLayout {
    int m, slots, states, cut;
    size_t off_status, off_gamma, off_seg, total;
};
LinearPrefillLayout linear_prefill_layout(int N, int T, int HV);

int launch_linear_decode(const LinearDecodeArgs& p, cudaStream_t stream);
int launch_linear_prefill(const LinearPrefillArgs& p, cudaStream_t stream);

}  // namespace gdn
