// linear_decode.cu -- one token of linear attention with a decay for each head, one pass over the
// k-last fp32 state.  For each (sequence b, v-head hv), q and k from q/k head hv / (HV / H):
//   g = exp(decay),   S'[v] = g S[v] + v[v] k,   out[v] = scale S'[v]·q = scale (g S[v]·q + v[v] (k·q))
// so one reduction per state row, taken from the old row, serves the readout.
//
// Bound by HBM: 128 KB of state traffic per head against 82 K fp32 operations.  Mapping as in decode.cu:
// 8 lanes share a 512-byte state row (four float4 each, every load instruction of a warp covers four
// full 128-byte lines), every element is read and written by one thread, so new_state may alias state,
// and all state loads are issued before any arithmetic.  A CTA takes 16 rows, one a lane: 250 x 32 heads in 152.6 us
// (6.9 TB/s), 64 x 8 in 11.0, 1 x 8 in 2.1; with two rows a lane 154.5, 11.3 and 2.4.
#include "common.cuh"
#include "linear.cuh"

namespace gdn {

constexpr int kThreads = 128, kRowsPerCta = 16, kSlices = kD / kRowsPerCta;

__global__ void __launch_bounds__(kThreads) gdn_linear_decode_kernel(LinearDecodeArgs p) {
    const int lane = threadIdx.x & 31;
    const int warp = threadIdx.x >> 5;
    const int j = lane & 7;     // position inside the row group
    const int rsub = lane >> 3; // row inside the warp's 4-row group
    const int slice = blockIdx.x % kSlices;
    const int bh = blockIdx.x / kSlices;
    const int bi = bh / p.HV, hv = bh % p.HV, hq = hv / (p.HV / p.H);
    const size_t head_off = (size_t)bh * kD * kD;
    const int row = slice * kRowsPerCta + warp * 4 + rsub;

    pdl_wait();  // everything above overlapped the previous kernel's tail
    float4 S[4];
    const float* src = p.state + head_off + (size_t)row * kD + 4 * j;
#pragma unroll
    for (int i = 0; i < 4; ++i) S[i] = p.state != nullptr ? ld_stream_f4(src + 32 * i) : make_float4(0.f, 0.f, 0.f, 0.f);
    pdl_trigger();

    float qf[16], kf[16];
    const uint16_t* qp = p.q + ((size_t)bi * p.H + hq) * kD + 4 * j;
    const uint16_t* kp = p.k + ((size_t)bi * p.H + hq) * kD + 4 * j;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint2 qq = ld_nc_u2(qp + 32 * i), kk = ld_nc_u2(kp + 32 * i);
        qf[4 * i + 0] = __uint_as_float(qq.x << 16);
        qf[4 * i + 1] = __uint_as_float(qq.x & 0xffff0000u);
        qf[4 * i + 2] = __uint_as_float(qq.y << 16);
        qf[4 * i + 3] = __uint_as_float(qq.y & 0xffff0000u);
        kf[4 * i + 0] = __uint_as_float(kk.x << 16);
        kf[4 * i + 1] = __uint_as_float(kk.x & 0xffff0000u);
        kf[4 * i + 2] = __uint_as_float(kk.y << 16);
        kf[4 * i + 3] = __uint_as_float(kk.y & 0xffff0000u);
    }
    const float g = expf(p.decay[p.per_token ? bh : hv]);
    float kq = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) kq = fmaf(kf[e], qf[e], kq);
#pragma unroll
    for (int off = 1; off < 8; off <<= 1) kq += __shfl_xor_sync(0xffffffffu, kq, off);

    const float vr = bf2f(p.v[(size_t)bh * kD + row]);
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        sq = fmaf(S[i].x, qf[4 * i + 0], sq);
        sq = fmaf(S[i].y, qf[4 * i + 1], sq);
        sq = fmaf(S[i].z, qf[4 * i + 2], sq);
        sq = fmaf(S[i].w, qf[4 * i + 3], sq);
    }
#pragma unroll
    for (int off = 1; off < 8; off <<= 1) sq += __shfl_xor_sync(0xffffffffu, sq, off);
    float* dst = p.new_state + head_off + (size_t)row * kD + 4 * j;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float4 s = S[i];
        s.x = fmaf(g, s.x, vr * kf[4 * i + 0]);
        s.y = fmaf(g, s.y, vr * kf[4 * i + 1]);
        s.z = fmaf(g, s.z, vr * kf[4 * i + 2]);
        s.w = fmaf(g, s.w, vr * kf[4 * i + 3]);
        st_stream_f4(dst + 32 * i, s);
    }
    if (j == 0) p.out[(size_t)bh * kD + row] = f2bf(p.scale * fmaf(g, sq, vr * kq));
}

int launch_linear_decode(const LinearDecodeArgs& p, cudaStream_t stream) {
    const dim3 grid((unsigned)((long long)p.B * p.HV * kSlices));
    return launch_pdl(gdn_linear_decode_kernel, grid, dim3(kThreads), 0, stream, p) == cudaSuccess ? 0 : -1;
}

}  // namespace gdn
