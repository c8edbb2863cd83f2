"""Linear attention with a decay for each head, token by token in 64 bits, and the error that the kernels may make."""
from __future__ import annotations

import torch

D = 128
U_BF16 = 2.0 ** -8  # half a step of bf16, relative to the value


def reference(q, k, v, state, log_decay, cu, scale):
    """(out [T,HV,128], state [N,HV,128,128], and for each the sum of the magnitudes of its terms), float64, CPU or GPU.

    Rows of tokens outside every sequence are zero.  The magnitudes follow the same recurrence on absolute values:
    they bound every partial sum, so a rounding of any intermediate to `u` moves a result by at most u times them.
    """
    q, k, v = (x.double() for x in (q, k, v))
    T, HV = v.shape[:2]
    group = HV // q.shape[1]
    q, k = q.repeat_interleave(group, 1), k.repeat_interleave(group, 1)
    a = log_decay.double().reshape(-1, HV).expand(T, HV)
    N = len(cu) - 1
    S = torch.zeros((N, HV, D, D), dtype=torch.float64, device=v.device) if state is None else state.double().clone()
    A = S.abs()
    out = torch.zeros_like(v)
    mag = torch.zeros_like(v)
    for n in range(N):
        for t in range(cu[n], cu[n + 1]):
            g = a[t].exp()[:, None, None]
            S[n] = g * S[n] + v[t][:, :, None] * k[t][:, None, :]
            A[n] = g * A[n] + v[t].abs()[:, :, None] * k[t].abs()[:, None, :]
            out[t] = scale * (S[n] @ q[t][:, :, None])[..., 0]
            mag[t] = abs(scale) * (A[n] @ q[t].abs()[:, :, None])[..., 0]
    return out, S, mag, A


def check(out, new_state, ref, chunked):
    """Every element within the sum of its roundings.

    Output: one rounding to bf16 at the end, and in the chunked form one of the state copy or of the decayed
    products before it, each u = 2^-8 of the terms' magnitudes (2 u covers both and the fp32 sums).  State: fp32
    sums, and in the chunked form the decayed v as bf16 parts, two of which are u^2 = 2^-16 off; 2^-15 covers that,
    the fp32 sums of up to 64 terms and of the chunks, and the decays (a prefix sum of at most 20 where the decay
    matters, so 20 * 2^-23 relative).
    """
    o, S, mag, A = ref
    e = (out.double() - o).abs()
    bound = U_BF16 * o.abs() + (1.05 * U_BF16 if chunked else 2.0 ** -18) * mag + 1e-30
    assert torch.isfinite(out.float()).all()
    assert (e <= bound).all(), f"output off by {(e / bound).max().item():.2f} times its bound"
    if new_state is not None:
        e = (new_state.double() - S).abs()
        bound = (2.0 ** -15 if chunked else 2.0 ** -20) * A + 1e-30
        assert torch.isfinite(new_state).all()
        assert (e <= bound).all(), f"state off by {(e / bound).max().item():.2f} times its bound"


def inputs(lens, H=4, HV=8, seed=0, per_token=True, with_state=True, device="cuda", lead=0, tail=0):
    """q, k, v, state, log_decay, cu (list): tokens of `lens`, with `lead` / `tail` rows outside every sequence."""
    g = torch.Generator().manual_seed(seed)
    T = lead + sum(lens) + tail
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    q, k, v = (x.to(torch.bfloat16).to(device) for x in (r(T, H, D) * 0.3, r(T, H, D) * 0.3, r(T, HV, D)))
    state = (r(len(lens), HV, D, D) * 0.1).to(device) if with_state else None
    slope = -torch.exp2(-6.0 * torch.rand((HV,), generator=g))
    decay = (slope * 2 * torch.rand((T, HV), generator=g) if per_token else slope).to(device)
    cu = [lead]
    for n in lens:
        cu.append(cu[-1] + n)
    return q, k, v, state, decay, cu
