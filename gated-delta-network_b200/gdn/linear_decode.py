"""Linear attention with a decay for each head on B200: one token per sequence.

The recurrence of ``gdn.decode`` without beta and without the delta correction, on the same tensors and
the same k-last fp32 state: ``S' = e^a S + v k^T``, ``out = scale S' q``.  The reference has no such operator.
Both entry points call ``gdn_linear_decode_fwd`` of libgdn_b200.so on the current CUDA stream; nothing
synchronises the host unless ``scale`` is a CUDA tensor.
"""
from __future__ import annotations

import torch

from . import _lib
from ._common import as_dev, call, check_heads, cuda_device, decay_rows, out_ok, ptr, resolve_scale, stream_handle


def _launch(dev, q, k, v, state, log_decay, scale, output, new_state):
    """`output` / `new_state` None: allocated here and returned."""
    qs, vs = q.shape, v.shape
    if len(qs) != 4 or len(vs) != 4 or qs[1] != 1 or k.shape != qs or vs[:2] != qs[:2]:
        raise ValueError(f"q, k must be [B, 1, H, 128] and v [B, 1, HV, 128] (got {tuple(qs)}, {tuple(k.shape)}, "
                         f"{tuple(vs)})")
    B, _, H, K = qs
    HV, V = vs[2], vs[3]
    check_heads(H, H, HV, K, V)
    s = scale if type(scale) is float and scale != 0.0 else resolve_scale(scale)
    q_ = as_dev(q, torch.bfloat16, dev)
    k_ = as_dev(k, torch.bfloat16, dev)
    v_ = as_dev(v, torch.bfloat16, dev)
    d_, per_token = decay_rows(log_decay, B, HV, dev)
    st = None
    if state is not None:
        if state.shape != (B, HV, V, K):
            raise ValueError(f"state must be [B, {HV}, 128, 128], got {tuple(state.shape)}")
        st = as_dev(state, torch.float32, dev)
    if output is None:
        output = torch.empty_like(v_)
        new_state = torch.empty((B, HV, V, K), dtype=torch.float32, device=dev) if st is None else torch.empty_like(st)
    else:
        if not out_ok(output, dev, torch.bfloat16, B * HV * V) or output.data_ptr() % 16:
            raise ValueError(f"output must be a contiguous, 16-byte aligned bf16 CUDA tensor with {B * HV * V} elements")
        if not out_ok(new_state, dev, torch.float32, B * HV * V * K) or new_state.data_ptr() % 16:
            raise ValueError(f"new_state must be a contiguous, 16-byte aligned fp32 CUDA tensor with {B * HV * V * K} elements")
    rc = call(dev, _lib.load().gdn_linear_decode_fwd, q_.data_ptr(), k_.data_ptr(), v_.data_ptr(), ptr(st), d_.data_ptr(),
              per_token, s, output.data_ptr(), new_state.data_ptr(), B, H, HV, K, V, stream_handle(dev), 0)
    if rc:
        _lib.check("gdn_linear_decode_fwd", rc)
    return output, new_state


def run(q, k, v, state, log_decay, scale):
    """One step.  Returns ``(output [B,1,HV,128] bf16, new_state [B,HV,128,128] fp32)``.

    q, k [B,1,H,128] bf16; v [B,1,HV,128] bf16, HV a multiple of H (v-head hv reads q/k head
    hv // (HV // H)); state [B,HV,128,128] fp32 (k-last) or None (zeros); log_decay fp32, <= 0, either [HV]
    (one decay for each head) or [B,1,HV] (one for each sequence and head; -inf forgets a finite state);
    scale float, 0-d tensor, or None/0 (1/sqrt(128)).
    """
    return _launch(cuda_device(q, "q"), q, k, v, state, log_decay, scale, None, None)


def kernel(q, k, v, state, log_decay, scale, output, new_state):
    """Destination-passing step: writes ``output`` and ``new_state`` (which may be ``state`` itself)."""
    if output is None or new_state is None:
        raise ValueError("output and new_state must be given")
    _launch(cuda_device(q, "q"), q, k, v, state, log_decay, scale, output, new_state)
