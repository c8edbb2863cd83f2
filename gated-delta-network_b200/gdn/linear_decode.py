"""Linear attention with a decay for each head on B200: one token per sequence.

The recurrence of ``gdn.decode`` without beta and without the delta correction, on the same tensors and
the same k-last fp32 state: ``S' = e^a S + v k^T``, ``out = scale S' q``.  The reference has no such operator.
Both entry points call ``gdn_linear_decode_fwd`` of libgdn_b200.so on the current CUDA stream; nothing
synchronises the host unless ``scale`` is a CUDA tensor.
"""
from __future__ import annotations

import torch

from . import _lib
from ._common import HEAD_DIM, as_dev, check_heads, cuda_device, decay_rows, on_device, out_ok, ptr, resolve_scale, stream_handle


def _launch(q, k, v, state, log_decay, scale, output, new_state):
    dev = cuda_device(q, "q")
    if q.dim() != 4 or v.dim() != 4 or q.shape[1] != 1 or k.shape != q.shape or v.shape[:2] != q.shape[:2]:
        raise ValueError(f"q, k must be [B, 1, H, 128] and v [B, 1, HV, 128] (got {tuple(q.shape)}, "
                         f"{tuple(k.shape)}, {tuple(v.shape)})")
    B, _, H, K = q.shape
    HV, V = v.shape[2], v.shape[3]
    check_heads(H, k.shape[2], HV, K, V)
    s = resolve_scale(scale)
    q_ = as_dev(q, torch.bfloat16, dev)
    k_ = as_dev(k, torch.bfloat16, dev)
    v_ = as_dev(v, torch.bfloat16, dev)
    d_, per_token = decay_rows(log_decay, B, HV, dev)
    st = None
    if state is not None:
        if tuple(state.shape) != (B, HV, V, K):
            raise ValueError(f"state must be [B, {HV}, 128, 128], got {tuple(state.shape)}")
        st = as_dev(state, torch.float32, dev)
    if not out_ok(output, dev, torch.bfloat16, B * HV * V) or output.data_ptr() % 16:
        raise ValueError(f"output must be a contiguous, 16-byte aligned bf16 CUDA tensor with {B * HV * V} elements")
    if not out_ok(new_state, dev, torch.float32, B * HV * V * K) or new_state.data_ptr() % 16:
        raise ValueError(f"new_state must be a contiguous, 16-byte aligned fp32 CUDA tensor with {B * HV * V * K} elements")
    lib = _lib.load()
    with on_device(dev):
        rc = lib.gdn_linear_decode_fwd(ptr(q_), ptr(k_), ptr(v_), ptr(st), ptr(d_), per_token, s, ptr(output),
                                       ptr(new_state), B, H, HV, K, V, stream_handle(dev), 0)
    _lib.check("gdn_linear_decode_fwd", rc)


def run(q, k, v, state, log_decay, scale):
    """One step.  Returns ``(output [B,1,HV,128] bf16, new_state [B,HV,128,128] fp32)``.

    q, k [B,1,H,128] bf16; v [B,1,HV,128] bf16, HV a multiple of H (v-head hv reads q/k head
    hv // (HV // H)); state [B,HV,128,128] fp32 (k-last) or None (zeros); log_decay fp32, <= 0, either [HV]
    (one decay for each head) or [B,1,HV] (one for each sequence and head; -inf forgets the state);
    scale float, 0-d tensor, or None/0 (1/sqrt(128)).
    """
    dev = cuda_device(q, "q")
    if v.dim() != 4:
        raise ValueError(f"v must be [B, 1, HV, 128] (got {tuple(v.shape)})")
    B, HV = q.shape[0], v.shape[2]
    output = torch.empty((B, 1, HV, HEAD_DIM), dtype=torch.bfloat16, device=dev)
    new_state = torch.empty((B, HV, HEAD_DIM, HEAD_DIM), dtype=torch.float32, device=dev)
    _launch(q, k, v, state, log_decay, scale, output, new_state)
    return output, new_state


def kernel(q, k, v, state, log_decay, scale, output, new_state):
    """Destination-passing step: writes ``output`` and ``new_state`` (which may be ``state`` itself)."""
    _launch(q, k, v, state, log_decay, scale, output, new_state)
