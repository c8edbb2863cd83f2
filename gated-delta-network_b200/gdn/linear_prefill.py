"""Linear attention with a decay for each head on B200: packed prompts, chunked.

The recurrence of ``gdn.linear_decode`` over every token of N packed sequences, with the tensors and the
k-last fp32 state of ``gdn.prefill``.  The reference has no such operator.  ``cu_seqlens`` is read on the
device only, so a call can be captured into a CUDA graph; calls that can overlap need workspaces of their
own (the default one comes from the torch caching allocator, for the current stream).
"""
from __future__ import annotations

import torch

from . import _lib
from ._common import (HEAD_DIM, NUM_QK_HEADS, NUM_V_HEADS, as_dev, call, check_heads, cu_on_device, cuda_device,
                      decay_rows, out_ok, ptr, resolve_scale, stream_handle, workspace_for)
from .prefill import read_status  # noqa: F401  (the status word is the workspace's first int here too)


def workspace_bytes(num_seqs: int, total_tokens: int, num_qk_heads: int = NUM_QK_HEADS,
                    num_v_heads: int = NUM_V_HEADS) -> int:
    return int(_lib.load().gdn_linear_prefill_workspace_bytes(int(num_seqs), int(total_tokens), int(num_qk_heads),
                                                              int(num_v_heads), HEAD_DIM, HEAD_DIM))


def _launch(dev, q, k, v, state, log_decay, cu_seqlens, scale, output, new_state, workspace, flags):
    """`output` / `new_state` None: allocated here and returned."""
    qs, vs = q.shape, v.shape
    if len(qs) != 3 or len(vs) != 3 or k.shape != qs or vs[0] != qs[0]:
        raise ValueError(f"q, k must be [T, H, 128] and v [T, HV, 128] (got {tuple(qs)}, {tuple(k.shape)}, {tuple(vs)})")
    T, H, K = qs
    HV, V = vs[1], vs[2]
    check_heads(H, H, HV, K, V, prefill=True)
    cu, cu64, N = cu_on_device(cu_seqlens, dev)
    s = scale if type(scale) is float and scale != 0.0 else resolve_scale(scale)
    q_ = as_dev(q, torch.bfloat16, dev)
    k_ = as_dev(k, torch.bfloat16, dev)
    v_ = as_dev(v, torch.bfloat16, dev)
    d_, per_token = decay_rows(log_decay, T, HV, dev)
    st = None
    if state is not None:
        if state.shape != (N, HV, V, K):
            raise ValueError(f"state must be [N, {HV}, 128, 128], got {tuple(state.shape)}")
        st = as_dev(state, torch.float32, dev)
    if output is None:
        output = torch.empty_like(v_)
        new_state = torch.empty((N, HV, V, K), dtype=torch.float32, device=dev) if st is None else torch.empty_like(st)
    else:
        if not out_ok(output, dev, torch.bfloat16, T * HV * V) or output.data_ptr() % 16:
            raise ValueError(f"output must be a contiguous, 16-byte aligned bf16 CUDA tensor with {T * HV * V} elements")
        if not out_ok(new_state, dev, torch.float32, N * HV * V * K) or new_state.data_ptr() % 16:
            raise ValueError(f"new_state must be a contiguous, 16-byte aligned fp32 CUDA tensor with {N * HV * V * K} elements")
    lib = _lib.load()
    need = lib.gdn_linear_prefill_workspace_bytes(N, T, H, HV, K, V)
    ws = workspace_for(workspace, need, dev)
    rc = call(dev, lib.gdn_linear_prefill_fwd, q_.data_ptr(), k_.data_ptr(), v_.data_ptr(), ptr(st), d_.data_ptr(), per_token,
              cu.data_ptr(), cu64, N, T, s, output.data_ptr(), new_state.data_ptr(), ws.data_ptr(), need, H, HV, K, V,
              stream_handle(dev), flags)
    if rc:
        _lib.check("gdn_linear_prefill_fwd", rc)
    return output, new_state


def run(q, k, v, state, log_decay, cu_seqlens, scale):
    """Packed prefill.  Returns ``(output [T,HV,128] bf16, new_state [N,HV,128,128] fp32)``.

    q, k [T,H,128] bf16; v [T,HV,128] bf16, HV a multiple of H (v-head hv reads q/k head hv // (HV // H));
    state [N,HV,128,128] fp32 or None (zeros); log_decay fp32, <= 0, either [HV] (one decay for each head) or
    [T,HV] (one for each token and head; -inf forgets a finite state before the token); cu_seqlens [N+1]
    int32/int64; scale float, 0-d tensor, or None/0 (1/sqrt(128)).  A value of v that is not finite makes its V
    column of the head NaN from its token on, in the outputs and the state; earlier tokens keep theirs.  A zero-length sequence keeps its state;
    tokens outside every sequence get a zero output.
    """
    return _launch(cuda_device(q, "q"), q, k, v, state, log_decay, cu_seqlens, scale, None, None, None,
                   _lib.GDN_FLAG_ZERO_UNOWNED)


def kernel(q, k, v, state, log_decay, cu_seqlens, scale, output, new_state, *, workspace=None):
    """Destination-passing prefill: writes ``new_state`` (which may be ``state`` itself) and the rows of
    ``output`` that belong to a sequence; the others are left as they were.  ``workspace``: a CUDA buffer of at
    least ``workspace_bytes(N, T, H, HV)`` bytes, 256-byte aligned, for callers that keep one; ``read_status`` of it tells
    whether the call went well (a call without a sequence leaves the status as it was)."""
    if output is None or new_state is None:
        raise ValueError("output and new_state must be given")
    _launch(cuda_device(q, "q"), q, k, v, state, log_decay, cu_seqlens, scale, output, new_state, workspace, 0)
