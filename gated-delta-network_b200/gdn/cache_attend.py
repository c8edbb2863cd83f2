"""Attention of the newest tokens over a paged cache of 8-bit codes with a scale for each page and head, on B200.

The softmax layers of a stack whose other layers are ``gdn.decode`` or ``gdn.linear_decode``: one call attends the
last Q tokens of every sequence (Q = 1: the decode step) over what ``gdn.cache_append`` wrote.  The reference has
no such operator.  Lengths are read on the device only, so a call can be captured into a CUDA graph; calls that
can overlap need workspaces of their own (the default one comes from the torch caching allocator, for the current
stream).
"""
from __future__ import annotations

import torch

from . import _lib
from ._common import (HEAD_DIM, as_dev, cache_rows, cache_tensors, call, cuda_device, out_ok, resolve_scale,
                      stream_handle, workspace_for)
from .prefill import read_status  # noqa: F401  (the status word is the workspace's first int here too)


_need = 0  # the library's answer, which does not change


def workspace_bytes() -> int:
    global _need
    if not _need:
        _need = int(_lib.load().gdn_cache_attend_workspace_bytes())
    return _need


def _launch(dev, q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, scale, output, workspace):
    """`output` None: allocated here and returned."""
    code, pages, Hkv, P = cache_tensors(k_cache, v_cache, k_scale, v_scale, dev)
    qs = q.shape
    if len(qs) != 4 or qs[3] != HEAD_DIM:
        raise ValueError(f"q must be [B, Q, Hq, {HEAD_DIM}] (got {tuple(qs)})")
    B, Q, Hq, _ = qs
    if Hkv < 1 or Hq < Hkv or Hq % Hkv:
        raise ValueError(f"q heads must be a multiple of the cache's heads (got {Hq} and {Hkv})")
    table, lens, len64, max_pages = cache_rows(block_table, seq_lens, B, dev)
    s = scale if type(scale) is float and scale != 0.0 else resolve_scale(scale)
    q_ = as_dev(q, torch.bfloat16, dev)
    if output is None:
        output = torch.empty_like(q_)
    elif not out_ok(output, dev, torch.bfloat16, q.numel()) or output.data_ptr() % 16:
        raise ValueError(f"output must be a contiguous, 16-byte aligned bf16 CUDA tensor with {q.numel()} elements")
    lib = _lib.load()
    need = _need or workspace_bytes()
    ws = workspace_for(workspace, need, dev)
    rc = call(dev, lib.gdn_cache_attend, q_.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(),
              v_scale.data_ptr(), code, table.data_ptr(), lens.data_ptr(), len64, pages, P, max_pages, B, Q, Hq, Hkv, HEAD_DIM,
              s, output.data_ptr(), ws.data_ptr(), need, stream_handle(dev), 0)
    if rc:
        _lib.check("gdn_cache_attend", rc)
    return output


def kernel(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, scale, output, *, workspace=None):
    """Destination-passing form of ``run``: writes ``output`` [B, Q, Hq, 128] bf16.  ``workspace``: a CUDA buffer of
    at least ``workspace_bytes()`` bytes, 256-byte aligned, for callers that keep one; ``read_status`` of it tells whether
    the call went well (a call without a sequence or a q row leaves the status as it was)."""
    if output is None:
        raise ValueError("output must be given")
    _launch(cuda_device(q, "q"), q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, scale, output, workspace)


def run(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, scale):
    """Attention of the last Q tokens of every sequence.  Returns ``output [B, Q, Hq, 128] bf16``.

    q [B, Q, Hq, 128] bf16, the tokens already appended; k_cache, v_cache [pages, Hkv, page_size, 128] int8 or
    float8_e4m3fn, k_scale, v_scale [pages, Hkv] fp32 (see ``gdn.cache_append``), Hq a multiple of Hkv (q head h
    reads head h // (Hq // Hkv)); block_table [B, max_pages] int32 (int64 is converted); seq_lens [B] int32/int64,
    the Q tokens included.  Row i sees the positions below seq_len - Q + 1 + i; a row that sees none (a padded row
    with seq_lens 0, say) is zero.  What a row does not see cannot reach it, be it NaN; a NaN or infinite value that it
    sees makes that dim of it NaN or infinite.  scale float, 0-d tensor, or None/0 (1/sqrt(128)).
    """
    return _launch(cuda_device(q, "q"), q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, scale, None, None)
