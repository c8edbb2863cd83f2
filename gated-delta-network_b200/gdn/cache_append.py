"""New keys and values into a paged cache of 8-bit codes with a scale for each page and head, on B200.

The cache is what ``gdn.cache_attend`` reads: ``k_cache``, ``v_cache`` [pages, Hkv, page_size, 128] int8 or
float8_e4m3fn and ``k_scale``, ``v_scale`` [pages, Hkv] fp32, a value being code * scale.  The reference has no
such operator.  Nothing is copied to the host, so a call can be captured into a CUDA graph.
"""
from __future__ import annotations

import torch

from . import _lib
from ._common import HEAD_DIM, as_dev, cache_rows, cache_tensors, call, cu_on_device, cuda_device, stream_handle


def kernel(k, v, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, cu_seqlens):
    """Writes the new rows, in place.

    k, v [T, Hkv, 128] bf16, packed by cu_seqlens [B+1] (int32/int64); block_table [B, max_pages] int32 (int64 is
    converted): page i of a sequence holds its tokens from i * page_size on (page_size 16, 32, 64 or 128);
    seq_lens [B] int32/int64: tokens of each sequence, the new ones included, so the n rows of a sequence become
    its last n tokens.

    Every (page, head) written to gets ``scale = max(scale before, max |x| / m)``, m = 127 (int8) or 448 (e4m3),
    from 0 if the page's first token is among the new ones; its older tokens are re-encoded if the scale grew.
    Codes are round(x / scale), ties to even; infinities become the largest code, a NaN a NaN (e4m3) or 0 (int8),
    and neither enters the scale.  Slots behind a sequence's last token stay as they were.  Rows before position 0
    (a padded row with seq_lens 0, say), beyond the block table or in a page outside the cache are dropped.  Two
    sequences must not write to one page in one call.

    Re-encoding rounds again, so tokens appended one by one come out less exact than in one call: for normal rows in
    pages of 64, 0.38 int8 steps rms instead of 0.29 (2.3 at most instead of 0.5), e4m3 3.5% rms instead of 2.6%.
    """
    dev = cuda_device(k, "k")
    code, pages, Hkv, P = cache_tensors(k_cache, v_cache, k_scale, v_scale, dev)
    ks = k.shape
    if len(ks) != 3 or ks[1] != Hkv or ks[2] != HEAD_DIM or not isinstance(v, torch.Tensor) or v.shape != ks:
        raise ValueError(f"k and v must be [T, {Hkv}, {HEAD_DIM}] tensors of one shape")
    cu, cu64, B = cu_on_device(cu_seqlens, dev)
    table, lens, len64, max_pages = cache_rows(block_table, seq_lens, B, dev)
    k_ = as_dev(k, torch.bfloat16, dev)
    v_ = as_dev(v, torch.bfloat16, dev)
    rc = call(dev, _lib.load().gdn_cache_append, k_.data_ptr(), v_.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
              k_scale.data_ptr(), v_scale.data_ptr(), code, table.data_ptr(), lens.data_ptr(), len64, cu.data_ptr(), cu64,
              pages, P, max_pages, B, k.shape[0], Hkv, HEAD_DIM, stream_handle(dev), 0)
    if rc:
        _lib.check("gdn_cache_append", rc)
