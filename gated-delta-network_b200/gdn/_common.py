"""Argument normalisation shared by the decode and prefill entry points."""
from __future__ import annotations

import contextlib
import math

import torch

NUM_QK_HEADS = 4
NUM_V_HEADS = 8
HEAD_DIM = 128


def resolve_scale(scale) -> float:
    """None / 0 -> 1/sqrt(128) (reference/gdn_decode_ref.py:38-39); 0-d tensors -> .item()
    (solutions/gdn_decode_qk4_v8_d128_k_last/solution/triton/kernel.py:92-93)."""
    if isinstance(scale, torch.Tensor):
        scale = scale.item()
    if scale is None or float(scale) == 0.0:
        return 1.0 / math.sqrt(HEAD_DIM)
    return float(scale)


def check_heads(Hq: int, Hk: int, HV: int, K: int, V: int, prefill: bool = False) -> None:
    """The reference asserts 4 q/k heads, 8 v-heads and head size 128
    (reference/gdn_decode_ref.py:32-36, reference/gdn_prefill_ref.py:33-36).  This library
    accepts any head counts with HV a multiple of H (v-head hv reads q/k head hv // (HV // H));
    the head size stays 128."""
    if Hk != Hq:
        raise ValueError(f"q and k must have the same number of heads (got {Hq} and {Hk})")
    if K != HEAD_DIM or V != HEAD_DIM:
        raise ValueError(f"head size must be {HEAD_DIM} (got K={K}, V={V})")
    if not (1 <= Hq <= HV and HV % Hq == 0):
        raise ValueError(f"v-heads must be a multiple of the q/k heads (got H={Hq}, HV={HV})")


def cuda_device(t: torch.Tensor, name: str) -> torch.device:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be a CUDA tensor (got {t.device}); there is no CPU path")
    return t.device


def as_dev(t: torch.Tensor, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """Contiguous, 16-byte aligned tensor of `dtype` on `device` (copies only when needed: the
    library reads its inputs with TMA tile copies, which need 16-byte aligned bases)."""
    if (t.dtype is dtype and t.is_cuda and t.get_device() == device.index and t.is_contiguous()
            and not t.data_ptr() & 15):
        return t  # the common case: nothing to convert (checked with cheap attribute reads)
    if t.device != device or t.dtype != dtype:
        t = t.to(device=device, dtype=dtype)
    t = t.contiguous()
    if t.data_ptr() % 16:
        t = t.clone()
    return t


def ptr(t):
    return None if t is None else t.data_ptr()


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream_handle(device: torch.device) -> int:
    """cudaStream_t of the current torch stream on `device`."""
    if _raw_stream is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def on_device(device: torch.device):
    """Make `device` current for the library call (a no-op context when it already is)."""
    if torch.cuda.current_device() == device.index:
        return contextlib.nullcontext()
    return torch.cuda.device(device)


_get_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def call(device: torch.device, fn, *args) -> int:
    """fn(*args) with `device` current; no context object when it already is."""
    if _get_device() == device.index:
        return fn(*args)
    with torch.cuda.device(device):
        return fn(*args)


def out_ok(t, device: torch.device, dtype: torch.dtype, numel: int) -> bool:
    return (isinstance(t, torch.Tensor) and t.is_cuda and t.get_device() == device.index and t.dtype is dtype
            and t.is_contiguous() and t.numel() == numel)


def decay_rows(log_decay, rows: int, HV: int, device: torch.device):
    """(fp32 log decays on `device`, 1 if they hold a row for each token else 0): [HV] or [rows, (1,) HV]."""
    if not isinstance(log_decay, torch.Tensor):
        raise TypeError("log_decay must be a torch.Tensor")
    shape = log_decay.shape
    if len(shape) == 1 and shape[0] == HV:
        per_token = 0
    elif len(shape) in (2, 3) and shape[0] == rows and shape[-1] == HV and log_decay.numel() == rows * HV:
        per_token = 1
    else:
        raise ValueError(f"log_decay must hold [{HV}] or [{rows}, {HV}] values (got {tuple(shape)})")
    return as_dev(log_decay, torch.float32, device), per_token


def cu_on_device(cu_seqlens, device: torch.device):
    """(contiguous cu_seqlens on `device`, 1 if int64 else 0, number of sequences)."""
    if not isinstance(cu_seqlens, torch.Tensor) or cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1:
        raise ValueError("cu_seqlens must be a tensor of at least one element")
    if cu_seqlens.dtype not in (torch.int32, torch.int64):
        raise ValueError("cu_seqlens must be int32 or int64")
    cu = cu_seqlens if (cu_seqlens.is_cuda and cu_seqlens.get_device() == device.index) else cu_seqlens.to(device)
    return cu.contiguous(), 1 if cu.dtype == torch.int64 else 0, cu_seqlens.shape[0] - 1


def workspace_for(workspace, need: int, device: torch.device) -> torch.Tensor:
    """The caller's workspace after its checks, or one from the caching allocator (for the current stream)."""
    if workspace is None:
        return torch.empty(max(need, 1), dtype=torch.uint8, device=device)
    if (not isinstance(workspace, torch.Tensor) or not workspace.is_cuda or workspace.get_device() != device.index
            or not workspace.is_contiguous() or workspace.numel() * workspace.element_size() < need
            or workspace.data_ptr() % 256):
        raise ValueError(f"workspace must be a contiguous, 256-byte aligned CUDA buffer of at least {need} bytes")
    return workspace


CODES = {torch.int8: 0, torch.float8_e4m3fn: 1}  # GDN_CODE_*
PAGE_SIZES = (16, 32, 64, 128)


def cache_tensors(k_cache, v_cache, k_scale, v_scale, device: torch.device):
    """Checks of a paged 8-bit cache, which is used in place; returns (code, pages, Hkv, page size)."""
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if (not isinstance(t, torch.Tensor) or not t.is_cuda or t.get_device() != device.index or t.dtype not in CODES
                or t.dim() != 4 or t.shape[3] != HEAD_DIM or not t.is_contiguous() or t.data_ptr() & 15):
            raise ValueError(f"{name} must be a contiguous, 16-byte aligned int8 or float8_e4m3fn CUDA tensor "
                             f"[pages, heads, page_size, {HEAD_DIM}]")
    shape, dtype = k_cache.shape, k_cache.dtype
    if v_cache.shape != shape or v_cache.dtype is not dtype:
        raise ValueError("k_cache and v_cache must have the same shape and type")
    pages, Hkv, P, _ = shape
    if P not in PAGE_SIZES:
        raise ValueError(f"page size must be one of {PAGE_SIZES} (got {P})")
    want = shape[:2]
    for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
        if (not isinstance(t, torch.Tensor) or t.dtype is not torch.float32 or not t.is_cuda
                or t.get_device() != device.index or t.shape != want or not t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous fp32 CUDA tensor [{pages}, {Hkv}]")
    return CODES[dtype], pages, Hkv, P


def cache_rows(block_table, seq_lens, B: int, device: torch.device):
    """(int32 block table, sequence lengths, 1 if those are int64 else 0, pages of a row), on `device`."""
    if not isinstance(block_table, torch.Tensor) or block_table.dim() != 2 or block_table.shape[0] != B:
        raise ValueError(f"block_table must be a tensor [{B}, max_pages]")
    if block_table.dtype not in (torch.int32, torch.int64):
        raise ValueError("block_table must be int32 or int64")
    if not isinstance(seq_lens, torch.Tensor) or seq_lens.dim() != 1 or seq_lens.shape[0] != B:
        raise ValueError(f"seq_lens must be a tensor [{B}]")
    if seq_lens.dtype not in (torch.int32, torch.int64):
        raise ValueError("seq_lens must be int32 or int64")
    table = as_dev(block_table, torch.int32, device)
    lens = as_dev(seq_lens, seq_lens.dtype, device)
    return table, lens, 1 if lens.dtype is torch.int64 else 0, table.shape[1]
