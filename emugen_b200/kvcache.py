"""Quantised key/value cache: rows (token, head) written to their slots in 8 or 4 bits, read back, and attended to.

A cache is four tensors (make_kv_cache): codes and scales of the keys and of the values, page by page:

  "fp8"     float8_e4m3fn [pages, page_size, heads, head_size], f32 scales [..., ceil(head_size / 128)]
            (emugen_b200.fp8's quantiser, blocks of 128 along a row)
  "mxfp4"   packed e2m1 uint8 [pages, page_size, heads, head_size / 2], scale bytes [..., head_size / 32]
            (quant_mxfp4's codes and exponents, without its swizzle)

attend_kv_cache is the attention of one new token for each sequence over its rows, read as they are stored.

Slot s is place s % page_size of page s // page_size.  The kernels run on the cache's device and its
current stream and synchronise nothing.  The reference has no cache.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .attention import _plain, _wants_grad
from .fp8 import _DTYPE, _on, _raw_stream


def make_kv_cache(num_pages: int, page_size: int, heads: int, head_size: int, fmt: str = "fp8", *,
                  values: bool = True, device: torch.device | str | int = "cuda"):
    """A cache of zeros: (k_cache, v_cache, k_scale, v_scale), the value tensors None without `values`."""
    if min(num_pages, page_size, heads, head_size) < 1:
        raise ValueError("num_pages, page_size, heads and head_size must be positive")
    lead = (num_pages, page_size, heads)
    if fmt == "fp8":
        if head_size % 16:
            raise ValueError("head_size must be a multiple of 16")
        code, scale = (head_size, torch.float8_e4m3fn), ((head_size + 127) // 128, torch.float32)
    elif fmt == "mxfp4":
        if head_size % 32:
            raise ValueError("head_size must be a multiple of 32")
        code, scale = (head_size // 2, torch.uint8), (head_size // 32, torch.uint8)
    else:
        raise ValueError(f"fmt must be 'fp8' or 'mxfp4', got {fmt!r}")

    def zeros(last):
        return torch.zeros((*lead, last[0]), dtype=torch.uint8 if last[1] == torch.float8_e4m3fn else last[1],
                           device=device).view(last[1])

    k, ks = zeros(code), zeros(scale)
    return (k, zeros(code), ks, zeros(scale)) if values else (k, None, ks, None)


def _geometry(k_cache, v_cache, k_scale, v_scale):
    """(format code, pages, page size, heads, head size) of a cache, after checking its tensors."""
    if k_cache.dim() != 4 or k_scale.dim() != 4:
        raise RuntimeError("cache tensors must be [pages, page_size, heads, ...]")
    if (v_cache is None) != (v_scale is None):
        raise RuntimeError("v_cache and v_scale go together")
    pages, page_size, heads, last = k_cache.shape
    if k_cache.dtype == torch.float8_e4m3fn:
        fmt, D, sd, sl = _lib.EMU_KV_FP8, last, torch.float32, (last + 127) // 128
    elif k_cache.dtype == torch.uint8:
        fmt, D, sd, sl = _lib.EMU_KV_MXFP4, 2 * last, torch.uint8, last // 16
    else:
        raise RuntimeError(f"cache must be float8_e4m3fn or uint8 (mxfp4), got {k_cache.dtype}")
    unit = 16 if fmt == _lib.EMU_KV_FP8 else 32
    if D < 1 or D % unit:
        raise RuntimeError(f"head_size must be a multiple of {unit}")
    want = (pages, page_size, heads, sl)
    if tuple(k_scale.shape) != want or k_scale.dtype != sd:
        raise RuntimeError(f"k_scale must be {sd} {list(want)}, got {k_scale.dtype} {list(k_scale.shape)}")
    if v_cache is not None:
        if v_cache.shape != k_cache.shape or v_cache.dtype != k_cache.dtype:
            raise RuntimeError("v_cache must have k_cache's shape and dtype")
        if v_scale.shape != k_scale.shape or v_scale.dtype != k_scale.dtype:
            raise RuntimeError("v_scale must have k_scale's shape and dtype")
    device = k_cache.get_device()
    for t in (k_cache, v_cache, k_scale, v_scale):
        if t is None:
            continue
        if not t.is_contiguous():
            raise RuntimeError("cache tensors must be contiguous")
        if device < 0 or t.get_device() != device:
            raise RuntimeError("cache tensors must be on one CUDA device")
    return fmt, pages, page_size, heads, D


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def write_kv_cache(k: torch.Tensor, v: Optional[torch.Tensor], slots: torch.Tensor, k_cache: torch.Tensor,
                   v_cache: Optional[torch.Tensor], k_scale: torch.Tensor, v_scale: Optional[torch.Tensor]) -> None:
    """Quantise k and v [tokens, heads, head_size] (fp16 / bf16; any token and head strides) into slots
    [tokens] int64 of the cache, in place.  A slot that is negative or past the cache writes nothing (padding);
    where several tokens have the same slot, the last one's row is kept.  v, v_cache and v_scale are None
    together for a cache of one tensor."""
    fmt, pages, page_size, heads, D = _geometry(k_cache, v_cache, k_scale, v_scale)
    dev = k_cache.device
    if (v is None) != (v_cache is None):
        raise RuntimeError("v and v_cache go together")
    if k.dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError(f"k and v must be float16 or bfloat16, got {k.dtype}")
    if k.dim() != 3 or tuple(k.shape[1:]) != (heads, D):
        raise RuntimeError(f"k must be [tokens, {heads}, {D}], got {list(k.shape)}")
    if v is not None and (v.shape != k.shape or v.dtype != k.dtype):
        raise RuntimeError("v must have k's shape and dtype")
    if slots.dtype != torch.int64 or slots.dim() != 1 or slots.shape[0] != k.shape[0]:
        raise RuntimeError(f"slots must be int64 [{k.shape[0]}], got {slots.dtype} {list(slots.shape)}")
    at = dev.index
    if k.get_device() != at or slots.get_device() != at or (v is not None and v.get_device() != at):
        raise RuntimeError("k, v and slots must be on the cache's device")
    if k.stride(2) != 1:
        k = k.contiguous()
    if v is not None and v.stride(2) != 1:
        v = v.contiguous()
    slots = slots.contiguous()
    L = _lib.load()
    with _on(dev.index):
        status = L.emu_kv_write(k.data_ptr(), _ptr(v), _DTYPE[k.dtype], k.shape[0], heads, D, k.stride(0), k.stride(1),
                                0 if v is None else v.stride(0), 0 if v is None else v.stride(1), slots.data_ptr(),
                                fmt, pages * page_size, k_cache.data_ptr(), _ptr(v_cache), k_scale.data_ptr(),
                                _ptr(v_scale), _raw_stream(dev.index))
    if status:
        _lib._check(status)


def read_kv_cache(k_cache: torch.Tensor, v_cache: Optional[torch.Tensor], k_scale: torch.Tensor,
                  v_scale: Optional[torch.Tensor], block_table: torch.Tensor, cu_lens: torch.Tensor, *,
                  total: Optional[int] = None, dtype: torch.dtype = torch.bfloat16, out=None):
    """The cached rows of a batch of sequences, packed: (k, v) [total, heads, head_size] of `dtype`.

    block_table int32 [sequences, pages of a sequence]; cu_lens int32 [sequences + 1], non-decreasing from 0:
    rows cu_lens[b] .. cu_lens[b + 1] are sequence b's positions from 0 on.  `total` rows are allocated (those that
    no sequence has are uninitialised), or `out` = (k, v) is written, whose rows behind the last sequence are left
    as they were.  Rows of a page that does not exist are zeros.  Without a value cache, v is None."""
    fmt, pages, page_size, heads, D = _geometry(k_cache, v_cache, k_scale, v_scale)
    dev = k_cache.device
    if block_table.dtype != torch.int32 or block_table.dim() != 2:
        raise RuntimeError(f"block_table must be int32 [sequences, pages], got {block_table.dtype} {list(block_table.shape)}")
    B, cols = block_table.shape
    if cu_lens.dtype != torch.int32 or cu_lens.dim() != 1 or cu_lens.shape[0] != B + 1:
        raise RuntimeError(f"cu_lens must be int32 [{B + 1}], got {cu_lens.dtype} {list(cu_lens.shape)}")
    if block_table.device != dev or cu_lens.device != dev:
        raise RuntimeError("block_table and cu_lens must be on the cache's device")
    if out is None:
        if total is None or total < 0:
            raise RuntimeError("read_kv_cache needs total (the number of rows) or out")
        if dtype not in _DTYPE:
            raise RuntimeError(f"dtype must be float16, bfloat16 or float32, got {dtype}")
        k_out = torch.empty((total, heads, D), dtype=dtype, device=dev)
        v_out = None if v_cache is None else torch.empty((total, heads, D), dtype=dtype, device=dev)
    else:
        k_out, v_out = out
        if (v_out is None) != (v_cache is None):
            raise RuntimeError("out must hold a tensor for each of the cache's")
        for t in (k_out, v_out):
            if t is None:
                continue
            if t.dim() != 3 or tuple(t.shape[1:]) != (heads, D) or t.shape[0] != k_out.shape[0]:
                raise RuntimeError(f"out must be [total, {heads}, {D}], got {list(t.shape)}")
            if t.dtype not in _DTYPE or t.dtype != k_out.dtype:
                raise RuntimeError("out must share one of float16, bfloat16, float32")
            if t.device != dev:
                raise RuntimeError("out must be on the cache's device")
            if t.shape[0] and (t.stride(2) != 1 and D > 1 or t.stride(1) != D and heads > 1 or
                               t.stride(0) < heads * D and t.shape[0] > 1):
                raise RuntimeError("out's rows must be contiguous and must not overlap")
        if total is not None and total != k_out.shape[0]:
            raise RuntimeError("total must be out's number of rows")
    total = k_out.shape[0]
    if block_table.stride(1) != 1 and cols > 1 or block_table.stride(0) < cols and B > 1:
        block_table = block_table.contiguous()
    cu_lens = cu_lens.contiguous()
    row = heads * D
    L = _lib.load()
    with _on(dev.index):
        status = L.emu_kv_read(k_cache.data_ptr(), _ptr(v_cache), k_scale.data_ptr(), _ptr(v_scale), fmt, pages, page_size,
                               heads, D, block_table.data_ptr(), B, cols, max(block_table.stride(0), cols),
                               cu_lens.data_ptr(), total, _DTYPE[k_out.dtype], k_out.data_ptr(), _ptr(v_out),
                               k_out.stride(0) if total > 1 else row,
                               0 if v_out is None else v_out.stride(0) if total > 1 else row, _raw_stream(dev.index))
    if status:
        _lib._check(status)
    return k_out, v_out


def attend_kv_cache(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                    v_scale: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor, *,
                    scale: Optional[float] = None, return_lse: bool = False):
    """Attention of one new token for each sequence over its cached rows: [sequences, query heads, head_size].

    q [sequences, query heads, head_size] (fp16 / bf16; any sequence and head strides); its heads are a multiple of the
    cache's, query head h reading the cache's head h // (query heads // heads).  lens int32 [sequences]: sequence b sees its
    positions 0 .. lens[b] - 1, from pages block_table[b] (int32 [sequences, pages of a sequence]); write the new token's
    own row first.  Positions on a page that does not exist are not seen, and a sequence that sees none gets zeros.
    scale: of the scores (default head_size ** -0.5).  With return_lse also f32 [sequences, query heads]: the logarithm of
    the sum of exp(score), -inf where nothing is seen.  head_size up to 256.  Scores, sums and the softmax in f32, the
    weights of the values rounded to fp16; the same result every run.  Not differentiable: a q that wants a gradient or has a
    forward-mode tangent is refused (torch.no_grad() or q.detach() around generation)."""
    if v_cache is None or v_scale is None:
        raise RuntimeError("attend_kv_cache needs a cache of keys and values")
    if _wants_grad(q, k_scale, v_scale):
        raise RuntimeError("attend_kv_cache is not differentiable: call it under torch.no_grad() or with detached tensors")
    _plain("attend_kv_cache", q, k_scale, v_scale)
    fmt, pages, page_size, heads, D = _geometry(k_cache, v_cache, k_scale, v_scale)
    dev = k_cache.device
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError(f"q must be float16 or bfloat16, got {q.dtype}")
    qs = q.shape
    if len(qs) != 3 or qs[2] != D or qs[1] < 1 or qs[1] % heads:
        raise RuntimeError(f"q must be [sequences, a multiple of {heads}, {D}], got {list(qs)}")
    if D > 256:
        raise RuntimeError(f"head_size must be at most 256, got {D}")
    B, Hq = qs[0], qs[1]
    table = block_table.shape
    if block_table.dtype != torch.int32 or len(table) != 2 or table[0] != B:
        raise RuntimeError(f"block_table must be int32 [{B}, pages], got {block_table.dtype} {list(table)}")
    if lens.dtype != torch.int32 or lens.shape != (B,):
        raise RuntimeError(f"lens must be int32 [{B}], got {lens.dtype} {list(lens.shape)}")
    at = dev.index
    if q.get_device() != at or block_table.get_device() != at or lens.get_device() != at:
        raise RuntimeError("q, block_table and lens must be on the cache's device")
    cols = table[1]
    if q.stride(2) != 1:
        q = q.contiguous()
    if block_table.stride(1) != 1 and cols > 1 or block_table.stride(0) < cols and B > 1:
        block_table = block_table.contiguous()
    lens = lens.contiguous()
    L = _lib.load()
    with _on(at):
        out = torch.empty((B, Hq, D), dtype=q.dtype, device=dev)
        lse = torch.empty((B, Hq), dtype=torch.float32, device=dev) if return_lse else None
        need = L.emu_kv_attend_workspace_size(B, Hq, heads, D)
        work = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        status = L.emu_kv_attend(q.data_ptr(), q.stride(0), q.stride(1), _DTYPE[q.dtype], B, Hq, heads, D,
                                 D ** -0.5 if scale is None else float(scale), fmt, k_cache.data_ptr(), v_cache.data_ptr(),
                                 k_scale.data_ptr(), v_scale.data_ptr(), pages, page_size, block_table.data_ptr(), cols,
                                 max(block_table.stride(0), cols), lens.data_ptr(), out.data_ptr(), _ptr(lse), _ptr(work),
                                 need, _raw_stream(at))
    if status:
        _lib._check(status)
    return (out, lse) if return_lse else out


__all__ = ["make_kv_cache", "write_kv_cache", "read_kv_cache", "attend_kv_cache"]
