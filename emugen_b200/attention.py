"""Attention of prompts and training batches, and what comes before it.

  qk_norm_rope      norms of queries and keys for each head with the position rotation, in one pass over them
  packed_attention  attention over sequences of different lengths packed one after another, with grouped heads

Both are differentiable (reverse mode).  Tensors are [tokens, heads, head_size]; keys and values come from a
projection or, for a prompt whose beginning is cached, from kvcache.read_kv_cache.  One new token for each sequence
attends with kvcache.attend_kv_cache.  The kernels run on the inputs' device and its current stream, allocate only through torch's
allocator and do not synchronise, so that CUDA graphs can capture them.  The reference has no attention.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _lib
from .fp8 import _DTYPE, _on, _raw_stream


def _plain(name: str, *tensors) -> None:
    """Refuse inputs with a forward-mode tangent (there are none outside of a dual level)."""
    if forward_ad._current_level < 0:
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{name} has no forward-mode derivative")


def _wants_grad(*tensors) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t [tokens, heads, head_size] with consecutive elements in each row."""
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


# ------------------------------------------------------------------------------------- norms and rotation

def _norm_rope_args(q, k, qw, kw, cos, sin, positions, eps: float, interleaved: bool):
    T, Hq, D = q.shape
    return _lib.EmuNormRopeArgs(q.data_ptr(), k.data_ptr(), q.stride(0), q.stride(1), k.stride(0), k.stride(1), _ptr(qw), _ptr(kw),
                                cos.data_ptr(), sin.data_ptr(), positions.data_ptr(), T, cos.shape[0], Hq, k.shape[1], D,
                                cos.shape[1], _DTYPE[q.dtype], int(interleaved), eps)


def _norm_rope(q, k, qw, kw, cos, sin, positions, eps, interleaved):
    dev = q.device
    q, k = _rows(q), _rows(k)
    with _on(dev.index):
        yq, yk = torch.empty(q.shape, dtype=q.dtype, device=dev), torch.empty(k.shape, dtype=k.dtype, device=dev)
        args = _norm_rope_args(q, k, qw, kw, cos, sin, positions, eps, interleaved)
        status = _lib.load().emu_qk_norm_rope(ctypes.byref(args), yq.data_ptr(), yk.data_ptr(), _raw_stream(dev.index))
    if status:
        _lib._check(status)
    return yq, yk


class _NormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, qw, kw, cos, sin, positions, eps, interleaved):
        ctx.save_for_backward(q, k, qw, kw, cos, sin, positions)
        ctx.rest = eps, interleaved
        return _norm_rope(q, k, qw, kw, cos, sin, positions, eps, interleaved)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gq, gk):
        q, k, qw, kw, cos, sin, positions = ctx.saved_tensors
        dev = q.device
        q, k, gq, gk = _rows(q), _rows(k), _rows(gq), _rows(gk)
        L = _lib.load()
        with _on(dev.index):
            dq, dk = (torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (q, k))
            dqw = torch.empty_like(qw) if qw is not None and ctx.needs_input_grad[2] else None
            dkw = torch.empty_like(kw) if kw is not None and ctx.needs_input_grad[3] else None
            args = _norm_rope_args(q, k, qw, kw, cos, sin, positions, *ctx.rest)
            need = L.emu_qk_norm_rope_workspace_size(q.shape[2])
            work = torch.empty(need, dtype=torch.uint8, device=dev)
            status = L.emu_qk_norm_rope_backward(ctypes.byref(args), gq.data_ptr(), gk.data_ptr(), gq.stride(0), gq.stride(1),
                                                 gk.stride(0), gk.stride(1), dq.data_ptr(), dk.data_ptr(), _ptr(dqw), _ptr(dkw),
                                                 work.data_ptr(), need, _raw_stream(dev.index))
        if status:
            _lib._check(status)
        return dq, dk, dqw, dkw, None, None, None, None, None


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
                 cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, *, eps: float = 1e-6,
                 interleaved: bool = False):
    """Each row (token, head) of q and k divided by its root mean square, times its tensor's weight, and turned by its
    position's angles: (q', k'), contiguous.  Differentiable in q, k and the weights.

    q [tokens, query heads, head_size] and k [tokens, key heads, head_size]: fp16 / bf16 / f32, any token and head
    strides (slices of a fused projection); weights [head_size] of the same dtype, or None for ones.  cos, sin f32
    [positions, half]; token t takes row positions[t] (int64 [tokens]).  With x the row, z = x / sqrt(mean(x^2) + eps) * weight:
    pairs (a, b) of z's first 2 * half elements become (a cos - b sin, b cos + a sin), pair i being (z[i], z[i + half]),
    or with `interleaved` (z[2i], z[2i + 1]); the rest stays.  A negative position is padding: its rows are zeros and give
    no gradients.  A position past the table turns its rows to NaN.  head_size is a multiple of 8 up to 256, half a
    multiple of 8 unless interleaved (0: norms alone).  Sums in f32, one rounding.

    The backward pass makes q's and k's gradients whenever it runs.  For one that a CUDA graph is to capture,
    see fp8.linear_fp8."""
    qs, ks, dtype = q.shape, k.shape, q.dtype
    if len(qs) != 3 or len(ks) != 3 or qs[0] != ks[0] or qs[2] != ks[2]:
        raise RuntimeError(f"q and k must be [tokens, heads, head_size] of the same tokens and head size, got {list(qs)} and {list(ks)}")
    if dtype != k.dtype or dtype not in _DTYPE:
        raise RuntimeError(f"q and k must share one of float16, bfloat16, float32, got {dtype} and {k.dtype}")
    T, Hq, D = qs
    if Hq < 1 or ks[1] < 1:
        raise RuntimeError("q and k must have heads")
    if D < 8 or D > 256 or D % 8:
        raise RuntimeError(f"head_size must be a multiple of 8 up to 256, got {D}")
    for n, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (w.dtype != dtype or w.shape != (D,)):
            raise RuntimeError(f"{n} must be {dtype} [{D}], got {w.dtype} {list(w.shape)}")
    table = cos.shape
    if cos.dtype != torch.float32 or sin.dtype != torch.float32 or len(table) != 2 or table != sin.shape:
        raise RuntimeError("cos and sin must be float32 [positions, half]")
    half = table[1]
    if 2 * half > D or not interleaved and half % 8:
        raise RuntimeError(f"half (cos.shape[1]) must be at most head_size / 2, a multiple of 8 unless interleaved, got {half}")
    if positions.dtype != torch.int64 or positions.shape != (T,):
        raise RuntimeError(f"positions must be int64 [{T}], got {positions.dtype} {list(positions.shape)}")
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    _plain("qk_norm_rope", q, k, q_weight, k_weight, cos, sin)
    if cos.requires_grad or sin.requires_grad:
        raise RuntimeError("qk_norm_rope has no gradient for cos and sin")
    at = q.get_device()
    if (at < 0 or k.get_device() != at or cos.get_device() != at or sin.get_device() != at or positions.get_device() != at
            or q_weight is not None and q_weight.get_device() != at or k_weight is not None and k_weight.get_device() != at):
        raise RuntimeError("q, k, the weights, cos, sin and positions must be on the same CUDA device")
    qw = None if q_weight is None else q_weight.contiguous()
    kw = None if k_weight is None else k_weight.contiguous()
    cos, sin, positions = cos.contiguous(), sin.contiguous(), positions.contiguous()
    if _wants_grad(q, k, qw, kw):
        return _NormRope.apply(q, k, qw, kw, cos, sin, positions, float(eps), bool(interleaved))
    return _norm_rope(q, k, qw, kw, cos, sin, positions, float(eps), bool(interleaved))


# ------------------------------------------------------------------------------------- attention

def _aligned(t: torch.Tensor) -> torch.Tensor:
    """t [tokens, heads, head_size] as the kernels take it: rows of consecutive elements on 16-byte boundaries that do not
    overlap; copied if it is laid out otherwise (an expanded gradient, say)."""
    n, h, d = t.shape
    s = t.stride()
    if s[2] == 1 and (s[0] % 8 == 0 and s[0] >= d or n == 1) and (s[1] % 8 == 0 and s[1] >= d or h == 1) and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _strides(t: torch.Tensor):
    """Elements between tokens and between heads; where there is one of them its stride means nothing."""
    n, h, d = t.shape
    head = t.stride(1) if h > 1 else d
    return t.stride(0) if n > 1 else h * d, head


def _attention_args(q, k, v, cu_q, cu_k, causal: bool, scale: float):
    return _lib.EmuAttentionArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), *_strides(q), *_strides(k), *_strides(v),
                                 cu_q.data_ptr(), cu_k.data_ptr(), q.shape[0], k.shape[0], cu_q.shape[0] - 1, q.shape[1], k.shape[1],
                                 q.shape[2], _DTYPE[q.dtype], int(causal), scale)


def _forward(q, k, v, cu_q, cu_k, causal, scale, want_lse, want_low=False):
    dev = q.device
    with _on(dev.index):
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        lse = torch.empty((q.shape[1], q.shape[0]), dtype=torch.float32, device=dev) if want_lse else None
        low = torch.empty(q.shape, dtype=q.dtype, device=dev) if want_low else None
        args = _attention_args(q, k, v, cu_q, cu_k, causal, scale)
        status = _lib.load().emu_attention(ctypes.byref(args), out.data_ptr(), _ptr(low), _ptr(lse), _raw_stream(dev.index))
    if status:
        _lib._check(status)
    return out, low, lse


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, causal, scale):
        out, low, lse = _forward(q, k, v, cu_q, cu_k, causal, scale, True, True)
        ctx.save_for_backward(q, k, v, cu_q, cu_k, out, low, lse)
        ctx.rest = causal, scale
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do, _):
        q, k, v, cu_q, cu_k, out, low, lse = ctx.saved_tensors
        if do is None:
            return None, None, None, None, None, None, None
        dev = q.device
        L = _lib.load()
        with _on(dev.index):
            do = _aligned(do)
            dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=dev) if need else None
                          for t, need in zip((q, k, v), ctx.needs_input_grad))
            args = _attention_args(q, k, v, cu_q, cu_k, *ctx.rest)
            need = L.emu_attention_backward_workspace_size(ctypes.byref(args))
            work = torch.empty(need, dtype=torch.uint8, device=dev)
            status = L.emu_attention_backward(ctypes.byref(args), out.data_ptr(), low.data_ptr(), lse.data_ptr(), do.data_ptr(), *_strides(do),
                                              _ptr(dq), _ptr(dk), _ptr(dv), work.data_ptr(), need, _raw_stream(dev.index))
        if status:
            _lib._check(status)
        return dq, dk, dv, None, None, None, None


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor,
                     cu_k: Optional[torch.Tensor] = None, *, causal: bool = True, scale: Optional[float] = None,
                     return_lse: bool = False):
    """Attention over packed sequences: q [query tokens, query heads, head_size], k and v [key tokens, key heads,
    head_size] -> [query tokens, query heads, head_size], differentiable in q, k and v.

    cu_q, cu_k int32 [sequences + 1], non-decreasing from 0: sequence b has the queries cu_q[b] .. cu_q[b + 1] - 1 and the keys
    cu_k[b] .. cu_k[b + 1] - 1 (cu_k None: the same as cu_q).  Query heads are a multiple of the key heads, query head h using
    key head h // (query heads // key heads).  causal: the last query of a sequence stands on its last key, the one before it sees
    one key less, and so on (a prompt's new piece against its cached beginning and itself).  scale: of the scores (default
    head_size ** -0.5; positive).  Queries that see no key and rows behind the last sequence give zeros; their keys' and
    values' gradients are zeros too.  What the mask hides reaches no result, whatever it holds.

    fp16 or bf16 tensors of one CUDA device, head_size a multiple of 8 up to 128; rows that do not start on 16-byte
    boundaries are copied first.  Scores, softmax and sums in f32; its weights, and in the backward pass the scores' gradients, are
    rounded to the inputs' dtype for the products (in fp16 after a power of two that keeps small ones, taken from the row, sequence
    and key head alone); a call that is differentiated also keeps what the output's rounding took away (as large as the output).
    The same result every run.  With return_lse also f32 [query heads,
    query tokens]: the logarithm of the sum of exp(score), -inf where no key is seen (not differentiable).
    Reverse mode only.  For a backward pass that a CUDA graph is to capture, see fp8.linear_fp8."""
    qs, ks, dtype = q.shape, k.shape, q.dtype
    if len(qs) != 3 or len(ks) != 3 or ks != v.shape or qs[2] != ks[2]:
        raise RuntimeError("q must be [query tokens, heads, head_size], k and v [key tokens, heads, head_size], got "
                           f"{list(qs)}, {list(ks)} and {list(v.shape)}")
    if dtype != k.dtype or dtype != v.dtype or dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError(f"q, k and v must share one of float16, bfloat16, got {dtype}, {k.dtype} and {v.dtype}")
    D = qs[2]
    if D < 8 or D > 128 or D % 8:
        raise RuntimeError(f"head_size must be a multiple of 8 up to 128, got {D}")
    if ks[1] < 1 or qs[1] < 1 or qs[1] % ks[1]:
        raise RuntimeError(f"query heads ({qs[1]}) must be a positive multiple of key heads ({ks[1]})")
    if cu_k is None:
        if qs[0] != ks[0]:
            raise RuntimeError("cu_k is needed where q and k have different numbers of tokens")
        cu_k = cu_q
    for n, c in (("cu_q", cu_q), ("cu_k", cu_k)):
        if c.dtype != torch.int32 or c.dim() != 1 or c.shape[0] < 1 or c.shape != cu_q.shape:
            raise RuntimeError(f"{n} must be int32 [sequences + 1], got {c.dtype} {list(c.shape)}")
    scale = D ** -0.5 if scale is None else float(scale)
    if not 0 < scale < float("inf"):
        raise ValueError("scale must be positive and finite")
    _plain("packed_attention", q, k, v)
    at = q.get_device()
    if at < 0 or k.get_device() != at or v.get_device() != at or cu_q.get_device() != at or cu_k.get_device() != at:
        raise RuntimeError("q, k, v, cu_q and cu_k must be on the same CUDA device")
    cu_q, cu_k = cu_q.contiguous(), cu_k.contiguous()
    q, k, v = _aligned(q), _aligned(k), _aligned(v)
    if _wants_grad(q, k, v):
        out, lse = _Attention.apply(q, k, v, cu_q, cu_k, bool(causal), scale)
    else:
        out, _, lse = _forward(q, k, v, cu_q, cu_k, bool(causal), scale, return_lse)
    return (out, lse) if return_lse else out


__all__ = ["qk_norm_rope", "packed_attention"]
