"""Block-scaled 8-bit floating point: the quantiser, the matrix product and a linear layer with its
backward pass.

Codes are ``torch.float8_e4m3fn`` or ``torch.float8_e5m2``; every block of 128 carries one f32 scale:
blocks of 1 x 128 along the rows ("row", activations and gradients) or 128 x 128 tiles ("tile",
weights).  An element stands for code * scale.

  quant_fp8   x -> codes and scales, and on request those of the transposed matrix in the same pass
  gemm_fp8    a @ b.T of two quantised matrices on the tensor cores, f32 sums
  linear_fp8  x @ weight.T with all three products of a training step in 8 bits

The kernels run on the inputs' device and its current stream, allocate only their outputs (through
torch's allocator) and do not synchronise, so that CUDA graphs can capture them.  The reference has no 8-bit path.
"""
from __future__ import annotations

import contextlib

import torch
from torch.autograd import forward_ad

from . import _lib

BLOCK = 128
_FP8 = {torch.float8_e4m3fn: _lib.EMU_FP8_E4M3, torch.float8_e5m2: _lib.EMU_FP8_E5M2}
_DTYPE = {torch.float16: _lib.EMU_DTYPE_F16, torch.bfloat16: _lib.EMU_DTYPE_BF16, torch.float32: _lib.EMU_DTYPE_F32}
_BLOCKS = {"row": _lib.EMU_BLOCK_ROW, "tile": _lib.EMU_BLOCK_TILE}


def _blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


_HERE = contextlib.nullcontext()
# current_stream(dev).cuda_stream and current_device() without their objects and start-up checks
_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


def _on(index: int):
    """Make device `index`, which holds a tensor, current for the call.  Where it already is, as in most calls,
    entering and leaving torch.cuda.device would cost a small launch's time."""
    return _HERE if _current_device() == index else torch.cuda.device(index)


def _codes(rows: int, cols: int, dtype: torch.dtype, dev: torch.device) -> torch.Tensor:
    """[rows, cols] codes whose rows start on 16 bytes, as the product wants them."""
    pitch = (cols + 15) // 16 * 16
    q = torch.empty((rows, pitch), dtype=dtype, device=dev)
    return q if pitch == cols else q[:, :cols]


def _row_scales(rows: int, blocks: int, dev: torch.device) -> torch.Tensor:
    """[rows, blocks] scales stored block after block, each block's row a multiple of 4 floats."""
    pitch = (rows + 3) // 4 * 4
    s = torch.empty_strided((pitch, blocks), (1, pitch), dtype=torch.float32, device=dev)
    return s if pitch == rows else s[:rows]


def quant_fp8(x: torch.Tensor, *, block: str = "row", dtype: torch.dtype = torch.float8_e4m3fn,
              transposed: bool = False):
    """x [..., K] (fp16 / bf16 / f32, leading dimensions flattened to M rows) -> (q, scale), or with
    `transposed` (q, scale, qt, scale_t), the second pair being x.T quantised in the same pass.

    q [M, K], qt [K, M]: codes of `dtype`; their rows start on 16-byte boundaries (so they need not be
    contiguous).  block "row": scale [M, ceil(K / 128)] and scale_t [K, ceil(M / 128)], stored block after
    block (strides 1, rows rounded up to 4); block "tile": scale [ceil(M / 128), ceil(K / 128)] and its
    transpose.  scale = max(max |x| / F, 2^-126) in f32 over the block's finite elements (F: the type's
    largest value), code = the nearest value to x / scale, ties to even; NaN and infinities become NaN.
    A CPU tensor is quantised on the current GPU, where its codes and scales stay.  Not differentiable."""
    if dtype not in _FP8:
        raise RuntimeError(f"quant_fp8 dtype must be torch.float8_e4m3fn or torch.float8_e5m2, got {dtype}")
    if block not in _BLOCKS:
        raise ValueError(f"block must be 'row' or 'tile', got {block!r}")
    if x.dtype not in _DTYPE:
        raise RuntimeError(f"quantiser input must be float16, bfloat16 or float32, got {x.dtype}")
    if x.dim() == 0:
        raise RuntimeError("quantiser input must have at least one dimension")
    if not x.is_cuda:
        x = x.to(_lib._device_for(x))
    if x.requires_grad:
        x = x.detach()
    return _quant(_matrix(x), _BLOCKS[block], dtype, transposed)


def _matrix(x: torch.Tensor) -> torch.Tensor:
    """x with its leading dimensions flattened."""
    return x if x.dim() == 2 else x.reshape(x.shape[:-1].numel(), x.shape[-1])


def _quant(x: torch.Tensor, block: int, dtype: torch.dtype, transposed: bool):
    """quant_fp8 of a checked CUDA matrix."""
    dev = x.device
    M, K = x.shape
    ldx, inner = x.stride()
    if inner != 1 and K > 1 or ldx < K and M > 1:   # overlapping or column-strided rows
        x = x.contiguous()
        ldx = K
    mb, kb = _blocks(M), _blocks(K)
    q = _codes(M, K, dtype, dev)
    if block == _lib.EMU_BLOCK_ROW:
        s, lds = _row_scales(M, kb, dev), (M + 3) // 4 * 4
    else:
        s, lds = torch.empty((mb, kb), dtype=torch.float32, device=dev), kb
    qt = st = None
    ldst = 0
    if transposed:
        qt = _codes(K, M, dtype, dev)
        if block == _lib.EMU_BLOCK_ROW:
            st, ldst = _row_scales(K, mb, dev), (K + 3) // 4 * 4
        else:
            st, ldst = torch.empty((kb, mb), dtype=torch.float32, device=dev), mb
    if M and K:
        L = _lib.load()
        with _on(dev.index):
            status = L.emu_quant_fp8(x.data_ptr(), _DTYPE[x.dtype], M, K, ldx if M > 1 else K, _FP8[dtype], block,
                                     q.data_ptr(), (K + 15) // 16 * 16, s.data_ptr(), lds,
                                     qt.data_ptr() if transposed else None, (M + 15) // 16 * 16,
                                     st.data_ptr() if transposed else None, ldst, _raw_stream(dev.index))
        if status:
            _lib._check(status)
    return (q, s, qt, st) if transposed else (q, s)


def _operand(t: torch.Tensor, dev: torch.device):
    """(tensor kept alive, pitch in bytes): rows that start on 16 bytes, copied there if they do not."""
    if t.device != dev:
        t = t.to(dev)
    rows, cols = t.shape
    ld, inner = t.stride()
    if inner != 1 and cols > 1 or rows > 1 and (ld % 16 or ld < cols) or t.data_ptr() % 16:
        c = _codes(rows, cols, t.dtype, dev)
        c.view(torch.uint8).copy_(t.view(torch.uint8))
        t = c
        ld = t.stride(0)
    return t, ld if rows > 1 else (cols + 15) // 16 * 16


def _scale_rows(s: torch.Tensor, dev: torch.device):
    """(tensor kept alive, floats between blocks): scales stored block after block on 16-byte rows that can
    be read up to a multiple of 4, copied there if they are not."""
    if s.device != dev:
        s = s.to(dev)
    rows, blocks = s.shape
    r4 = (rows + 3) // 4 * 4
    inner, ld = s.stride()
    if blocks == 1:
        ld = r4
    good = (rows == 1 or inner == 1) and ld % 4 == 0 and ld >= r4 and s.data_ptr() % 16 == 0
    if good and r4 != rows:
        good = (s.storage_offset() + (blocks - 1) * ld + r4) * 4 <= s.untyped_storage().nbytes()
    if not good:
        c = _row_scales(rows, blocks, dev)
        c.copy_(s)
        s, ld = c, r4
    return s, ld


def gemm_fp8(a: torch.Tensor, b: torch.Tensor, scale_a: torch.Tensor, scale_b: torch.Tensor, *,
             out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a [M, K] @ b [N, K].T with quant_fp8's codes and scales -> [M, N] fp16 / bf16 / f32.

    scale_a [M, ceil(K / 128)]: a scale for each row of a and block of K.  scale_b: the same for b
    ([N, ceil(K / 128)]) or one for each 128 x 128 tile ([ceil(N / 128), ceil(K / 128)]).  a and b may be of
    different 8-bit types.  Sums in f32, one rounding at the end, the same result every run.  Operands
    and scales laid out otherwise than quant_fp8 leaves them are copied first."""
    if a.dim() != 2 or b.dim() != 2 or scale_a.dim() != 2 or scale_b.dim() != 2:
        raise RuntimeError("a, b, scale_a and scale_b must be 2D")
    if a.dtype not in _FP8 or b.dtype not in _FP8:
        raise RuntimeError(f"a and b must be float8_e4m3fn or float8_e5m2, got {a.dtype} and {b.dtype}")
    if scale_a.dtype != torch.float32 or scale_b.dtype != torch.float32:
        raise RuntimeError("scale_a and scale_b must be float32")
    if out_dtype not in _DTYPE:
        raise RuntimeError(f"out_dtype must be float16, bfloat16 or float32, got {out_dtype}")
    M, K = a.shape
    N = b.shape[0]
    if b.shape[1] != K:
        raise RuntimeError("K mismatch between a and b")
    kb = _blocks(K)
    if tuple(scale_a.shape) != (M, kb):
        raise RuntimeError(f"scale_a must be [{M}, {kb}], got {list(scale_a.shape)}")
    rows = tuple(scale_b.shape) == (N, kb)
    if not rows and tuple(scale_b.shape) != (_blocks(N), kb):
        raise RuntimeError(f"scale_b must be [{N}, {kb}] or [{_blocks(N)}, {kb}], got {list(scale_b.shape)}")
    if a.is_cuda:
        return _gemm(a, b, scale_a, scale_b, rows, out_dtype, a.device)
    on_cpu = not (b.is_cuda or scale_a.is_cuda or scale_b.is_cuda)
    dev = _lib._device_for(a, b, scale_a, scale_b)
    out = _gemm(a, b, scale_a, scale_b, rows, out_dtype, dev)
    if on_cpu:
        _lib.device_status(dev)
        return out.cpu()
    return out


def _gemm(a, b, scale_a, scale_b, rows: bool, out_dtype: torch.dtype, dev: torch.device) -> torch.Tensor:
    """gemm_fp8 of checked operands on `dev`; rows: scale_b has a row for each of b's."""
    M, K = a.shape
    N = b.shape[0]
    out = torch.empty((M, N), dtype=out_dtype, device=dev)
    if not (M and N):
        return out
    with _on(dev.index):
        if not K:
            return out.zero_()
        a_, lda = _operand(a, dev)
        b_, ldb = _operand(b, dev)
        sa, ldsa = _scale_rows(scale_a, dev)
        if rows:
            sb, ldsb = _scale_rows(scale_b, dev)
        else:
            sb, ldsb = scale_b.to(dev).contiguous(), scale_b.shape[1]
        status = _lib.load().emu_gemm_fp8(a_.data_ptr(), lda, _FP8[a.dtype], b_.data_ptr(), ldb, _FP8[b.dtype],
                                          sa.data_ptr(), ldsa, sb.data_ptr(), ldsb,
                                          _lib.EMU_BLOCK_ROW if rows else _lib.EMU_BLOCK_TILE, M, N, K,
                                          _DTYPE[out_dtype], out.data_ptr(), N, _raw_stream(dev.index))
    if status:
        _lib._check(status)
    return out


def _up(n: int, m: int) -> int:
    return (n + m - 1) // m * m


class _Quantised:
    """Codes and scales of a [rows, cols] matrix inside a byte buffer, at 256-byte places, as the product
    takes them; `tile`: 128 x 128 blocks.  One buffer for a layer's operands in place of a tensor for each."""

    def __init__(self, rows: int, cols: int, tile: bool, at: int = 0):
        self.rows, self.cols, self.tile, self.codes = rows, cols, tile, at
        self.ld = _up(cols, 16)
        self.ld_scale = _blocks(cols) if tile else _up(rows, 4)
        self.scale = at + _up(rows * self.ld, 256)
        self.end = self.scale + _up(4 * self.ld_scale * (_blocks(rows) if tile else _blocks(cols)), 256)


def _quant_into(x: torch.Tensor, block: int, q, base: int, t, base_t: int, stream: int) -> None:
    """quant_fp8 of a matrix into q at address `base` and of its transpose into t at base_t; either may be None."""
    rows, cols = x.shape
    ldx, inner = x.stride()
    if inner != 1 and cols > 1 or ldx < cols and rows > 1:
        x = x.contiguous()
        ldx = cols
    status = _lib.load().emu_quant_fp8(
        x.data_ptr(), _DTYPE[x.dtype], rows, cols, ldx if rows > 1 else cols, _lib.EMU_FP8_E4M3, block,
        *((base + q.codes, q.ld, base + q.scale, q.ld_scale) if q else (None, 0, None, 0)),
        *((base_t + t.codes, t.ld, base_t + t.scale, t.ld_scale) if t else (None, 0, None, 0)), stream)
    if status:
        _lib._check(status)


def _product(a: _Quantised, base_a: int, b: _Quantised, base_b: int, dtype: torch.dtype, dev: torch.device, stream: int):
    out = torch.empty((a.rows, b.rows), dtype=dtype, device=dev)
    status = _lib.load().emu_gemm_fp8(
        base_a + a.codes, a.ld, _lib.EMU_FP8_E4M3, base_b + b.codes, b.ld, _lib.EMU_FP8_E4M3, base_a + a.scale, a.ld_scale,
        base_b + b.scale, b.ld_scale, _lib.EMU_BLOCK_TILE if b.tile else _lib.EMU_BLOCK_ROW, a.rows, b.rows, a.cols,
        _DTYPE[dtype], out.data_ptr(), b.rows, stream)
    if status:
        _lib._check(status)
    return out


def _linear(x: torch.Tensor, weight: torch.Tensor, need_x: bool, need_w: bool):
    """(y [M, N], what the wanted gradients need): x.T's codes for the weight's, weight.T's for x's, each a
    byte buffer or None."""
    (M, K), N, dev = x.shape, weight.shape[0], x.device
    if not (M and N and K):
        return torch.zeros((M, N), dtype=x.dtype, device=dev), None, None
    q = _Quantised(M, K, False)
    w = _Quantised(N, K, True, q.end)
    qt, wt = _Quantised(K, M, False) if need_w else None, _Quantised(K, N, True) if need_x else None
    with _on(dev.index):
        now = torch.empty(w.end, dtype=torch.uint8, device=dev)
        xt = torch.empty(qt.end, dtype=torch.uint8, device=dev) if need_w else None
        wtt = torch.empty(wt.end, dtype=torch.uint8, device=dev) if need_x else None
        base, stream = now.data_ptr(), _raw_stream(dev.index)
        _quant_into(x, _lib.EMU_BLOCK_ROW, q, base, qt, xt.data_ptr() if need_w else 0, stream)
        _quant_into(weight, _lib.EMU_BLOCK_TILE, w, base, wt, wtt.data_ptr() if need_x else 0, stream)
        return _product(q, base, w, base, x.dtype, dev, stream), xt, wtt


def _linear_backward(dy: torch.Tensor, xt, wt, K: int, need_x: bool, need_w: bool):
    """(dx [M, K], dw [N, K]), each None where it is not wanted."""
    (M, N), dtype, dev = dy.shape, dy.dtype, dy.device
    if not (M and N and K):
        return (torch.zeros((M, K), dtype=dtype, device=dev) if need_x else None,
                torch.zeros((N, K), dtype=dtype, device=dev) if need_w else None)
    # dx takes dy's codes along its rows, dw those along its columns
    g = _Quantised(M, N, False) if need_x else None
    gt = _Quantised(N, M, False, g.end if g else 0) if need_w else None
    with _on(dev.index):
        now = torch.empty((gt or g).end, dtype=torch.uint8, device=dev)
        base, stream = now.data_ptr(), _raw_stream(dev.index)
        _quant_into(dy, _lib.EMU_BLOCK_ROW, g, base, gt, base, stream)
        return (_product(g, base, _Quantised(K, N, True), wt.data_ptr(), dtype, dev, stream) if need_x else None,
                _product(gt, base, _Quantised(K, M, False), xt.data_ptr(), dtype, dev, stream) if need_w else None)


class _LinearFp8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight):
        need_x, need_w = ctx.needs_input_grad
        y, xt, wt = _linear(_matrix(x), weight, need_x, need_w)
        ctx.save_for_backward(xt, wt)
        ctx.x_shape = x.shape
        return y if x.dim() == 2 else y.reshape(*x.shape[:-1], weight.shape[0])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        need_x, need_w = ctx.needs_input_grad
        shape = ctx.x_shape
        dx, dw = _linear_backward(_matrix(dy), *ctx.saved_tensors, shape[-1], need_x, need_w)
        return dx if dx is None or len(shape) == 2 else dx.reshape(shape), dw


def linear_fp8(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    """x [..., K] @ weight [N, K].T -> [..., N] in x's dtype, differentiable in both.

    With Q the quantiser (E4M3; rows in blocks of 128, the weight in 128 x 128 tiles):
      y  = Q(x) Q(weight)^T,   dx = Q(dy) Q(weight),   dw = Q(dy^T) Q(x^T)^T
    (the gradients treat Q as the identity).  The forward pass keeps the 8-bit transposes of x and the weight
    for the backward pass, not x itself.  fp16, bf16 or f32 CUDA tensors of one device and dtype.  Reverse mode only: inputs
    with a forward-mode tangent are refused.

    A backward pass that a CUDA graph is to capture follows torch's rule for every operator: no eager graph of
    the same leaves may be alive (their gradient accumulators belong to its stream, and torch ends the process over
    it) -- warm up on a side stream and drop the outputs first, as torch.cuda.make_graphed_callables does."""
    if x.dim() < 1 or weight.dim() != 2:
        raise RuntimeError("x must have at least one dimension and weight two")
    if x.shape[-1] != weight.shape[1]:
        raise RuntimeError("K mismatch between x and weight")
    if x.dtype != weight.dtype or x.dtype not in _DTYPE:
        raise RuntimeError(f"x and weight must share one of float16, bfloat16, float32, got {x.dtype} and {weight.dtype}")
    if forward_ad.unpack_dual(x).tangent is not None or forward_ad.unpack_dual(weight).tangent is not None:
        raise RuntimeError("linear_fp8 has no forward-mode derivative")
    if not x.is_cuda or x.device != weight.device:
        raise RuntimeError("x and weight must be on the same CUDA device")
    if not (torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad)):
        y = _linear(_matrix(x.detach()), weight.detach(), False, False)[0]
        return y if x.dim() == 2 else y.reshape(*x.shape[:-1], weight.shape[0])
    return _LinearFp8.apply(x, weight)


__all__ = ["quant_fp8", "gemm_fp8", "linear_fp8"]
