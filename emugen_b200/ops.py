"""The emulated GEMMs as registered torch operators: ``torch.ops.emugen.*``.

Registered with ``torch.library.custom_op`` together with a fake (shape-only) implementation, so that
``torch.compile`` traces through them as single opaque nodes with known [M, N] outputs, and CUDA-graph
capture records their launches (the library allocates only through torch's allocator and does not
synchronise the host).  Each op calls the same C ABI as the Python drop-ins:

  torch.ops.emugen.emulated_scaled_fp4_mm  <- nvfp_cpp_emul.emulated_scaled_fp4_mm (nvfp_emulation.cpp:90-156)
  torch.ops.emugen.emulated_mxfp4_mm       <- mxfp_cpp_emul.emulated_mxfp4_mm     (mxfp_emulation.cpp:98-166)
  torch.ops.emugen.gemm                     every format / block size / rounding / output mode (emu_gemm_ws)

Importing this module registers the ops (``import emugen_b200.ops``); the reference has no torch-op
registration of its own (it loads its C++ emulators as Python extension modules).
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib, attention, fp8, kvcache

_OUT_DTYPE = {_lib.EMU_OUT_F16: torch.float16, _lib.EMU_OUT_BF16_VIA_F16: torch.bfloat16,
              _lib.EMU_OUT_F32: torch.float32}


def _rounding(code: int) -> int:
    """The C++ emulators' rounding codes: 0 is RZ, any other value RNE."""
    return _lib.EMU_RZ if int(code) == 0 else _lib.EMU_RNE


@torch.library.custom_op("emugen::gemm", mutates_args=())
def gemm(a_fp4: torch.Tensor, b_fp4: torch.Tensor, scale_a: torch.Tensor, scale_b: torch.Tensor,
         alpha: Optional[torch.Tensor], fmt: int, group_size: int, w_reduce: int, stage3_rounding: int,
         stage4_rounding: int, out_mode: int) -> torch.Tensor:
    """Emulated scaled FP4 GEMM [M, K/2] x [N, K/2] -> [M, N] (fp16 / bf16 / f32 by out_mode)."""
    return _lib.gemm(a_fp4, b_fp4, scale_a, scale_b, fmt=fmt, group_size=group_size, w_reduce=w_reduce,
                     stage3_rounding=stage3_rounding, stage4_rounding=stage4_rounding, alpha=alpha,
                     out_mode=out_mode)


@gemm.register_fake
def _gemm_fake(a_fp4, b_fp4, scale_a, scale_b, alpha, fmt, group_size, w_reduce, stage3_rounding,
               stage4_rounding, out_mode):
    torch._check(a_fp4.dim() == 2 and b_fp4.dim() == 2, lambda: "a_fp4, b_fp4 must be 2D")
    torch._check(a_fp4.shape[1] == b_fp4.shape[1], lambda: "K mismatch between a and b")
    return a_fp4.new_empty((a_fp4.shape[0], b_fp4.shape[0]), dtype=_OUT_DTYPE[out_mode])


@torch.library.custom_op("emugen::emulated_scaled_fp4_mm", mutates_args=())
def emulated_scaled_fp4_mm(a_fp4: torch.Tensor, b_fp4: torch.Tensor, scale_a: torch.Tensor,
                           scale_b: torch.Tensor, alpha: torch.Tensor, m_chunk_size: int = 128,
                           stage3_rounding: int = 0, stage4_rounding: int = 0) -> torch.Tensor:
    """NVFP4 (16-element groups, E4M3 scales, 4 groups per block) -> [M, N] fp16, as the reference's."""
    if int(m_chunk_size) <= 0:
        raise RuntimeError("m_chunk_size must be positive")
    return _lib.gemm(a_fp4, b_fp4, scale_a, scale_b, fmt=_lib.EMU_FMT_NVFP4, group_size=16, w_reduce=4,
                     stage3_rounding=_rounding(stage3_rounding), stage4_rounding=_rounding(stage4_rounding),
                     alpha=alpha, out_mode=_lib.EMU_OUT_F16)


@emulated_scaled_fp4_mm.register_fake
def _nvfp_fake(a_fp4, b_fp4, scale_a, scale_b, alpha, m_chunk_size=128, stage3_rounding=0, stage4_rounding=0):
    torch._check(a_fp4.shape[1] == b_fp4.shape[1], lambda: "K mismatch between a and b")
    return a_fp4.new_empty((a_fp4.shape[0], b_fp4.shape[0]), dtype=torch.float16)


@torch.library.custom_op("emugen::emulated_mxfp4_mm", mutates_args=())
def emulated_mxfp4_mm(a_fp4: torch.Tensor, b_fp4: torch.Tensor, scale_a: torch.Tensor, scale_b: torch.Tensor,
                      group_size: int = 32, m_chunk_size: int = 128, stage3_rounding: int = 0,
                      stage4_rounding: int = 0) -> torch.Tensor:
    """MXFP4 (32-element groups, UE8M0 scales, 2 groups per block) -> [M, N] fp16, as the reference's."""
    if int(group_size) != 32:
        raise RuntimeError("only MXFP4 group_size=32 is supported")
    if int(m_chunk_size) <= 0:
        raise RuntimeError("m_chunk_size must be positive")
    return _lib.gemm(a_fp4, b_fp4, scale_a, scale_b, fmt=_lib.EMU_FMT_MXFP4, group_size=32, w_reduce=2,
                     stage3_rounding=_rounding(stage3_rounding), stage4_rounding=_rounding(stage4_rounding),
                     alpha=None, out_mode=_lib.EMU_OUT_F16)


@emulated_mxfp4_mm.register_fake
def _mxfp_fake(a_fp4, b_fp4, scale_a, scale_b, group_size=32, m_chunk_size=128, stage3_rounding=0,
               stage4_rounding=0):
    torch._check(a_fp4.shape[1] == b_fp4.shape[1], lambda: "K mismatch between a and b")
    return a_fp4.new_empty((a_fp4.shape[0], b_fp4.shape[0]), dtype=torch.float16)


@torch.library.custom_op("emugen::quant_fp8", mutates_args=())
def quant_fp8(x: torch.Tensor, block: str = "row", dtype: torch.dtype = torch.float8_e4m3fn) -> tuple[torch.Tensor, torch.Tensor]:
    """Block-scaled 8-bit quantiser: (codes [M, K], scales), laid out as fp8.quant_fp8 does."""
    return fp8.quant_fp8(x, block=block, dtype=dtype)


def _device(*tensors) -> torch.device:
    """The device that _lib._device_for picks, without a GPU: the first CUDA tensor's, else the current one."""
    for t in tensors:
        if t.device.type == "cuda":
            return t.device
    return torch.device("cuda")


@quant_fp8.register_fake
def _quant_fp8_fake(x, block="row", dtype=torch.float8_e4m3fn):
    dev = _device(x)
    M, K = x.numel() // x.shape[-1] if x.shape[-1] else x.shape[:-1].numel(), x.shape[-1]
    kb = fp8._blocks(K)
    s = (fp8._row_scales(M, kb, dev) if block == "row"
         else torch.empty((fp8._blocks(M), kb), dtype=torch.float32, device=dev))
    return fp8._codes(M, K, dtype, dev), s


@torch.library.custom_op("emugen::gemm_fp8", mutates_args=())
def gemm_fp8(a: torch.Tensor, b: torch.Tensor, scale_a: torch.Tensor, scale_b: torch.Tensor,
             out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """Block-scaled 8-bit product a [M, K] @ b [N, K].T -> [M, N]."""
    return fp8.gemm_fp8(a, b, scale_a, scale_b, out_dtype=out_dtype)


@gemm_fp8.register_fake
def _gemm_fp8_fake(a, b, scale_a, scale_b, out_dtype=torch.bfloat16):
    torch._check(a.dim() == 2 and b.dim() == 2, lambda: "a, b, scale_a and scale_b must be 2D")
    torch._check(a.shape[1] == b.shape[1], lambda: "K mismatch between a and b")
    on_cpu = not any(t.device.type == "cuda" for t in (a, b, scale_a, scale_b))
    dev = a.device if on_cpu else _device(a, b, scale_a, scale_b)
    return torch.empty((a.shape[0], b.shape[0]), dtype=out_dtype, device=dev)


@torch.library.custom_op("emugen::write_kv_cache", mutates_args=("k_cache", "v_cache", "k_scale", "v_scale"))
def write_kv_cache(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_cache: torch.Tensor,
                   v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor) -> None:
    """Quantise k and v [tokens, heads, head_size] into their slots of the cache."""
    kvcache.write_kv_cache(k, v, slots, k_cache, v_cache, k_scale, v_scale)


@write_kv_cache.register_fake
def _write_kv_cache_fake(k, v, slots, k_cache, v_cache, k_scale, v_scale):
    return None


@torch.library.custom_op("emugen::read_kv_cache", mutates_args=())
def read_kv_cache(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                  block_table: torch.Tensor, cu_lens: torch.Tensor, total: int,
                  dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """The cached rows of a batch of sequences, packed: (k, v) [total, heads, head_size]."""
    return kvcache.read_kv_cache(k_cache, v_cache, k_scale, v_scale, block_table, cu_lens, total=total, dtype=dtype)


@read_kv_cache.register_fake
def _read_kv_cache_fake(k_cache, v_cache, k_scale, v_scale, block_table, cu_lens, total, dtype=torch.bfloat16):
    D = k_cache.shape[3] if k_cache.dtype == torch.float8_e4m3fn else 2 * k_cache.shape[3]
    shape = (total, k_cache.shape[2], D)
    return k_cache.new_empty(shape, dtype=dtype), k_cache.new_empty(shape, dtype=dtype)


@torch.library.custom_op("emugen::attend_kv_cache", mutates_args=())
def attend_kv_cache(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                    v_scale: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor,
                    scale: Optional[float] = None) -> torch.Tensor:
    """Attention of one new token for each sequence over its cached rows: [sequences, query heads, head_size]."""
    with torch.no_grad():
        return kvcache.attend_kv_cache(q, k_cache, v_cache, k_scale, v_scale, block_table, lens, scale=scale)


@attend_kv_cache.register_fake
def _attend_kv_cache_fake(q, k_cache, v_cache, k_scale, v_scale, block_table, lens, scale=None):
    return q.new_empty(q.shape)


@torch.library.custom_op("emugen::qk_norm_rope", mutates_args=())
def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
                 cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, eps: float = 1e-6,
                 interleaved: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """Norms of queries and keys [tokens, heads, head_size] with the position rotation (without gradients)."""
    with torch.no_grad():
        return attention.qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps=eps, interleaved=interleaved)


@qk_norm_rope.register_fake
def _qk_norm_rope_fake(q, k, q_weight, k_weight, cos, sin, positions, eps=1e-6, interleaved=False):
    return q.new_empty(q.shape), k.new_empty(k.shape)


@torch.library.custom_op("emugen::packed_attention", mutates_args=())
def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor, cu_k: Optional[torch.Tensor] = None,
                     causal: bool = True, scale: Optional[float] = None) -> torch.Tensor:
    """Attention over packed sequences [tokens, heads, head_size] (without gradients)."""
    with torch.no_grad():
        return attention.packed_attention(q, k, v, cu_q, cu_k, causal=causal, scale=scale)


@packed_attention.register_fake
def _packed_attention_fake(q, k, v, cu_q, cu_k=None, causal=True, scale=None):
    return q.new_empty(q.shape)


__all__ = ["gemm", "emulated_scaled_fp4_mm", "emulated_mxfp4_mm", "quant_fp8", "gemm_fp8", "write_kv_cache", "read_kv_cache",
           "attend_kv_cache", "qk_norm_rope", "packed_attention"]
