"""emugen_b200 — EmuGen's emulated NVFP4 / MXFP4 scaled GEMM on NVIDIA B200 (sm_100a).

The compute lives in ``libemugen.so`` (C ABI in include/emugen.h, CUDA kernels in csrc/).  The
Python modules mirror the reference interfaces that call it:

  emugen_b200.nvfp_cpp_emul   <- nvfp_cpp_emul            (emulated_scaled_fp4_mm, RZ, RNE)
  emugen_b200.mxfp_cpp_emul   <- mxfp_cpp_emul            (emulated_mxfp4_mm)
  emugen_b200.emulation       <- search.emulation         (MMAEngine, emulate_nvfp_scaled_fp4_mm, ...)
  emugen_b200.backends        <- gemm_compare.backends    (build_nvfp_fns, build_mxfp_fns, states)

and, beyond the reference, block-scaled 8-bit operators:

  emugen_b200.fp8             quantiser, matrix product, linear layer with its backward pass
  emugen_b200.kvcache         quantised key/value cache (8 or 4 bits): write, read back, attention of one token over it
  emugen_b200.attention       norms of queries and keys with the position rotation, attention over packed sequences
"""
from . import _lib
from ._lib import EmuError, gemm, nvfp4_global_scales, quant_mxfp4, quant_nvfp4
from .attention import packed_attention, qk_norm_rope
from .fp8 import gemm_fp8, linear_fp8, quant_fp8
from .kvcache import attend_kv_cache, make_kv_cache, read_kv_cache, write_kv_cache

__all__ = ["EmuError", "gemm", "nvfp4_global_scales", "quant_mxfp4", "quant_nvfp4", "quant_fp8", "gemm_fp8", "linear_fp8",
           "make_kv_cache", "write_kv_cache", "read_kv_cache", "attend_kv_cache", "qk_norm_rope", "packed_attention", "load_library"]


def load_library():
    """Load libemugen.so (raises if it has not been built)."""
    return _lib.load()
