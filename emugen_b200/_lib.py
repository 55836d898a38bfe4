"""ctypes binding of libemugen.so (include/emugen.h) plus the torch-tensor glue.

The library is the product: every emulated GEMM and quantisation below runs in its CUDA kernels.
There is no CPU fallback.  If the shared library is missing this module raises at first use
(build it with ``python -m emugen_b200.build``); CPU tensors are computed on the current CUDA
device and copied back, and without a CUDA device every call raises.
"""
from __future__ import annotations

import ctypes
import threading
from pathlib import Path

import torch

PKG = Path(__file__).resolve().parent
LIB_PATH = PKG / "libemugen.so"

# enums of include/emugen.h
EMU_OK = 0
EMU_FMT_NVFP4, EMU_FMT_MXFP4 = 0, 1
EMU_RZ, EMU_RNE = 0, 1
EMU_OUT_F16, EMU_OUT_BF16_VIA_F16, EMU_OUT_F32 = 0, 1, 2
EMU_DTYPE_F16, EMU_DTYPE_BF16, EMU_DTYPE_F32 = 0, 1, 2
EMU_FP8_E4M3, EMU_FP8_E5M2 = 0, 1
EMU_BLOCK_ROW, EMU_BLOCK_TILE = 0, 1
EMU_KV_FP8, EMU_KV_MXFP4 = 0, 1
ABI_VERSION = 1

SYMBOLS = ("emu_abi_version", "emu_last_error", "emu_status_string", "emu_gemm", "emu_gemm_workspace_size", "emu_gemm_tc_workspace_size",
           "emu_gemm_ws", "emu_gemm_tc_path_offset", "emu_gemm_static", "emu_nvfp4_global_scales", "emu_nvfp4_amax",
           "emu_nvfp4_scales_from_amax", "emu_quant_nvfp4", "emu_quant_mxfp4",
           "emu_gemm_model", "emu_gemm_sweep", "emu_gemm_compare", "emu_gemm_batch", "emu_compare", "emu_dequant_fp4", "emu_device_status",
           "emu_set_wait_limit", "emu_test_hold_first_ready", "emu_quant_fp8", "emu_gemm_fp8", "emu_kv_write", "emu_kv_read")
STATIC_SCRATCH_BYTES = 64 << 20   # EMU_STATIC_SCRATCH_BYTES


class EmuGemmParams(ctypes.Structure):
    _fields_ = [("format", ctypes.c_int32), ("group_size", ctypes.c_int32), ("w_reduce", ctypes.c_int32),
                ("stage3_rounding", ctypes.c_int32), ("stage4_rounding", ctypes.c_int32),
                ("out_mode", ctypes.c_int32)]


class EmuCompareStats(ctypes.Structure):
    _fields_ = [("mismatches", ctypes.c_int64), ("first_index", ctypes.c_int64), ("max_diff", ctypes.c_float),
                ("max_sq_error", ctypes.c_float), ("sq_error_sum", ctypes.c_double), ("ref_sq_sum", ctypes.c_double),
                ("numel", ctypes.c_int64)]


class EmuAccumModel(ctypes.Structure):
    _fields_ = [("align3", ctypes.c_int32), ("align4", ctypes.c_int32), ("align_rounding", ctypes.c_int32),
                ("order", ctypes.c_int32)]


class EmuSweepModel(ctypes.Structure):
    _fields_ = [("w_reduce", ctypes.c_int32), ("stage4_rounding", ctypes.c_int32), ("align3", ctypes.c_int32),
                ("align4", ctypes.c_int32), ("align_rounding", ctypes.c_int32), ("order", ctypes.c_int32)]


class EmuError(RuntimeError):
    """A failing libemugen call; ``status`` is the emu_status code."""

    def __init__(self, status: int, message: str):
        super().__init__(message)
        self.status = status


_lib = None
_lock = threading.Lock()


def load() -> ctypes.CDLL:
    """Load libemugen.so once and declare its signatures.  Raises if it is missing."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        if not LIB_PATH.is_file():
            raise ImportError(f"{LIB_PATH} not found: build it with `python -m emugen_b200.build`")
        L = ctypes.CDLL(str(LIB_PATH))
        vp, i32, i64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64
        L.emu_abi_version.restype = i32
        L.emu_abi_version.argtypes = []
        L.emu_last_error.restype = ctypes.c_char_p
        L.emu_last_error.argtypes = []
        L.emu_status_string.restype = ctypes.c_char_p
        L.emu_status_string.argtypes = [i32]
        L.emu_gemm.restype = i32
        L.emu_gemm.argtypes = [vp, vp, vp, vp, i64, i64, i64, i64, i64, i64, i64, vp,
                               ctypes.POINTER(EmuGemmParams), vp, vp]
        L.emu_gemm_workspace_size.restype = ctypes.c_size_t
        L.emu_gemm_workspace_size.argtypes = [i64, i64, i64, ctypes.POINTER(EmuGemmParams)]
        L.emu_gemm_tc_workspace_size.restype = ctypes.c_size_t
        L.emu_gemm_tc_workspace_size.argtypes = [i64, i64, i64, ctypes.POINTER(EmuGemmParams)]
        L.emu_gemm_tc_path_offset.restype = ctypes.c_size_t
        L.emu_gemm_tc_path_offset.argtypes = [i64, i64, i64, ctypes.POINTER(EmuGemmParams)]
        L.emu_gemm_ws.restype = i32
        L.emu_gemm_ws.argtypes = [vp, vp, vp, vp, i64, i64, i64, i64, i64, i64, i64, vp,
                                  ctypes.POINTER(EmuGemmParams), vp, vp, ctypes.c_size_t, vp]
        L.emu_gemm_static.restype = i32
        L.emu_gemm_static.argtypes = [vp, vp, vp, vp, i64, i64, i64, i64, i64, i64, i64, vp,
                                      ctypes.POINTER(EmuGemmParams), vp, vp]
        L.emu_nvfp4_global_scales.restype = i32
        L.emu_nvfp4_global_scales.argtypes = [vp, i64, vp, i64, i32, vp, vp, vp, vp]
        L.emu_nvfp4_amax.restype = i32
        L.emu_nvfp4_amax.argtypes = [vp, i64, vp, i64, i32, vp, vp, vp]
        L.emu_nvfp4_scales_from_amax.restype = i32
        L.emu_nvfp4_scales_from_amax.argtypes = [vp, vp, vp, vp, vp, vp]
        L.emu_quant_nvfp4.restype = i32
        L.emu_quant_nvfp4.argtypes = [vp, i32, i64, i64, vp, vp, vp, vp]
        L.emu_quant_mxfp4.restype = i32
        L.emu_quant_mxfp4.argtypes = [vp, i32, i64, i64, vp, vp, vp]
        L.emu_gemm_model.restype = i32
        L.emu_gemm_model.argtypes = [vp, vp, vp, vp, i64, i64, i64, i64, i64, i64, i64, vp,
                                     ctypes.POINTER(EmuGemmParams), ctypes.POINTER(EmuAccumModel), vp, vp]
        L.emu_gemm_sweep.restype = i32
        L.emu_gemm_sweep.argtypes = [vp, vp, vp, vp, i64, i64, i64, i64, i64, i64, i64, vp, i32, i32,
                                     ctypes.POINTER(EmuSweepModel), i32, vp, i32, vp, vp]
        L.emu_gemm_compare.restype = i32
        L.emu_gemm_compare.argtypes = [vp, vp, vp, vp, i64, i64, i64, i64, i64, i64, i64, vp,
                                       ctypes.POINTER(EmuGemmParams), vp, vp, vp, vp, ctypes.c_size_t, vp]
        L.emu_gemm_batch.restype = i32
        L.emu_gemm_batch.argtypes = [vp, vp, vp, vp, i64, i64, i64, i64, i64, i64, i64, vp,
                                     ctypes.POINTER(EmuGemmParams), i32, vp, vp, vp, vp, ctypes.c_size_t, vp]
        L.emu_compare.restype = i32
        L.emu_compare.argtypes = [vp, vp, i32, i64, vp, vp]
        L.emu_dequant_fp4.restype = i32
        L.emu_dequant_fp4.argtypes = [vp, vp, i64, i64, i64, i32, vp, vp, vp]
        L.emu_device_status.restype = i32
        L.emu_device_status.argtypes = [vp]
        L.emu_set_wait_limit.restype = i64
        L.emu_set_wait_limit.argtypes = [i64]
        L.emu_test_hold_first_ready.restype = i32
        L.emu_test_hold_first_ready.argtypes = [i32]
        L.emu_quant_fp8.restype = i32
        L.emu_quant_fp8.argtypes = [vp, i32, i64, i64, i64, i32, i32, vp, i64, vp, i64, vp, i64, vp, i64, vp]
        L.emu_gemm_fp8.restype = i32
        L.emu_gemm_fp8.argtypes = [vp, i64, i32, vp, i64, i32, vp, i64, vp, i64, i32, i64, i64, i64, i32, vp, i64, vp]
        L.emu_kv_write.restype = i32
        L.emu_kv_write.argtypes = [vp, vp, i32, i64, i64, i64, i64, i64, i64, i64, vp, i32, i64, vp, vp, vp, vp, vp]
        L.emu_kv_read.restype = i32
        L.emu_kv_read.argtypes = [vp, vp, vp, vp, i32, i64, i64, i64, i64, vp, i64, i64, i64, vp, i64, i32, vp, vp,
                                  i64, i64, vp]
        v = L.emu_abi_version()
        if v != ABI_VERSION:
            raise ImportError(f"libemugen ABI version {v}, expected {ABI_VERSION}: rebuild it")
        _lib = L
    return _lib


def _check(status: int) -> None:
    if status != EMU_OK:
        L = load()
        raise EmuError(status, L.emu_last_error().decode() or L.emu_status_string(status).decode())


EMU_ERR_TIMEOUT = 10


def device_status(device: torch.device | int | None = None) -> None:
    """Synchronise the device's current stream and raise EmuError if a tensor-core pipeline wait ran
    out since the last check (emu_device_status); the outputs of those calls are undefined."""
    L = load()
    if device is None:
        dev = torch.device("cuda", torch.cuda.current_device())
    else:
        dev = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
    with torch.cuda.device(dev):
        _check(L.emu_device_status(_stream(dev)))


def set_wait_limit(cycles: int) -> int:
    """Bound (SM cycles) of each pipeline wait in later tensor-core launches; <= 0 restores the
    default (2^31).  Returns the previous bound."""
    return int(load().emu_set_wait_limit(int(cycles)))


def _device_for(*tensors: torch.Tensor) -> torch.device:
    for t in tensors:
        if t.is_cuda:
            return t.device
    if not torch.cuda.is_available():
        raise RuntimeError("emugen_b200 needs a CUDA device (sm_100a); no CPU fallback exists")
    return torch.device("cuda", torch.cuda.current_device())


def _stream(dev: torch.device) -> int:
    return torch.cuda.current_stream(dev).cuda_stream


def _bytes2d(t: torch.Tensor, dev: torch.device, name: str) -> torch.Tensor:
    if t.dim() != 2:
        raise RuntimeError(f"{name} must be 2D")
    if t.element_size() != 1:
        raise RuntimeError(f"{name} must be a 1-byte dtype (uint8 / float8), got {t.dtype}")
    return t.to(dev).contiguous().view(torch.uint8)


def gemm(a_fp4: torch.Tensor, b_fp4: torch.Tensor, scale_a: torch.Tensor, scale_b: torch.Tensor, *,
         fmt: int, group_size: int, w_reduce: int, stage3_rounding: int, stage4_rounding: int,
         alpha: torch.Tensor | None, out_mode: int, path: str = "auto") -> torch.Tensor:
    """Emulated scaled FP4 GEMM through ``emu_gemm_ws``.  Returns [M, N] fp16 / bf16 / f32 on the
    inputs' CUDA device (or on CPU if every input was on CPU).

    path: "auto" gives the library the workspace it asks for (the tensor-core kernel where it applies
    and the problem is large enough to gain from it); "tc" gives the tensor-core kernel's workspace
    whatever the size; "simt" passes none, which selects the CUDA-core kernels.  All are bit-identical;
    "tc" and "simt" exist for tests."""
    L = load()
    on_cpu = not any(t.is_cuda for t in (a_fp4, b_fp4, scale_a, scale_b))
    dev = _device_for(a_fp4, b_fp4, scale_a, scale_b)
    if a_fp4.dim() != 2 or b_fp4.dim() != 2:
        raise RuntimeError("a_fp4, b_fp4 must be 2D")
    M, N, K = a_fp4.shape[0], b_fp4.shape[0], a_fp4.shape[1] * 2
    if b_fp4.shape[1] * 2 != K:
        raise RuntimeError("K mismatch between a and b")
    a = _bytes2d(a_fp4, dev, "a_fp4")
    b = _bytes2d(b_fp4, dev, "b_fp4")
    if scale_a.dim() != 2 or scale_b.dim() != 2:
        raise RuntimeError("scale tensor must be 2D")
    sa = _bytes2d(scale_a, dev, "scale_a")
    sb = _bytes2d(scale_b, dev, "scale_b")
    al = None
    if alpha is not None:
        if alpha.numel() != 1:
            raise RuntimeError(f"a Tensor with {alpha.numel()} elements cannot be converted to Scalar")
        al = alpha.detach().reshape(1).to(device=dev, dtype=torch.float32).contiguous()
    odt = {EMU_OUT_F16: torch.float16, EMU_OUT_BF16_VIA_F16: torch.bfloat16, EMU_OUT_F32: torch.float32}[out_mode]
    out = torch.empty((M, N), dtype=odt, device=dev)
    params = EmuGemmParams(fmt, group_size, w_reduce, stage3_rounding, stage4_rounding, out_mode)
    ws_ptr, ws_bytes, ws = None, 0, None
    if path in ("auto", "tc") and M > 0 and N > 0 and K > 0:
        query = L.emu_gemm_workspace_size if path == "auto" else L.emu_gemm_tc_workspace_size
        need = query(M, N, K, ctypes.byref(params))
        if need:
            ws = torch.empty(need + 1024, dtype=torch.uint8, device=dev)
            ws_ptr = (ws.data_ptr() + 1023) // 1024 * 1024
            ws_bytes = need
    elif path not in ("auto", "tc", "simt"):
        raise ValueError(f"unknown path {path!r}")
    with torch.cuda.device(dev):
        st = L.emu_gemm_ws(a.data_ptr(), b.data_ptr(), sa.data_ptr(), sb.data_ptr(), M, N, K,
                           sa.shape[0], sa.shape[1], sb.shape[0], sb.shape[1],
                           None if al is None else al.data_ptr(), ctypes.byref(params), out.data_ptr(),
                           ws_ptr, ws_bytes, _stream(dev))
    _check(st)
    if on_cpu:   # the copy back synchronises anyway: report a failed device pipeline here
        device_status(dev)
        return out.cpu()
    return out


def _dtype_code(x: torch.Tensor) -> int:
    if x.dtype == torch.float16:
        return EMU_DTYPE_F16
    if x.dtype == torch.bfloat16:
        return EMU_DTYPE_BF16
    raise RuntimeError(f"quantiser input must be float16 or bfloat16, got {x.dtype}")


def nvfp4_global_scales(a: torch.Tensor, b: torch.Tensor):
    """(gs_a, gs_b, alpha) as device float32[1] tensors, computed on the device."""
    L = load()
    dev = _device_for(a, b)
    if a.dtype != b.dtype:
        raise RuntimeError("a and b must have the same dtype")
    a_ = a.to(dev).contiguous()
    b_ = b.to(dev).contiguous()
    gsa = torch.empty(1, dtype=torch.float32, device=dev)
    gsb = torch.empty(1, dtype=torch.float32, device=dev)
    al = torch.empty(1, dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        st = L.emu_nvfp4_global_scales(a_.data_ptr(), a_.numel(), b_.data_ptr(), b_.numel(), _dtype_code(a_),
                                       gsa.data_ptr(), gsb.data_ptr(), al.data_ptr(), _stream(dev))
    _check(st)
    return gsa, gsb, al


def nvfp4_amax(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """max|a| and max|b| as an int32 [2] device tensor of f32 bit patterns (emu_nvfp4_amax): shards of
    an operand combine with an integer MAX (torch.distributed all_reduce MAX)."""
    L = load()
    dev = _device_for(a, b)
    if a.dtype != b.dtype:
        raise RuntimeError("a and b must have the same dtype")
    a_, b_ = a.to(dev).contiguous(), b.to(dev).contiguous()
    words = torch.empty(2, dtype=torch.int32, device=dev)
    with torch.cuda.device(dev):
        st = L.emu_nvfp4_amax(a_.data_ptr(), a_.numel(), b_.data_ptr(), b_.numel(), _dtype_code(a_),
                              words.data_ptr(), words.data_ptr() + 4, _stream(dev))
    _check(st)
    return words


def nvfp4_scales_from_amax(words: torch.Tensor):
    """(gs_a, gs_b, alpha) device float32[1] tensors from nvfp4_amax words (emu_nvfp4_scales_from_amax)."""
    L = load()
    if words.dtype != torch.int32 or words.numel() != 2 or not words.is_cuda:
        raise RuntimeError("words must be the int32 [2] CUDA tensor nvfp4_amax returns")
    w = words.contiguous()
    out = torch.empty(3, dtype=torch.float32, device=w.device)
    with torch.cuda.device(w.device):
        st = L.emu_nvfp4_scales_from_amax(w.data_ptr(), w.data_ptr() + 4, out.data_ptr(), out.data_ptr() + 4,
                                          out.data_ptr() + 8, _stream(w.device))
    _check(st)
    return out[0:1], out[1:2], out[2:3]


def _quant(x: torch.Tensor, sf_vec: int, gs: torch.Tensor | None):
    L = load()
    dev = _device_for(x)
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    x_ = x.to(dev).contiguous()
    M, K = x_.shape
    if K % sf_vec != 0:
        raise RuntimeError(f"K must be a multiple of {sf_vec}")
    q = torch.empty((M, K // 2), dtype=torch.uint8, device=dev)
    rows = (M + 127) // 128 * 128
    cols = (K // sf_vec + 3) // 4 * 4
    sf = torch.empty((rows, cols), dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        if sf_vec == 16:
            g = gs.reshape(1).to(device=dev, dtype=torch.float32).contiguous()
            st = L.emu_quant_nvfp4(x_.data_ptr(), _dtype_code(x_), M, K, g.data_ptr(), q.data_ptr(), sf.data_ptr(),
                                   _stream(dev))
        else:
            st = L.emu_quant_mxfp4(x_.data_ptr(), _dtype_code(x_), M, K, q.data_ptr(), sf.data_ptr(), _stream(dev))
    _check(st)
    return q, sf


def quant_nvfp4(x: torch.Tensor, global_scale: torch.Tensor):
    """x [M, K] fp16/bf16 -> (q uint8 [M, K/2], sf uint8 [pad128(M), pad4(K/16)] swizzled E4M3)."""
    return _quant(x, 16, global_scale)


def quant_mxfp4(x: torch.Tensor):
    """x [M, K] fp16/bf16 -> (q uint8 [M, K/2], sf uint8 [pad128(M), pad4(K/32)] swizzled UE8M0)."""
    return _quant(x, 32, None)


def _cmp_dtype(t: torch.Tensor) -> int:
    codes = {torch.float16: EMU_DTYPE_F16, torch.bfloat16: EMU_DTYPE_BF16, torch.float32: EMU_DTYPE_F32}
    if t.dtype not in codes:
        raise RuntimeError(f"compare supports float16, bfloat16 and float32 tensors, got {t.dtype}")
    return codes[t.dtype]


def compare_stats(ref: torch.Tensor, out: torch.Tensor) -> dict:
    """emu_compare on the device: mismatch count, first mismatch index, max |diff|, squared-error sums.
    Both tensors are moved to one CUDA device (the first CUDA one given) and must share shape and dtype."""
    L = load()
    if ref.shape != out.shape:
        raise RuntimeError(f"shape mismatch: {tuple(ref.shape)} vs {tuple(out.shape)}")
    if ref.dtype != out.dtype:
        raise RuntimeError(f"dtype mismatch: {ref.dtype} vs {out.dtype}")
    dev = _device_for(ref, out)
    r = ref.to(dev).contiguous()
    o = out.to(dev).contiguous()
    st = torch.empty(ctypes.sizeof(EmuCompareStats), dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        status = L.emu_compare(r.data_ptr(), o.data_ptr(), _cmp_dtype(r), r.numel(), st.data_ptr(), _stream(dev))
    _check(status)
    device_status(dev)   # reading the statistics synchronises anyway
    host = EmuCompareStats.from_buffer_copy(bytes(st.cpu().numpy()))
    return {k: getattr(host, k) for k, _ in EmuCompareStats._fields_}


def dequant_fp4(q: torch.Tensor, sf: torch.Tensor, *, fmt: int, global_scale: torch.Tensor | None = None
                ) -> torch.Tensor:
    """Packed e2m1 [rows, K/2] + swizzled scales -> f32 [rows, K] on the device (emu_dequant_fp4)."""
    L = load()
    dev = _device_for(q, sf)
    q_ = _bytes2d(q, dev, "q")
    sf_ = _bytes2d(sf, dev, "sf")
    rows, K = q_.shape[0], q_.shape[1] * 2
    out = torch.empty((rows, K), dtype=torch.float32, device=dev)
    g = None
    if fmt == EMU_FMT_NVFP4:
        if global_scale is None:
            raise RuntimeError("NVFP4 dequantisation needs the global scale")
        g = global_scale.reshape(1).to(device=dev, dtype=torch.float32).contiguous()
    with torch.cuda.device(dev):
        status = L.emu_dequant_fp4(q_.data_ptr(), sf_.data_ptr(), rows, K, sf_.shape[1], fmt,
                                   None if g is None else g.data_ptr(), out.data_ptr(), _stream(dev))
    _check(status)
    return out


def gemm_compare(a_fp4: torch.Tensor, b_fp4: torch.Tensor, scale_a: torch.Tensor, scale_b: torch.Tensor,
                 ref: torch.Tensor, *, fmt: int, group_size: int, w_reduce: int, stage3_rounding: int,
                 stage4_rounding: int, alpha: torch.Tensor | None, out_mode: int, write_out: bool = False,
                 path: str = "auto"):
    """Emulated GEMM compared with `ref` on the device (emu_gemm_compare).  Returns (stats dict,
    output or None).  With the tensor-core path and write_out=False the output is never written."""
    L = load()
    dev = _device_for(a_fp4, b_fp4, scale_a, scale_b)
    M, N, K = a_fp4.shape[0], b_fp4.shape[0], a_fp4.shape[1] * 2
    a = _bytes2d(a_fp4, dev, "a_fp4")
    b = _bytes2d(b_fp4, dev, "b_fp4")
    sa = _bytes2d(scale_a, dev, "scale_a")
    sb = _bytes2d(scale_b, dev, "scale_b")
    odt = {EMU_OUT_F16: torch.float16, EMU_OUT_BF16_VIA_F16: torch.bfloat16, EMU_OUT_F32: torch.float32}[out_mode]
    r = ref.to(device=dev).contiguous()
    if r.dtype != odt or tuple(r.shape) != (M, N):
        raise RuntimeError(f"ref must be {odt} [{M}, {N}], got {r.dtype} {tuple(r.shape)}")
    al = None if alpha is None else alpha.detach().reshape(1).to(device=dev, dtype=torch.float32).contiguous()
    params = EmuGemmParams(fmt, group_size, w_reduce, stage3_rounding, stage4_rounding, out_mode)
    ws_ptr, ws_bytes, ws = None, 0, None
    if path in ("auto", "tc"):
        query = L.emu_gemm_workspace_size if path == "auto" else L.emu_gemm_tc_workspace_size
        need = query(M, N, K, ctypes.byref(params))
        if need:
            ws = torch.empty(need + 1024, dtype=torch.uint8, device=dev)
            ws_ptr = (ws.data_ptr() + 1023) // 1024 * 1024
            ws_bytes = need
    out = torch.empty((M, N), dtype=odt, device=dev) if (write_out or ws_ptr is None) else None
    st = torch.empty(ctypes.sizeof(EmuCompareStats), dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        status = L.emu_gemm_compare(a.data_ptr(), b.data_ptr(), sa.data_ptr(), sb.data_ptr(), M, N, K,
                                    sa.shape[0], sa.shape[1], sb.shape[0], sb.shape[1],
                                    None if al is None else al.data_ptr(), ctypes.byref(params), r.data_ptr(),
                                    None if out is None else out.data_ptr(), st.data_ptr(), ws_ptr, ws_bytes,
                                    _stream(dev))
    _check(status)
    device_status(dev)   # reading the statistics synchronises anyway
    host = EmuCompareStats.from_buffer_copy(bytes(st.cpu().numpy()))
    return {k: getattr(host, k) for k, _ in EmuCompareStats._fields_}, out


def gemm_batch(a_fp4: torch.Tensor, b_fp4: torch.Tensor, scale_a: torch.Tensor, scale_b: torch.Tensor,
               params, *, alpha: torch.Tensor | None = None, ref: torch.Tensor | None = None, write_out: bool = True,
               path: str = "auto"):
    """Several parameter sets on the same operands in one call (emu_gemm_batch).  `params`: a sequence of
    (fmt, group_size, w_reduce, stage3_rounding, stage4_rounding, out_mode), every set with the first's
    format, group size and out mode.  Returns (outputs [n, M, N] or None, a stats dict per set or None):
    outputs when write_out, stats when `ref` is given (with write_out=False the comparisons run in the
    tensor-core epilogue and no output is written)."""
    L = load()
    dev = _device_for(a_fp4, b_fp4, scale_a, scale_b)
    M, N, K = a_fp4.shape[0], b_fp4.shape[0], a_fp4.shape[1] * 2
    a = _bytes2d(a_fp4, dev, "a_fp4")
    b = _bytes2d(b_fp4, dev, "b_fp4")
    sa = _bytes2d(scale_a, dev, "scale_a")
    sb = _bytes2d(scale_b, dev, "scale_b")
    sets = [EmuGemmParams(*[int(x) for x in p]) for p in params]
    n = len(sets)
    arr = (EmuGemmParams * max(n, 1))(*sets)
    odt = {EMU_OUT_F16: torch.float16, EMU_OUT_BF16_VIA_F16: torch.bfloat16, EMU_OUT_F32: torch.float32}[
        sets[0].out_mode if n else EMU_OUT_F16]
    r = None
    if ref is not None:
        r = ref.to(device=dev).contiguous()
        if r.dtype != odt or tuple(r.shape) != (M, N):
            raise RuntimeError(f"ref must be {odt} [{M}, {N}], got {r.dtype} {tuple(r.shape)}")
    al = None if alpha is None else alpha.detach().reshape(1).to(device=dev, dtype=torch.float32).contiguous()
    ws_ptr, ws_bytes, ws = None, 0, None
    if path in ("auto", "tc") and n and M > 0 and N > 0 and K > 0:
        query = L.emu_gemm_workspace_size if path == "auto" else L.emu_gemm_tc_workspace_size
        need = query(M, N, K, ctypes.byref(sets[0]))
        if need:
            ws = torch.empty(need + 1024, dtype=torch.uint8, device=dev)
            ws_ptr = (ws.data_ptr() + 1023) // 1024 * 1024
            ws_bytes = need
    out = torch.empty((n, M, N), dtype=odt, device=dev) if write_out else None
    st = torch.empty(max(n, 1) * ctypes.sizeof(EmuCompareStats), dtype=torch.uint8, device=dev) if r is not None else None
    with torch.cuda.device(dev):
        status = L.emu_gemm_batch(a.data_ptr(), b.data_ptr(), sa.data_ptr(), sb.data_ptr(), M, N, K,
                                  sa.shape[0], sa.shape[1], sb.shape[0], sb.shape[1],
                                  None if al is None else al.data_ptr(), arr, n,
                                  None if r is None else r.data_ptr(), None if out is None else out.data_ptr(),
                                  None if st is None else st.data_ptr(), ws_ptr, ws_bytes, _stream(dev))
    _check(status)
    stats = None
    if st is not None:
        device_status(dev)
        raw = bytes(st.cpu().numpy())
        size = ctypes.sizeof(EmuCompareStats)
        stats = []
        for i in range(n):
            h = EmuCompareStats.from_buffer_copy(raw[i * size:(i + 1) * size])
            stats.append({k: getattr(h, k) for k, _ in EmuCompareStats._fields_})
    return out, stats


def gemm_model(a_fp4: torch.Tensor, b_fp4: torch.Tensor, scale_a: torch.Tensor, scale_b: torch.Tensor, *,
               fmt: int, group_size: int, w_reduce: int, stage3_rounding: int, stage4_rounding: int,
               alpha: torch.Tensor | None, out_mode: int, align3: int = 0, align4: int = 0,
               align_rounding: int = EMU_RZ, order: int = 0) -> torch.Tensor:
    """Emulated GEMM under an accumulator model (emu_gemm_model); all-zero model = gemm()."""
    L = load()
    on_cpu = not any(t.is_cuda for t in (a_fp4, b_fp4, scale_a, scale_b))
    dev = _device_for(a_fp4, b_fp4, scale_a, scale_b)
    M, N, K = a_fp4.shape[0], b_fp4.shape[0], a_fp4.shape[1] * 2
    a = _bytes2d(a_fp4, dev, "a_fp4")
    b = _bytes2d(b_fp4, dev, "b_fp4")
    sa = _bytes2d(scale_a, dev, "scale_a")
    sb = _bytes2d(scale_b, dev, "scale_b")
    al = None if alpha is None else alpha.detach().reshape(1).to(device=dev, dtype=torch.float32).contiguous()
    odt = {EMU_OUT_F16: torch.float16, EMU_OUT_BF16_VIA_F16: torch.bfloat16, EMU_OUT_F32: torch.float32}[out_mode]
    out = torch.empty((M, N), dtype=odt, device=dev)
    params = EmuGemmParams(fmt, group_size, w_reduce, stage3_rounding, stage4_rounding, out_mode)
    model = EmuAccumModel(align3, align4, align_rounding, order)
    with torch.cuda.device(dev):
        status = L.emu_gemm_model(a.data_ptr(), b.data_ptr(), sa.data_ptr(), sb.data_ptr(), M, N, K,
                                  sa.shape[0], sa.shape[1], sb.shape[0], sb.shape[1],
                                  None if al is None else al.data_ptr(), ctypes.byref(params), ctypes.byref(model),
                                  out.data_ptr(), _stream(dev))
    _check(status)
    return out.cpu() if on_cpu else out


def gemm_sweep(a_fp4: torch.Tensor, b_fp4: torch.Tensor, scale_a: torch.Tensor, scale_b: torch.Tensor,
               ref: torch.Tensor, models: list, *, fmt: int, stage3_rounding: int = EMU_RZ,
               alpha: torch.Tensor | None = None) -> list[int]:
    """Mismatch count of each accumulator model against `ref` (emu_gemm_sweep).  `models` holds
    (w_reduce, stage4_rounding, align3, align4, align_rounding, order) tuples."""
    L = load()
    dev = _device_for(a_fp4, b_fp4, scale_a, scale_b, ref)
    M, N, K = a_fp4.shape[0], b_fp4.shape[0], a_fp4.shape[1] * 2
    a = _bytes2d(a_fp4, dev, "a_fp4")
    b = _bytes2d(b_fp4, dev, "b_fp4")
    sa = _bytes2d(scale_a, dev, "scale_a")
    sb = _bytes2d(scale_b, dev, "scale_b")
    r = ref.to(device=dev).contiguous()
    if tuple(r.shape) != (M, N):
        raise RuntimeError(f"ref must be [{M}, {N}], got {tuple(r.shape)}")
    al = None if alpha is None else alpha.detach().reshape(1).to(device=dev, dtype=torch.float32).contiguous()
    arr = (EmuSweepModel * max(1, len(models)))(*[EmuSweepModel(*m) for m in models])
    counts = torch.empty(max(1, len(models)), dtype=torch.int64, device=dev)
    with torch.cuda.device(dev):
        st = L.emu_gemm_sweep(a.data_ptr(), b.data_ptr(), sa.data_ptr(), sb.data_ptr(), M, N, K, sa.shape[0],
                              sa.shape[1], sb.shape[0], sb.shape[1], None if al is None else al.data_ptr(), fmt,
                              stage3_rounding, arr, len(models), r.data_ptr(), _cmp_dtype(r), counts.data_ptr(),
                              _stream(dev))
    _check(st)
    device_status(dev)   # reading the counts synchronises anyway
    return [int(x) for x in counts[: len(models)].cpu()]
