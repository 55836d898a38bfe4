"""Plain 64-bit restatement of the 8-bit block formats and the cache formats, on the CPU (numpy), for the tests."""
import numpy as np
import torch

MAX = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}


def values(dtype):
    """The value of every code, as f64 (NaN and infinities included)."""
    return torch.arange(256, dtype=torch.int32).to(torch.uint8).view(dtype).float().double().numpy()


def decode(q: torch.Tensor) -> np.ndarray:
    return values(q.dtype)[q.detach().cpu().contiguous().view(torch.uint8).numpy()]


def nearest_code(y: np.ndarray, dtype) -> np.ndarray:
    """Code of the value nearest to y (f64, finite, at most the type's largest), ties to the even code."""
    v = values(dtype)[:128]
    v = v[np.isfinite(v)]                      # codes 0 .. n-1 in increasing order
    a = np.abs(y)
    mid = (v[1:] + v[:-1]) / 2
    lo, hi = np.searchsorted(mid, a, "left"), np.searchsorted(mid, a, "right")
    code = np.where(lo % 2 == 0, lo, hi).astype(np.uint8)
    return code | (np.signbit(y).astype(np.uint8) << 7)


def _scale(block, dtype):
    b = np.abs(block[np.isfinite(block)])
    amax = np.float32(b.max()) if b.size else np.float32(0)
    return max(np.float32(amax / np.float32(MAX[dtype])), np.float32(2.0 ** -126))


def quant(x: torch.Tensor, block: str, dtype):
    """(codes uint8 with 0x7F for NaN, scales f32) of x [M, K]."""
    x = x.detach().cpu().float().numpy()
    M, K = x.shape
    kb, mb = -(-K // 128), -(-M // 128)
    rows = 1 if block == "row" else 128
    codes = np.zeros((M, K), np.uint8)
    scales = np.zeros((M if block == "row" else mb, kb), np.float32)
    for r in range(scales.shape[0]):
        for c in range(kb):
            sl = np.s_[r * rows:(r + 1) * rows, c * 128:(c + 1) * 128]
            s = _scale(x[sl], dtype)
            scales[r, c] = s
            fin = np.isfinite(x[sl])
            y = np.where(fin, x[sl], 0).astype(np.float64) / np.float64(s)
            codes[sl] = np.where(fin, nearest_code(y, dtype), 0x7F)
    return codes, scales


def codes_of(q: torch.Tensor) -> np.ndarray:
    """Codes with every NaN as 0x7F."""
    c = q.detach().cpu().contiguous().view(torch.uint8).numpy()
    return np.where(np.isnan(values(q.dtype)[c]), 0x7F, c).astype(np.uint8)


def spread(s, n_rows, n_cols, rows):
    """Block scales -> one f64 factor per element."""
    s = np.asarray(s, np.float64)
    s = np.repeat(s, 128, 1)[:, :n_cols]
    return s if rows else np.repeat(s, 128, 0)[:n_rows]


def gemm(a, b, sa, sb):
    """(product, sum of magnitudes) in f64 of quantised a [M, K], b [N, K] (torch tensors)."""
    x = decode(a) * spread(sa.cpu().numpy(), *a.shape, True)
    w = decode(b) * spread(sb.cpu().numpy(), *b.shape, sb.shape[0] == b.shape[0])
    return x @ w.T, np.abs(x) @ np.abs(w).T


def gemm_tolerance(ref, mag, K, out_dtype):
    """Bound of the product's error.  Within a block of 128 the tensor core aligns 128 addends and 4 running sums
    and may drop up to one unit of f32's last place for each (2^-23 of the magnitudes' sum): 132 * 2^-23.  Each of
    the ceil(K / 128) scaled additions and the scales' product round to f32 (2^-24 each, twice for margin of
    the running sum).  Then one rounding to the output type, half a step of it (for fp16 also below its
    normal range: 2^-25)."""
    eps = torch.finfo(out_dtype).eps / 2
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}[out_dtype]
    inner = (132 * 2.0 ** -23 + (2 * -(-K // 128) + 2) * 2.0 ** -24) * mag
    return inner + eps * (np.abs(ref) + inner) + tiny
