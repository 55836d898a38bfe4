"""The 8-bit operators and the quantised cache without a GPU: every refusal is made on the host before any
CUDA call, and the test oracle agrees with torch's own casts."""
import ctypes

import numpy as np
import pytest
import torch

from emugen_b200 import _lib, fp8, kvcache
from tests import fp8_oracle as O

P = 64   # a 64-byte aligned address that no call below gets to read


def _quant(**kw):
    a = dict(x=P, dtype=1, M=4, K=200, ldx=200, t=0, block=0, q=P, ldq=208, s=P, lds=4, qt=P, ldqt=16, st=P, ldst=200)
    a.update(kw)
    L = _lib.load()
    st = L.emu_quant_fp8(*a.values(), None)
    return st, L.emu_last_error().decode()


@pytest.mark.parametrize("kw,status,msg", [
    (dict(M=-1), 1, "negative size"), (dict(dtype=3), 1, "dtype must be"), (dict(t=2), 1, "unknown fp8_type"),
    (dict(block=2), 1, "unknown block"), (dict(x=None), 1, "NULL"), (dict(q=None, qt=None), 1, "NULL"),
    (dict(s=None), 1, "NULL"), (dict(st=None), 1, "NULL"), (dict(ldx=199), 1, "ldx"), (dict(ldq=192), 1, "code rows"),
    (dict(ldq=201), 1, "16-byte"), (dict(q=P + 8), 1, "16-byte"), (dict(qt=P + 1), 1, "16-byte"), (dict(ldqt=2), 1, "code rows"),
    (dict(x=P + 1), 1, "aligned"), (dict(s=P + 2), 1, "aligned"), (dict(lds=3), 1, "scale rows"), (dict(ldst=199), 1, "scale rows"), (dict(block=1, lds=1), 1, "scale rows"),
    (dict(M=1 << 40, ldqt=1 << 40, lds=1 << 40), 8, "2^31"),
])
def test_quant_refusals(kw, status, msg):
    st, got = _quant(**kw)
    assert st == status and msg in got


def _gemm(**kw):
    a = dict(a=P, lda=208, at=0, b=P, ldb=208, bt=1, sa=P, ldsa=8, sb=P, ldsb=12, block=0, M=7, N=9, K=200, od=1, out=P,
             ldo=9)
    a.update(kw)
    L = _lib.load()
    st = L.emu_gemm_fp8(*a.values(), None)
    return st, L.emu_last_error().decode()


@pytest.mark.parametrize("kw,status,msg", [
    (dict(K=-1), 1, "negative size"), (dict(at=2), 1, "operand type"), (dict(bt=-1), 1, "operand type"),
    (dict(block=7), 1, "b_block"), (dict(od=5), 1, "out_dtype"), (dict(out=None), 1, "NULL"), (dict(ldo=8), 1, "ldo"),
    (dict(out=P + 1), 1, "aligned"), (dict(a=None), 1, "NULL"), (dict(sb=None), 1, "NULL"), (dict(lda=192), 1, "at least K"),
    (dict(lda=201), 1, "16-byte"), (dict(b=P + 4), 1, "16-byte"), (dict(ldsa=9), 6, "scale_a"), (dict(ldsa=4), 6, "scale_a"),
    (dict(sa=P + 4), 6, "scale_a"), (dict(ldsb=8), 6, "scale_b"), (dict(sb=P + 8), 6, "scale_b"),
    (dict(block=1, ldsb=1), 6, "scale_b"), (dict(M=128 * 65535 + 1, ldsa=1 << 24), 8, "65535"),
    (dict(K=1 << 31, lda=1 << 32, ldb=1 << 32), 8, "K too large"),
])
def test_gemm_refusals(kw, status, msg):
    st, got = _gemm(**kw)
    assert st == status and msg in got


def _write(**kw):
    a = dict(k=P, v=P, dtype=1, T=3, H=2, D=64, kt=128, kh=64, vt=128, vh=64, slots=P, fmt=0, n=32, kc=P, vc=P, ks=P, vs=P)
    a.update(kw)
    L = _lib.load()
    st = L.emu_kv_write(*a.values(), None)
    return st, L.emu_last_error().decode()


@pytest.mark.parametrize("kw,status,msg", [
    (dict(T=-1), 1, "negative size"), (dict(n=-1), 1, "negative size"), (dict(dtype=2), 1, "dtype must be"),
    (dict(fmt=2), 1, "cache format"), (dict(H=0), 8, "heads"), (dict(H=65536, D=65536), 8, "2^28"), (dict(D=72), 3, "multiple of 16"),
    (dict(fmt=1, D=48), 3, "multiple of 32"), (dict(k=None), 1, "NULL"), (dict(vc=None), 1, "NULL"), (dict(ks=None), 1, "NULL"),
    (dict(slots=P + 4), 1, "aligned"), (dict(k=P + 1), 1, "aligned"), (dict(kc=P + 8), 1, "16-byte"),
    (dict(ks=P + 2), 1, "4-byte"),
])
def test_write_refusals(kw, status, msg):
    st, got = _write(**kw)
    assert st == status and msg in got


def _read(**kw):
    a = dict(kc=P, vc=P, ks=P, vs=P, fmt=0, pages=4, page=8, H=2, D=64, table=P, B=2, cols=2, ts=2, cu=P, total=20, od=1,
             ko=P, vo=P, kt=128, vt=128)
    a.update(kw)
    L = _lib.load()
    st = L.emu_kv_read(*a.values(), None)
    return st, L.emu_last_error().decode()


@pytest.mark.parametrize("kw,status,msg", [
    (dict(total=-1), 1, "negative size"), (dict(page=0), 1, "page_size"), (dict(od=3), 1, "out_dtype"), (dict(fmt=9), 1, "cache format"),
    (dict(D=8), 3, "multiple of 16"), (dict(cu=None), 1, "NULL"), (dict(ko=None), 1, "NULL"), (dict(vo=None), 1, "NULL"),
    (dict(vs=None), 1, "NULL"), (dict(table=None), 1, "NULL"), (dict(ts=1), 1, "table_stride"), (dict(kt=127), 1, "output rows"),
    (dict(vt=0), 1, "output rows"), (dict(cu=P + 2), 1, "aligned"), (dict(vc=P + 4), 1, "16-byte"), (dict(vs=P + 1), 1, "4-byte"),
])
def test_read_refusals(kw, status, msg):
    st, got = _read(**kw)
    assert st == status and msg in got


def test_empty_calls_succeed_without_pointers():
    assert _quant(M=0, x=None, q=None, qt=None)[0] == 0
    assert _gemm(M=0, a=None, out=None)[0] == 0
    assert _write(T=0, k=None, slots=None)[0] == 0
    assert _read(total=0, ko=None, vo=None)[0] == 0


def test_python_refusals():
    x = torch.zeros(4, 128)
    with pytest.raises(RuntimeError, match="dtype must be"):
        fp8.quant_fp8(x, dtype=torch.float16)
    with pytest.raises(ValueError, match="block"):
        fp8.quant_fp8(x, block="column")
    with pytest.raises(RuntimeError, match="input must be"):
        fp8.quant_fp8(x.double())
    q = torch.zeros(4, 128, dtype=torch.uint8).view(torch.float8_e4m3fn)
    s = torch.ones(4, 1)
    for bad, msg in [((q, q[:, :64], s, s), "K mismatch"), ((q, q, s[:3], s), "scale_a"), ((q, q, s, torch.ones(2, 1)), "scale_b"),
                     ((q.view(torch.uint8), q, s, s), "must be float8"), ((q, q, s.double(), s), "float32"), ((q[0], q, s, s), "2D")]:
        with pytest.raises(RuntimeError, match=msg):
            fp8.gemm_fp8(*bad)
    with pytest.raises(RuntimeError, match="out_dtype"):
        fp8.gemm_fp8(q, q, s, s, out_dtype=torch.float64)
    with pytest.raises(RuntimeError, match="CUDA"):
        fp8.linear_fp8(x, x)
    with pytest.raises(RuntimeError, match="K mismatch"):
        fp8.linear_fp8(x, x[:, :64])
    with pytest.raises(RuntimeError, match="share one"):
        fp8.linear_fp8(x, x.half())


def test_python_cache_refusals():
    for kw, msg in [(dict(head_size=40), "multiple of 16"), (dict(head_size=48, fmt="mxfp4"), "multiple of 32"),
                    (dict(fmt="int8"), "fmt"), (dict(page_size=0), "positive")]:
        a = dict(num_pages=2, page_size=4, heads=2, head_size=64, device="cpu")
        a.update(kw)
        with pytest.raises(ValueError, match=msg):
            kvcache.make_kv_cache(**a)
    c = kvcache.make_kv_cache(2, 4, 2, 64, device="cpu")
    assert c[0].dtype == torch.float8_e4m3fn and tuple(c[2].shape) == (2, 4, 2, 1)
    m = kvcache.make_kv_cache(2, 4, 2, 64, "mxfp4", values=False, device="cpu")
    assert m[1] is None and tuple(m[0].shape) == (2, 4, 2, 32) and tuple(m[2].shape) == (2, 4, 2, 2)
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    slots = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA"):
        kvcache.write_kv_cache(k, k, slots, *c)
    with pytest.raises(RuntimeError, match="k_scale"):
        kvcache.write_kv_cache(k, k, slots, c[0], c[1], c[2][:1], c[3])
    with pytest.raises(RuntimeError, match="go together"):
        kvcache.write_kv_cache(k, k, slots, c[0], c[1], c[2], None)
    with pytest.raises(RuntimeError, match="v_cache must"):
        kvcache.write_kv_cache(k, k, slots, c[0], c[1][:1], c[2], c[3])
    with pytest.raises(RuntimeError, match="contiguous"):
        kvcache.write_kv_cache(k, k, slots, c[0].transpose(0, 1).contiguous().transpose(0, 1), *c[1:])


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float8_e5m2])
def test_oracle_rounds_as_torch_casts(dtype):
    """Every f32 with few significant bits in the types' range: the oracle's code is torch's cast."""
    y = np.concatenate([np.ldexp(np.arange(1, 256), e) for e in range(-30, 10)]).astype(np.float32)
    y = y[np.abs(y) <= O.MAX[dtype]]
    y = np.concatenate([y, -y, [0.0, -0.0]]).astype(np.float32)
    want = torch.from_numpy(y).to(dtype).view(torch.uint8).numpy()
    assert (O.nearest_code(y.astype(np.float64), dtype) == want).all()


def test_signatures_match_the_header():
    L = _lib.load()
    for name, n in (("emu_quant_fp8", 16), ("emu_gemm_fp8", 18), ("emu_kv_write", 18), ("emu_kv_read", 21)):
        assert len(getattr(L, name).argtypes) == n
        assert getattr(L, name).restype is ctypes.c_int32


def test_ops_fakes_give_the_layouts():
    from torch._subclasses.fake_tensor import FakeTensorMode

    import emugen_b200.ops  # noqa: F401

    with FakeTensorMode():
        x = torch.empty(7, 200, dtype=torch.bfloat16)
        q, s = torch.ops.emugen.quant_fp8(x)
        assert q.shape == (7, 200) and q.stride() == (208, 1) and s.shape == (7, 2) and s.stride() == (1, 8)
        w, ws = torch.ops.emugen.quant_fp8(torch.empty(300, 200, dtype=torch.bfloat16), "tile")
        assert ws.shape == (3, 2)
        out = torch.ops.emugen.gemm_fp8(q, w, s, ws, torch.float32)
        assert out.shape == (7, 300) and out.dtype == torch.float32
        c = torch.empty(4, 16, 2, 32, dtype=torch.uint8)
        k, v = torch.ops.emugen.read_kv_cache(c, c, c[..., :2], c[..., :2], torch.empty(1, 2, dtype=torch.int32),
                                              torch.empty(2, dtype=torch.int32), 9)
        assert k.shape == v.shape == (9, 2, 64)
