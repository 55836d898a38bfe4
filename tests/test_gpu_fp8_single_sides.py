"""One side alone: the quantiser's transposed form by itself (C entry, q NULL) and backward passes that want one
gradient, bit for bit what the full forms give."""
import pytest
import torch

from emugen_b200 import _lib, fp8
from tests.test_gpu_fp8 import E4, E5, _check, _x

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,K", [(1, 1), (5, 129), (127, 300), (257, 513), (130, 256)])
@pytest.mark.parametrize("block", ["row", "tile"])
@pytest.mark.parametrize("dtype", [E4, E5])
@pytest.mark.parametrize("xt", [torch.bfloat16, torch.float16, torch.float32])
def test_transposed_codes_alone(M, K, block, dtype, xt):
    x = _x(M, K, xt, seed=M + K)
    xc = x.cuda()
    kb, mb = -(-K // 128), -(-M // 128)
    ldqt = -(-M // 16) * 16
    qt = torch.full((K + 1, ldqt), 0xCD, dtype=torch.uint8, device="cuda")
    st = torch.full((mb, K) if block == "row" else (kb, mb), 9.0, device="cuda")
    rc = _lib.load().emu_quant_fp8(xc.data_ptr(), fp8._DTYPE[xt], M, K, K, fp8._FP8[dtype], fp8._BLOCKS[block], None, 0, None, 0,
                                   qt.data_ptr(), ldqt, st.data_ptr(), st.shape[1], torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    _check(x.t(), block, dtype, qt[:K, :M].view(dtype), st.t() if block == "row" else st)
    assert (qt[K] == 0xCD).all() and (qt[:, M:] == 0xCD).all()


@pytest.mark.parametrize("M,N,K", [(1, 40, 72), (33, 130, 200), (301, 500, 257), (700, 1100, 640)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_one_gradient_is_the_full_pass_s(M, N, K, dtype):
    g = torch.Generator().manual_seed(M)
    x, w, dy = [torch.randn(s, generator=g).to(dtype).cuda() for s in ((M, K), (N, K), (M, N))]
    p, q = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = fp8.linear_fp8(p, q)
    want = torch.autograd.grad(y, (p, q), dy)
    a = x.clone().requires_grad_()
    ya = fp8.linear_fp8(a, w)
    dx, = torch.autograd.grad(ya, a, dy)
    b = w.clone().requires_grad_()
    yb = fp8.linear_fp8(x, b)
    dw, = torch.autograd.grad(yb, b, dy)
    assert torch.equal(ya, y) and torch.equal(yb, y)
    assert torch.equal(dx, want[0]) and torch.equal(dw, want[1])


def test_weight_gradient_alone_launches_no_row_quantiser(monkeypatch):
    """Where only the weight's gradient is wanted, dy's row codes, which dx alone would use, are not made."""
    x = torch.randn(64, 128, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(96, 128, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = fp8.linear_fp8(x, w)
    seen = []
    real = _lib.load()

    class Spy:
        def __getattr__(self, name):
            return getattr(real, name)

        def emu_quant_fp8(self, *a):
            seen.append((a[7], a[11]))                 # q and qt
            return real.emu_quant_fp8(*a)

    monkeypatch.setattr(_lib, "load", lambda: Spy())
    y.backward(torch.ones_like(y))
    assert len(seen) == 1 and seen[0][0] is None and seen[0][1]
