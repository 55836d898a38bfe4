"""Attention's gradients in fp16 where sequences, heads and rows differ much in size: what one of them rounds to does not depend on the
others."""
import pytest
import torch

from emugen_b200 import _lib, attention
from tests import attention_oracle as O

pytestmark = pytest.mark.gpu


def _randn(g, t, h, d, f=1.0):
    return (f * torch.randn(t, h, d, generator=g)).half().cuda()


def _grads(q, k, v, cu_q, cu_k, causal, do):
    x = [t.detach().requires_grad_() for t in (q, k, v)]
    c = [torch.tensor(c, dtype=torch.int32, device="cuda") for c in (cu_q, cu_k)]
    r = torch.autograd.grad(attention.packed_attention(*x, *c, causal=causal), x, do)
    _lib.device_status()
    return r


def _check(got, want, name):
    """As O.check; a value that is within its tolerance of 65520, half a step past fp16's largest, may also round to infinity."""
    value, tol = want
    past = got.double().isinf() & (got.double().sign() == value.sign()) & (value.abs() + tol >= 65520)
    O.check(torch.where(past, value, got.double()), want, name)


@pytest.mark.parametrize("lens", [([1500, 70], [1500, 70]), ([40, 130, 0, 900], [300, 130, 5, 1900])], ids=str)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("Hq,Hk,D", [(4, 2, 64), (3, 3, 128), (6, 1, 40)])
def test_a_sequence_beside_one_with_far_larger_gradients(lens, causal, Hq, Hk, D):
    """The first sequence's dO and v are 2^22 times the others' in their product: each against 64 bits."""
    g = torch.Generator().manual_seed(D)
    nq, nk = lens
    parts = []
    for i, (a, b) in enumerate(zip(nq, nk)):
        f, e = (2.0 ** 8, 2.0 ** 6) if i == 0 else (2.0 ** -6, 2.0 ** -2)
        parts.append((_randn(g, a, Hq, D, 2.0 ** -4), _randn(g, b, Hk, D, 2.0 ** 4), _randn(g, b, Hk, D, e), _randn(g, a, Hq, D, f)))
    q, k, v, do = (torch.cat(t) for t in zip(*parts))
    cu_q, cu_k = ([0] + torch.tensor(n).cumsum(0).tolist() for n in lens)
    want = O.attention(q, k, v, cu_q, cu_k, causal, D ** -0.5, do)
    for name, got in zip(("dq", "dk", "dv"), _grads(q, k, v, cu_q, cu_k, causal, do)):
        _check(got, want[name], name)


@pytest.mark.parametrize("axis", ["rows", "heads", "key heads"])
def test_scaled_gradients_scale(axis):
    """dO 2^20 times smaller in some rows, or heads: their gradients are smaller by exactly that, up to fp16's normal numbers."""
    n, Hq, Hk, D, f = 1000, 4, 2, 64, 2.0 ** -20
    g = torch.Generator().manual_seed(7)
    q, k, v, do = _randn(g, n, Hq, D), _randn(g, n, Hk, D), _randn(g, n, Hk, D), _randn(g, n, Hq, D, 2.0 ** 13)
    some = torch.zeros(n, Hq, 1, dtype=torch.bool, device="cuda")
    some[{"rows": slice(1, None, 3), "heads": (slice(None), slice(0, 1)), "key heads": (slice(None), slice(2, 4))}[axis]] = True
    small = torch.where(some, (do.float() * f).half(), do)
    do = torch.where(some, (small.float() / f).half(), do)       # (as the smaller one was rounded)
    cu = [0, n]
    want, got = _grads(q, k, v, cu, cu, True, do), _grads(q, k, v, cu, cu, True, small)
    scaled = torch.where(some, want[0].double() * f, want[0].double())
    normal = scaled.abs() >= 2.0 ** -14
    assert int((normal & some).sum()) > 1000 and torch.equal(got[0].double()[normal], scaled[normal])
    if axis == "key heads":
        for a, b in zip(got[1:], want[1:]):
            b = b[:, 1].double() * f
            normal = b.abs() >= 2.0 ** -14
            assert int(normal.sum()) > 1000 and torch.equal(a[:, 1].double()[normal], b[normal])
            assert torch.equal(a[:, 0], want[1 if a is got[1] else 2][:, 0])
