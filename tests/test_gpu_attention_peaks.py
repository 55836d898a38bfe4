"""Attention with scores as trained models have them, against 64 bits: even ones with a key far above the rest late in the sequence,
a first key that has nearly all of the weight, recent keys above old ones."""
import pytest
import torch

from emugen_b200 import _lib, attention
from tests import attention_oracle as O

pytestmark = pytest.mark.gpu


def _scored(n, bonus, D, dtype, seed, Hq=2, Hk=1):
    """q, k, v of n tokens whose scores are small random numbers plus bonus[key]."""
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(n, h, D, generator=g) for h in (Hq, Hk, Hk))
    q, k = 0.3 * q, 0.3 * k
    q[..., 0] = 4
    k[..., 0] = bonus[:, None] * D ** 0.5 / 4
    return [t.to(dtype).cuda() for t in (q, k, v)]


def _cu(n):
    return torch.tensor([0, n], dtype=torch.int32, device="cuda")


def _check(q, k, v, causal, do=None):
    n = q.shape[0]
    x = [t.detach().requires_grad_(do is not None) for t in (q, k, v)]
    out, lse = attention.packed_attention(*x, _cu(n), causal=causal, return_lse=True)
    want = O.attention(q, k, v, [0, n], [0, n], causal, q.shape[2] ** -0.5, do)
    O.check(out, want["out"], "out")
    O.check(lse, want["lse"], "lse")
    if do is not None:
        for name, got in zip(("dq", "dk", "dv"), torch.autograd.grad(out, x, do)):
            O.check(got, want[name], name)
    _lib.device_status()                              # no wait ran out


@pytest.mark.parametrize("tile", [1, 2, 3, 4, 5, 6])
@pytest.mark.parametrize("D", [16, 64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads", [2, 40])             # one tile of rows to a CTA, and two
def test_even_tiles_and_then_a_higher_one(tile, D, causal, heads):
    """The maximum stays for `tile` tiles of 128 keys and then grows by more than 2^8, for one key or for all from there on."""
    n = 900
    for late in (slice(128 * tile + 3, 128 * tile + 4), slice(128 * tile, n)):
        for rise, dtype in ((7.0, torch.float16), (7.0, torch.bfloat16), (40.0, torch.bfloat16)):
            bonus = torch.zeros(n)
            bonus[late] = rise
            _check(*_scored(n, bonus, D, dtype, tile, heads, heads // 2), causal)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("above", [10.0, 14.0, 16.0, 17.0, 18.0])
@pytest.mark.parametrize("heads", [2, 160])            # one tile of rows to a CTA, and two
def test_a_first_key_above_the_rest(dtype, above, heads):
    """A key without a value has nearly all of the weight; the output is what the weights of the 16384 others, down to 2^-26,
    leave of theirs."""
    nq, nk, D = 64, 16385, 64
    bonus = torch.zeros(nk)
    bonus[0] = above
    q, k, v = _scored(nk, bonus, D, dtype, int(above), heads, heads // 2)
    q, v = q[:nq].contiguous(), (1 + 0.25 * v.float()).to(dtype)
    v[0] = 0
    out, lse = attention.packed_attention(q, k, v, _cu(nq), _cu(nk), causal=False, return_lse=True)
    want = O.attention(q, k, v, [0, nq], [0, nk], False, D ** -0.5)
    O.check(out, want["out"], "out")
    O.check(lse, want["lse"], "lse")
    _lib.device_status()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", ["first", "recent", "both"])
@pytest.mark.parametrize("heads", [2, 40])
@pytest.mark.parametrize("causal", [True, False])
def test_gradients_of_peaked_rows(dtype, shape, heads, causal):
    """A first key 9 above the rest, and scores that rise by 1 every 32 keys, so that the recent ones are far above the old."""
    n, D = 700, 64
    bonus = torch.arange(n) / 32.0 if shape != "first" else torch.zeros(n)
    if shape != "recent":
        bonus[0] = bonus[-1] + 9
    q, k, v = _scored(n, bonus, D, dtype, 3, heads, heads // 2)
    do = torch.randn(q.shape, generator=torch.Generator().manual_seed(4)).to(dtype).cuda()
    _check(q, k, v, causal, do)
