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
