"""Attention of one token over the quantised cache with a first key far above the rest and recent keys above old ones, against 64
bits on the rows as they are stored."""
import pytest
import torch

from emugen_b200 import kvcache
from tests import attention_oracle as O
from tests.test_gpu_kv_attend import _want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", ["first", "recent", "both"])
@pytest.mark.parametrize("lens", [[16385], [4000, 77, 900]], ids=str)
def test_peaked_rows(fmt, dtype, shape, lens):
    Hq, Hk, D, page = 8, 2, 64, 16
    g = torch.Generator().manual_seed(5)
    cols = (max(lens) + page - 1) // page
    table = torch.randperm(len(lens) * cols, generator=g).to(torch.int32).view(len(lens), cols)
    cache = kvcache.make_kv_cache(len(lens) * cols, page, Hk, D, fmt)
    for b, n in enumerate(lens):
        pos = torch.arange(n)
        bonus = pos * (20.0 / n) if shape != "first" else torch.zeros(n)
        if shape != "recent":
            bonus[0] = bonus[-1] + 14
        k, v = (torch.randn(n, Hk, D, generator=g) for _ in range(2))
        k, v = 0.3 * k, 1 + 0.25 * v
        k[..., 0] = bonus[:, None] * D ** 0.5 / 4
        v[0] = 0
        slots = table[b].long()[pos // page] * page + pos % page
        kvcache.write_kv_cache(k.to(dtype).cuda(), v.to(dtype).cuda(), slots.cuda(), *cache)
    q = 0.3 * torch.randn(len(lens), Hq, D, generator=g)
    q[..., 0] = 4
    q, table, n = q.to(dtype).cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    out, lse = kvcache.attend_kv_cache(q, *cache, table, n, return_lse=True)
    o, l = _want(q, cache, table, n, fmt, D ** -0.5, page)
    O.check(out, o, "out")
    O.check(lse, l, "lse")
