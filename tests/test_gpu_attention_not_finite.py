"""Infinities and NaN that attention meets by right: they go where they belong, nothing else changes, and they cost no row-by-row work."""
import pytest
import torch

from emugen_b200 import _lib, attention
from tests import attention_oracle as O

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


def _make(n, Hq, Hk, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(n, h, D, generator=g).to(dtype).cuda() for h in (Hq, Hk, Hk, Hq)]


def _run(q, k, v, do, cu, causal=True):
    x = [t.detach().requires_grad_() for t in (q, k, v)]
    out = attention.packed_attention(*x, torch.tensor(cu, dtype=torch.int32, device="cuda"), causal=causal)
    grads = torch.autograd.grad(out, x, do)
    _lib.device_status()
    return out.detach(), *grads


def _rest(got, want, touched, name):
    """Everything but the places `touched` as in the oracle."""
    O.check(torch.where(touched, want[0], got.double()), want, name)


@pytest.mark.parametrize("heads", [(4, 2), (40, 20)], ids=str)         # one tile of rows to a CTA, and two
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", [INF, -INF, NAN])
@pytest.mark.parametrize("at", [0, 200, 299])
def test_a_value(heads, dtype, D, bad, at):
    """An element of a value: the same element of the queries that see it; those before it in the same tile keep theirs."""
    n = 300
    q, k, v, do = _make(n, *heads, D, dtype)
    want = O.attention(q, k, v, [0, n], [0, n], True, D ** -0.5, do)
    v2 = v.clone()
    v2[at, 0, 5] = bad
    out, dq, dk, dv = _run(q, k, v2, do, [0, n])
    group = heads[0] // heads[1]
    touched = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
    touched[at:, :group, 5] = True
    _rest(out, want["out"], touched, "out")
    got = out[touched]
    assert got.isnan().all() if bad != bad else (got == bad).all()
    # the queries that see it have no finite gradient; the others, and dv, which no value enters, are as they were
    rows = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
    rows[at:, :group] = True
    _rest(dq, want["dq"], rows, "dq")
    assert not dq[at:, :group].isfinite().any()
    O.check(dv, want["dv"], "dv")
    O.check(dk[:, 1:], tuple(t[:, 1:] for t in want["dk"]), "dk")


@pytest.mark.parametrize("heads", [(4, 2), (3, 3), (130, 1)], ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("what", ["do", "q"])
@pytest.mark.parametrize("at,causal", [(0, True), (70, True), (219, True), (100, False)])
def test_a_query_or_its_gradient(heads, dtype, what, at, causal):
    """One infinity in dO, one NaN in q, with a sequence on each side: the gradients of the keys that the query sees, and no others."""
    n, D = 220, 64
    cu = [0, 150, 150 + n, 150 + n + 70]
    q, k, v, do = _make(cu[-1], *heads, D, dtype, 1)
    want = O.attention(q, k, v, cu, cu, causal, D ** -0.5, do)
    t = 150 + at
    (do if what == "do" else q)[t, 0, 5] = INF if what == "do" else NAN
    out, dq, dk, dv = _run(q, k, v, do, cu, causal)
    seen = slice(150, t + 1 if causal else cu[2])
    row = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
    row[t, 0] = True
    keys = torch.zeros(dk.shape, dtype=torch.bool, device="cuda")
    keys[seen, 0] = True
    _rest(dq, want["dq"], row, "dq")
    assert not dq[t, 0].isfinite().any()
    _rest(dk, want["dk"], keys, "dk")
    assert not dk[keys].isfinite().any()
    if what == "do":
        O.check(out, want["out"], "out")
        keys[:, :, :5] = keys[:, :, 6:] = False
        assert (dv[keys] == INF).all()
    else:
        _rest(out, want["out"], row, "out")
        assert out[t, 0].isnan().all() and dv[keys].isnan().all()
    _rest(dv, want["dv"], keys, "dv")


@pytest.mark.parametrize("heads", [1, 160])
def test_values_near_the_end_of_bf16(heads):
    """Weights are held to the maximum up to 2^8: values near 2^127 leave f32's range beside them, the result does not."""
    n, D = 5, 64
    q = torch.zeros(n, heads, D, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros_like(q)
    q[..., 0], k[1:, :, 0] = 4, 10.0                                   # the first key at 0, the others 5 above it
    v = torch.full_like(q, 0.25)
    v[1] = 1e38
    out = attention.packed_attention(q, k, v, torch.tensor([0, n], dtype=torch.int32, device="cuda"), scale=0.125)
    want = O.attention(q, k, v, [0, n], [0, n], True, 0.125)["out"]
    O.check(out, want, "out")
    assert out[1].isfinite().all() and (out[1] > 9e37).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("what", ["do", "all of do", "v", "q"])
def test_they_cost_no_row_by_row_work(dtype, what):
    """2048 tokens: the products take half a millisecond, one row after the other 25 to 100; tenfold is far from both.  (Without the
    mask where all of dO is infinite: on the diagonal some of it would be hidden, and 0 times it is not by right.)"""
    n, Hq, Hk, D = 2048, 32, 8, 128
    causal = what != "all of do"
    q, k, v, do = _make(n, Hq, Hk, D, dtype, 2)

    def times(q, v, do):
        best = [1e9, 1e9]
        for _ in range(4):
            x = [t.detach().clone().requires_grad_() for t in (q, k, v)]
            e = [torch.cuda.Event(enable_timing=True) for _ in range(4)]
            c = torch.tensor([0, n], dtype=torch.int32, device="cuda")
            torch.cuda.synchronize()
            e[0].record()
            out = attention.packed_attention(*x, c, causal=causal)
            e[1].record()
            e[2].record()
            torch.autograd.grad(out, x, do)
            e[3].record()
            torch.cuda.synchronize()
            best = [min(best[0], e[0].elapsed_time(e[1])), min(best[1], e[2].elapsed_time(e[3]))]
        return best

    clean = times(q, v, do)
    q2, v2, do2 = q.clone(), v.clone(), do.clone()
    if what == "do":
        do2[n - 3, 1, 5] = INF
    elif what == "all of do":
        do2[:] = INF
    elif what == "v":
        v2[3, 1, 5] = INF
    else:
        q2[n - 3, 1, 5] = NAN
    got = times(q2, v2, do2)
    assert got[0] < 10 * clean[0] + 1 and got[1] < 10 * clean[1] + 1, (clean, got)


@pytest.mark.parametrize("heads", [(4, 1), (6, 6), (130, 1), (40, 20)], ids=str)
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.bfloat16, 40)])
@pytest.mark.parametrize("what", ["q", "k", "v", "do"])
@pytest.mark.parametrize("lens", [([300], [300]), ([30, 150, 9], [200, 150, 80]), ([260, 40], [70, 41])], ids=str)
def test_what_does_not_see_it_is_as_without_it(heads, dtype, D, what, lens):
    """NaN and infinities in the middle of sequences: rows of the same tiles that do not see them, against 64 bits without them."""
    Hq, Hk = heads
    nq, nk = lens
    cq, ck = ([0] + torch.tensor(n).cumsum(0).tolist() for n in lens)
    g = torch.Generator().manual_seed(D)
    x = [torch.randn(t, h, D, generator=g).to(dtype).cuda() for t, h in ((cq[-1], Hq), (ck[-1], Hk), (ck[-1], Hk), (cq[-1], Hq))]
    want = O.attention(*x[:3], cq, ck, True, D ** -0.5, x[3])
    queries, keys = torch.ones(cq[-1], Hq, dtype=torch.bool), torch.ones(ck[-1], Hk, dtype=torch.bool)
    group, bad = Hq // Hk, iter([NAN, INF, -INF, NAN, INF, -INF])
    x = [t.clone() for t in x]
    for s, (a, b) in enumerate(zip(nq, nk)):
        kh = Hk - 1
        if what in "kv":
            j = b // 2
            x["qkv".index(what)][ck[s] + j, kh, 3:] = next(bad)
            queries[cq[s] + max(0, j - (b - a)):cq[s + 1], kh * group:] = False
            if j - (b - a) < a:
                keys[ck[s]:ck[s + 1], kh] = False
        else:
            i = a // 2
            x[0 if what == "q" else 3][cq[s] + i, Hq - 1, 3:] = next(bad)
            queries[cq[s] + i, Hq - 1] = False
            keys[ck[s]:ck[s] + min(b, max(0, i + 1 + b - a)), kh] = False
    y = [t.requires_grad_() for t in x[:3]]
    out = attention.packed_attention(*y, *(torch.tensor(c, dtype=torch.int32, device="cuda") for c in (cq, ck)))
    dq, dk, dv = torch.autograd.grad(out, y, x[3])
    _lib.device_status()
    queries, keys = (~t.cuda()[..., None].expand(-1, -1, D) for t in (queries, keys))
    _rest(out, want["out"], torch.zeros_like(queries) if what == "do" else queries, "out")
    _rest(dq, want["dq"], queries, "dq")
    _rest(dk, want["dk"], keys, "dk")
    _rest(dv, want["dv"], torch.zeros_like(keys) if what == "v" else keys, "dv")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_are_made_again_together(dtype):
    """One infinity in the middle of dO: the keys behind it in its tile are made again from half of the queries, 8 at a time (2048 tokens
    about 3.5 ms beside 0.3; one after the other 46)."""
    n, Hq, Hk, D = 2048, 32, 8, 128
    q, k, v, do = _make(n, Hq, Hk, D, dtype, 3)
    x = [t.requires_grad_() for t in (q, k, v)]
    c = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    times = []
    for place in (None, n // 2 + 2):
        d = do.clone()
        if place:
            d[place, 1, 5] = INF
        best = 1e9
        for _ in range(4):
            out = attention.packed_attention(*x, c)
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            torch.cuda.synchronize()
            a.record()
            torch.autograd.grad(out, x, d)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        times.append(best)
    assert times[1] < 40 * times[0] + 2, times
