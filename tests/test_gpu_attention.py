"""Attention over packed sequences on the GPU against 64 bits: forward, gradients, masks, lengths, layouts."""
import pytest
import torch

from emugen_b200 import attention
from tests import attention_oracle as O

pytestmark = pytest.mark.gpu


def _cu(lens):
    c = [0]
    for n in lens:
        c.append(c[-1] + n)
    return c


def _make(nq, nk, Hq, Hk, D, dtype, seed, extra=0, peak=1.0):
    g = torch.Generator().manual_seed(seed)
    tq, tk = sum(nq) + extra, sum(nk) + extra
    q, k, v, do = ((torch.randn(t, h, D, generator=g) * torch.exp(0.4 * torch.randn(1, h, D, generator=g))).to(dtype).cuda()
                   for t, h in ((tq, Hq), (tk, Hk), (tk, Hk), (tq, Hq)))
    q = (q.float() * peak).to(dtype)
    return q, k, v, do


def _tensor(c):
    return torch.tensor(c, dtype=torch.int32, device="cuda")


def _check(nq, nk, Hq, Hk, D, dtype, causal, seed=0, scale=None, peak=1.0, extra=0, back=True):
    q, k, v, do = _make(nq, nk, Hq, Hk, D, dtype, seed, extra, peak)
    cq, ck = _cu(nq), _cu(nk)
    if back:
        for t in (q, k, v):
            t.requires_grad_()
    out, lse = attention.packed_attention(q, k, v, _tensor(cq), _tensor(ck), causal=causal, scale=scale, return_lse=True)
    want = O.attention(q, k, v, cq, ck, causal, D ** -0.5 if scale is None else scale, do if back else None)
    O.check(out, want["out"], "out")
    O.check(lse, want["lse"], "lse")
    if back:
        for name, got in zip(("dq", "dk", "dv"), torch.autograd.grad(out, (q, k, v), do)):
            O.check(got, want[name], name)


LENGTHS = [
    ([1], [1]), ([5], [5]), ([0, 3, 0, 1], [2, 0, 0, 7]), ([128], [128]), ([127, 1, 129], [127, 1, 129]), ([300], [300]),
    ([64, 200], [190, 3]), ([17], [1000]), ([513, 0, 40], [513, 5, 41]), ([257], [256]), ([1, 1, 1], [129, 257, 1]), ([700], [20]),
]


@pytest.mark.parametrize("lens", LENGTHS, ids=str)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_lengths(lens, causal, dtype):
    _check(*lens, 4, 2, 64, dtype, causal, seed=len(lens[0]))


@pytest.mark.parametrize("D", [8, 16, 24, 40, 56, 64, 72, 80, 96, 104, 120, 128])
@pytest.mark.parametrize("Hq,Hk", [(1, 1), (6, 2), (8, 1), (3, 3)])
@pytest.mark.parametrize("causal", [True, False])
def test_head_sizes_and_groups(D, Hq, Hk, causal):
    _check([70, 150, 3], [70, 150, 9], Hq, Hk, D, torch.bfloat16 if D % 16 else torch.float16, causal, seed=D)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,causal", [(1000, True), (2049, True), (1531, False)])
def test_long(dtype, n, causal):
    _check([n], [n], 4, 2, 128, dtype, causal, seed=n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_sequences(dtype):
    lens = [(7 * i) % 31 for i in range(150)]
    _check(lens, [n + (i % 3) for i, n in enumerate(lens)], 2, 1, 64, dtype, True, seed=5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("peak,scale", [(30.0, None), (1.0, 1.5), (0.01, None), (1.0, 1e-4)])
def test_peaked_and_flat_scores(dtype, peak, scale):
    """Rows where one key has nearly all of the weight, maxima that keep rising, and nearly uniform ones."""
    _check([400], [400], 2, 2, 64, dtype, True, seed=9, peak=peak, scale=scale)


def test_rising_scores():
    """Each key scores above all before it, far enough that every tile moves the running maximum."""
    D, n = 64, 900
    q = torch.zeros(n, 1, D, device="cuda", dtype=torch.bfloat16)
    q[..., 0] = 8
    k = torch.zeros_like(q)
    k[:, 0, 0] = torch.linspace(-200, 200, n, device="cuda").to(torch.bfloat16)
    v = torch.randn(n, 1, D, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(torch.bfloat16)
    c = [0, n]
    for flip in (False, True):
        kk = k.flip(0).contiguous() if flip else k
        out = attention.packed_attention(q, kk, v, _tensor(c), scale=0.5)
        O.check(out, O.attention(q, kk, v, c, c, True, 0.5)["out"], "out")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_small_gradients_in_fp16(dtype):
    """Gradients far below and above one: what is rounded on the way stays in the type's range."""
    for factor in (2.0 ** -14, 2.0 ** 9):
        q, k, v, do = _make([300], [300], 4, 2, 64, dtype, 4)
        do = (do.float() * factor).to(dtype)
        for t in (q, k, v):
            t.requires_grad_()
        c = [0, 300]
        out = attention.packed_attention(q, k, v, _tensor(c))
        want = O.attention(q, k, v, c, c, True, 64 ** -0.5, do)
        for name, got in zip(("dq", "dk", "dv"), torch.autograd.grad(out, (q, k, v), do)):
            O.check(got, want[name], name)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_hidden_places_reach_nothing(bad, dtype):
    """NaN and infinities in keys and values that a query does not see, in queries that see no key, in their gradients and
    behind the last sequence."""
    nq, nk, Hq, Hk, D = [150, 10, 40], [150, 4, 40], 2, 1, 64
    q, k, v, do = _make(nq, nk, Hq, Hk, D, dtype, 3, extra=20)
    cq, ck = _cu(nq), _cu(nk)
    clean = [t.clone() for t in (q, k, v, do)]
    for t in (q, do):
        t[cq[1]:cq[1] + 6] = bad                      # see no key (10 queries, 4 keys)
        t[cq[-1]:] = bad
    for t in (k, v):
        t[ck[-1]:] = bad
    # the last sequence's last key and value: its last query alone sees them
    k2, v2 = k.clone(), v.clone()
    k2[ck[-1] - 1] = bad
    v2[ck[-1] - 1] = bad
    for kk, vv, rows in ((k, v, cq[-1]), (k2, v2, cq[-1] - 1)):
        x = [t.clone().requires_grad_() for t in (q, kk, vv)]
        out = attention.packed_attention(*x, _tensor(cq), _tensor(ck))
        want = O.attention(*clean[:3], cq, ck, True, D ** -0.5, clean[3])
        O.check(out[:rows], tuple(w[:rows] for w in want["out"]), "out")
        assert (out[cq[-1]:] == 0).all() and (out[cq[1]:cq[1] + 6] == 0).all()
        g = torch.autograd.grad(out, x, do)
        O.check(g[0][:rows], tuple(w[:rows] for w in want["dq"]), "dq")
        assert (g[0][cq[-1]:] == 0).all() and (g[0][cq[1]:cq[1] + 6] == 0).all()
        assert (g[1][ck[-1]:] == 0).all() and (g[2][ck[-1]:] == 0).all()
        keys = ck[-1] if rows == cq[-1] else ck[2]     # the other sequences' gradients are untouched by the bad key
        for name, t in (("dk", g[1]), ("dv", g[2])):
            O.check(t[:keys], tuple(w[:keys] for w in want[name]), name)


@pytest.mark.parametrize("causal", [True, False])
def test_seen_nan_spreads_where_it_should(causal):
    n, D = 300, 64
    q, k, v, _ = _make([n], [n], 2, 1, D, torch.bfloat16, 8)
    v[200, 0, 5] = float("nan")
    out = attention.packed_attention(q, k, v, _tensor([0, n]), causal=causal)
    first = 200 if causal else 0
    nan = out.isnan()
    assert nan[first:, :, 5].all() and int(nan.sum()) == (n - first) * 2


def test_layouts():
    """Slices of a fused projection, heads before tokens, rows that start off 16 bytes, expanded gradients: the same bits."""
    T, Hq, Hk, D = 333, 4, 2, 72
    q, k, v, do = _make([T], [T], Hq, Hk, D, torch.bfloat16, 11)
    c = _tensor([0, 100, T])

    def run(q, k, v, do):
        x = [t.detach().requires_grad_() for t in (q, k, v)]
        out = attention.packed_attention(*x, c)
        return (out.detach(), *torch.autograd.grad(out, x, do))

    want = run(q, k, v, do)
    fused = torch.cat([q, k, v], 1)
    odd = torch.empty(T * Hq * D + 1, dtype=q.dtype, device="cuda")[1:].view(T, Hq, D).copy_(q)
    heads_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v, do)]
    wide = [torch.empty(T, t.shape[1], D + 4, dtype=t.dtype, device="cuda")[..., :D].copy_(t) for t in (q, k, v, do)]
    columns = [t.permute(2, 0, 1).contiguous().permute(1, 2, 0) for t in (q, k, v, do)]
    for args in ((fused[:, :Hq], fused[:, Hq:Hq + Hk], fused[:, Hq + Hk:], do), (odd, k, v, do), heads_first, wide, columns):
        for a, b in zip(run(*args), want):
            assert torch.equal(a, b)
    one = do[:1, :1, :1].expand(T, Hq, D)
    for a, b in zip(run(q, k, v, one), run(q, k, v, one.contiguous())):
        assert torch.equal(a, b)


def test_same_result_every_run():
    q, k, v, do = _make([700, 333], [700, 333], 8, 2, 128, torch.bfloat16, 12)
    c = _tensor([0, 700, 1033])
    runs = []
    for _ in range(3):
        x = [t.detach().requires_grad_() for t in (q, k, v)]
        out = attention.packed_attention(*x, c)
        runs.append((out.detach(), *torch.autograd.grad(out, x, do)))
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


def test_wanted_gradients_alone():
    q, k, v, do = _make([200], [200], 4, 2, 64, torch.bfloat16, 13)
    c = _tensor([0, 200])
    x = [t.detach().requires_grad_() for t in (q, k, v)]
    want = torch.autograd.grad(attention.packed_attention(*x, c), x, do)
    for wanted in ((0,), (1,), (2,), (0, 2)):
        x = [t.detach().requires_grad_(i in wanted) for i, t in enumerate((q, k, v))]
        got = torch.autograd.grad(attention.packed_attention(*x, c), [x[i] for i in wanted], do)
        for i, t in zip(wanted, got):
            assert torch.equal(t, want[i])


def test_gradients_against_differences():
    """The loss along random directions: central differences of the forward pass in 64 bits."""
    nq, nk, Hq, Hk, D = [40, 9], [50, 9], 4, 2, 32
    q, k, v, do = _make(nq, nk, Hq, Hk, D, torch.bfloat16, 14)
    cq, ck = _cu(nq), _cu(nk)
    x = [t.detach().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(attention.packed_attention(*x, _tensor(cq), _tensor(ck)), x, do)
    want = O.attention(q, k, v, cq, ck, True, D ** -0.5, do)

    def loss(t):
        return float((O.attention(*t, cq, ck, True, D ** -0.5)["out"][0] * do.double()).sum())

    g = torch.Generator(device="cuda").manual_seed(2)
    for i, name in enumerate(("dq", "dk", "dv")):
        r = torch.randn(x[i].shape, generator=g, device="cuda", dtype=torch.float64)
        e = 2.0 ** -14
        plus, minus = ([t.detach().double() + (e * r if j == i else 0) * s for j, t in enumerate((q, k, v))] for s in (1, -1))
        # the oracle takes 16-bit tensors' types for its tolerances alone
        slope = (_loss64(plus, do, cq, ck, D) - _loss64(minus, do, cq, ck, D)) / (2 * e)
        tol = float((want[name][1] * r.abs()).sum()) + 1e-6 * abs(slope) + 1e-4
        assert abs(float((grads[i].double() * r).sum()) - slope) <= tol, name


def _loss64(t, do, cq, ck, D):
    q, k, v = t
    total = 0.0
    for s in range(len(cq) - 1):
        nq, nk = cq[s + 1] - cq[s], ck[s + 1] - ck[s]
        seen = torch.arange(nk, device="cuda")[None] <= torch.arange(nq, device="cuda")[:, None] + nk - nq
        for h in range(q.shape[1]):
            g = h * k.shape[1] // q.shape[1]
            x = (q[cq[s]:cq[s + 1], h] @ k[ck[s]:ck[s + 1], g].t() * D ** -0.5).masked_fill(~seen, float("-inf"))
            total += float((torch.softmax(x, 1) @ v[ck[s]:ck[s + 1], g] * do[cq[s]:cq[s + 1], h].double()).sum())
    return total


def test_streams_and_graph_replay():
    """Two streams at once, and a captured forward and backward pass that is replayed on new inputs."""
    q, k, v, do = _make([500], [500], 4, 2, 64, torch.bfloat16, 15)
    c = _tensor([0, 123, 500])

    def run(q, k, v):
        x = [t.detach().requires_grad_() for t in (q, k, v)]
        out = attention.packed_attention(*x, c)
        return (out.detach(), *torch.autograd.grad(out, x, do))

    want = run(q, k, v)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append([run(q, k, v) for _ in range(3)])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for per in got for r in per for a, b in zip(r, want))
    q2 = q.flip(0).contiguous()
    want2 = run(q2, k, v)
    static = q.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(static, k, v)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = run(static, k, v)
    for source, w in ((q, want), (q2, want2)):
        static.copy_(source)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(r, w))


def test_fresh_thread():
    """A thread whose first CUDA work is this call."""
    import threading

    q, k, v, _ = _make([90], [90], 4, 2, 64, torch.bfloat16, 16)
    c = _tensor([0, 90])
    want = attention.packed_attention(q, k, v, c)
    torch.cuda.synchronize()
    got = []
    t = threading.Thread(target=lambda: got.append(attention.packed_attention(q, k, v, c)))
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want)


def test_empty_calls():
    for tq, tk, B in ((0, 0, 0), (0, 5, 1), (6, 0, 1), (6, 5, 0)):
        q = torch.randn(tq, 4, 64, device="cuda", dtype=torch.float16, requires_grad=True)
        k, v = (torch.randn(tk, 2, 64, device="cuda", dtype=torch.float16, requires_grad=True) for _ in range(2))
        cq, ck = _tensor([0] + [tq] * B), _tensor([0] + [tk] * B)
        out, lse = attention.packed_attention(q, k, v, cq, ck, return_lse=True)
        assert out.shape == q.shape and (out == 0).all() and (lse == float("-inf")).all()
        for t, g in zip((q, k, v), torch.autograd.grad(out, (q, k, v), torch.ones_like(out))):
            assert g.shape == t.shape and (g == 0).all()


def test_registered_operator():
    import emugen_b200.ops  # noqa: F401

    q, k, v, _ = _make([90], [90], 4, 2, 64, torch.bfloat16, 16)
    c = _tensor([0, 90])
    want = attention.packed_attention(q, k, v, c, causal=False)
    assert torch.equal(torch.ops.emugen.packed_attention(q, k, v, c, None, False), want)
    fn = torch.compile(lambda *a: torch.ops.emugen.packed_attention(*a, None, False), fullgraph=True, backend="aot_eager")
    assert torch.equal(fn(q, k, v, c), want)


# Calls with so many (sequence, key head) pairs of tiles that a CTA takes two of them: the tests above take one.
WIDE = dict(Hq=128, Hk=64)


@pytest.mark.parametrize("lens", [([300], [300]), ([0, 3, 0, 130], [2, 0, 0, 7]), ([127, 1, 129], [127, 1, 129]), ([64, 200], [190, 3]),
                                  ([9], [1000]), ([257, 30], [256, 30]), ([70] * 5, [70, 69, 71, 0, 140])], ids=str)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.bfloat16, 40), (torch.float16, 104)])
def test_two_tiles_to_a_cta(lens, causal, dtype, D):
    _check(*lens, **WIDE, D=D, dtype=dtype, causal=causal, seed=len(lens[0]), back=D == 40)


@pytest.mark.parametrize("peak,scale", [(30.0, None), (1.0, 1.5), (1.0, 1e-4)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_two_tiles_peaked_and_flat(dtype, peak, scale):
    _check([520], [520], 80, 80, 64, dtype, True, seed=9, peak=peak, scale=scale, back=False)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("D", [64, 128])
def test_two_tiles_hidden_places(bad, D):
    nq, nk, Hq, Hk = [150, 10, 140], [150, 4, 140], 64, 64
    q, k, v, _ = _make(nq, nk, Hq, Hk, D, torch.bfloat16, 3, extra=20)
    cq, ck = _cu(nq), _cu(nk)
    want = O.attention(q, k, v, cq, ck, True, D ** -0.5)
    q, k, v = (t.clone() for t in (q, k, v))
    q[cq[1]:cq[1] + 6] = bad
    q[cq[-1]:] = bad
    for t in (k, v):
        t[ck[-1] - 1:] = bad                           # the last query alone sees the last key
    out = attention.packed_attention(q, k, v, _tensor(cq), _tensor(ck))
    O.check(out[:cq[-1] - 1], tuple(w[:cq[-1] - 1] for w in want["out"]), "out")
    assert (out[cq[-1]:] == 0).all() and (out[cq[1]:cq[1] + 6] == 0).all() and out[cq[-1] - 1].isnan().all()


def test_two_tiles_layouts_and_replay():
    """Slices of a fused projection and heads before tokens, on another stream and replayed: the same bits."""
    T, Hq, Hk, D = 300, 128, 64, 64
    q, k, v, _ = _make([T], [T], Hq, Hk, D, torch.bfloat16, 11)
    c = _tensor([0, 101, T])
    want = attention.packed_attention(q, k, v, c)
    fused = torch.cat([q, k, v], 1)
    parts = fused[:, :Hq], fused[:, Hq:Hq + Hk], fused[:, Hq + Hk:]
    assert torch.equal(attention.packed_attention(*parts, c), want)
    assert torch.equal(attention.packed_attention(*(t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)), c), want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attention.packed_attention(*parts, c)
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("Hq,Hk,T", [(130, 1, 40), (200, 1, 400), (258, 2, 33)])
def test_groups_of_more_than_a_tile(Hq, Hk, T):
    """More query heads to a key head than a tile has rows."""
    _check([T - 7, 7], [T - 7, 7], Hq, Hk, 64, torch.bfloat16, True, seed=T, back=T < 100)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_delta_from_the_output_before_its_rounding(dtype):
    """Two keys of equal weight whose values have much in common: p is exact, the output's rounding is far above the
    differences dp - delta, and dq has to come out to its own roundings all the same."""
    n, D = 64, 128
    g = torch.Generator().manual_seed(6)
    q = torch.zeros(2 * n, 2, D, dtype=dtype, device="cuda")
    k = torch.randn(2 * n, 2, D, generator=g).to(dtype).cuda()
    v = (100 + torch.randn(2 * n, 2, D, generator=g)).to(dtype).cuda()
    do = torch.randn(2 * n, 2, D, generator=g).to(dtype).cuda()
    cu = list(range(0, 2 * n + 1, 2))
    x = [t.requires_grad_() for t in (q, k, v)]
    out = attention.packed_attention(*x, _tensor(cu), causal=False)
    want = O.attention(q, k, v, cu, cu, False, D ** -0.5, do, p_step=0)
    O.check(out, want["out"], "out")
    for name, got in zip(("dq", "dk", "dv"), torch.autograd.grad(out, x, do)):
        O.check(got, want[name], name)


@pytest.mark.parametrize("heads,what", [(4, "forward"), (128, "forward"), (4, "gradients")])
def test_timed_out_wait_is_reported_and_the_context_survives(heads, what):
    """A tile of scores that is never announced: the kernel gives up and returns, the next query of the device's status
    tells, and the next call is right."""
    from emugen_b200 import _lib

    L = _lib.load()
    q, k, v, do = _make([200], [200], heads, heads, 64, torch.bfloat16, 17)
    c = _tensor([0, 200])
    x = [t.requires_grad_() for t in (q, k, v)]

    def run():
        out = attention.packed_attention(*x, c)
        return out, torch.autograd.grad(out, x, do)

    want = run()
    torch.cuda.synchronize()
    _lib.device_status()
    out = attention.packed_attention(*x, c)
    torch.cuda.synchronize()
    prev = _lib.set_wait_limit(1 << 20)
    L.emu_test_hold_first_ready(1)
    try:
        if what == "forward":
            with torch.no_grad():
                attention.packed_attention(q, k, v, c)
        else:
            torch.autograd.grad(out, x, do)
        with pytest.raises(_lib.EmuError) as err:
            _lib.device_status()
        assert err.value.status == _lib.EMU_ERR_TIMEOUT and "wait ran out" in str(err.value)
        _lib.device_status()
    finally:
        L.emu_test_hold_first_ready(0)
        _lib.set_wait_limit(prev)
    got = run()
    _lib.device_status()
    assert torch.equal(got[0], want[0]) and all(torch.equal(a, b) for a, b in zip(got[1], want[1]))


def test_offsets_past_32_bits():
    """Tensors of more than 2^31 elements: the last sequences as on their own."""
    T, Hq, Hk, D, n = 135000, 128, 8, 128, 100
    g = torch.Generator(device="cuda").manual_seed(3)
    q, do = (torch.randn(T, Hq, D, device="cuda", dtype=torch.bfloat16, generator=g) for _ in range(2))
    k, v = (torch.randn(T, Hk, D, device="cuda", dtype=torch.bfloat16, generator=g) for _ in range(2))
    assert q.numel() > 2 ** 31
    x = [t.requires_grad_() for t in (q, k, v)]
    out = attention.packed_attention(*x, _tensor(list(range(0, T + 1, n))))
    grads = torch.autograd.grad(out, x, do)
    tail = [t[-2 * n:].detach() for t in x]
    want = O.attention(*tail, [0, n, 2 * n], [0, n, 2 * n], True, D ** -0.5, do[-2 * n:])
    O.check(out[-2 * n:], want["out"], "out")
    for name, t in zip(("dq", "dk", "dv"), grads):
        O.check(t[-2 * n:], want[name], name)
