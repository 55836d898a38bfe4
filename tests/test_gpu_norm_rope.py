"""Norms of queries and keys with the position rotation on the GPU against 64 bits."""
import pytest
import torch

from emugen_b200 import attention
from tests import attention_oracle as O

pytestmark = pytest.mark.gpu


def _table(rows, half, seed=0):
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * torch.pow(10000.0, -torch.arange(half, dtype=torch.float64) / max(half, 1))
    return torch.cos(angle).float().cuda(), torch.sin(angle).float().cuda()


def _make(T, Hq, Hk, D, dtype, seed, rows=500):
    g = torch.Generator().manual_seed(seed)
    q, k, gq, gk = ((torch.randn(T, h, D, generator=g) * torch.exp(torch.randn(T, h, 1, generator=g))).to(dtype).cuda()
                    for h in (Hq, Hk, Hq, Hk))
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g)).to(dtype).cuda() for _ in range(2))
    pos = torch.randint(0, rows, (T,), generator=g).cuda()
    return q, k, wq, wk, pos, gq, gk


def _check(q, k, wq, wk, cos, sin, pos, gq, gk, interleaved, eps=1e-6):
    x = [None if t is None else t.detach().requires_grad_() for t in (q, k, wq, wk)]
    yq, yk = attention.qk_norm_rope(*x, cos, sin, pos, eps=eps, interleaved=interleaved)
    live = [t for t in x if t is not None]
    grads = iter(torch.autograd.grad((yq, yk), live, (gq, gk)))
    got = [next(grads) if t is not None else None for t in x]
    for name, y, t, w, g, dx, dw in (("q", yq, q, wq, gq, got[0], got[2]), ("k", yk, k, wk, gk, got[1], got[3])):
        r = O.norm_rope(t, w, cos, sin, pos, eps, interleaved, g)
        assert y.is_contiguous()
        O.check(y, r[0:2], name)
        O.check(dx, r[2:4], "d" + name)
        if w is not None:
            O.check(dw, r[4:6], "dw" + name)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,Hq,Hk,D,R,interleaved", [
    (1, 1, 1, 8, 2, True), (3, 2, 1, 16, 16, False), (7, 5, 3, 24, 16, False), (40, 8, 2, 64, 64, False), (33, 4, 4, 72, 30, True),
    (130, 32, 8, 128, 128, False), (65, 17, 1, 128, 64, False), (9, 3, 2, 200, 96, False), (50, 20, 4, 256, 256, False),
    (50, 6, 2, 256, 256, True), (77, 40, 40, 32, 32, True), (21, 2, 2, 64, 0, False), (1000, 3, 1, 96, 48, True),
])
def test_against_64_bits(dtype, T, Hq, Hk, D, R, interleaved):
    q, k, wq, wk, pos, gq, gk = _make(T, Hq, Hk, D, dtype, T + D)
    _check(q, k, wq, wk, *_table(500, R // 2), pos, gq, gk, interleaved)


def test_many_rows_and_weights_left_out():
    q, k, wq, wk, pos, gq, gk = _make(5000, 6, 2, 128, torch.bfloat16, 1)
    cos, sin = _table(500, 64)
    _check(q, k, wq, wk, cos, sin, pos, gq, gk, False)
    _check(q, k, None, wk, cos, sin, pos, gq, gk, False)
    _check(q, k, wq, None, cos, sin, pos, gq, gk, True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_padding_and_positions_past_the_table(dtype):
    """Padding gives zeros whatever its rows hold; a position past the table shows itself as NaN where elements are turned."""
    q, k, wq, wk, pos, gq, gk = _make(40, 4, 2, 64, dtype, 3)
    cos, sin = _table(500, 16)
    pos[::3] = -1
    pos[1] = -(2 ** 60)
    for t in (q, k, gq, gk):
        t[pos < 0] = float("nan")
    zero = [torch.where((pos < 0)[:, None, None], torch.zeros_like(t), t) for t in (q, k, gq, gk)]
    x = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    got = attention.qk_norm_rope(*x, cos, sin, pos)
    grads = torch.autograd.grad(got, x, (gq, gk))
    for y, dx, dw, t, w, g in zip(got, grads[:2], grads[2:], zero[:2], (wq, wk), zero[2:]):
        r = O.norm_rope(t, w, cos, sin, pos, 1e-6, False, g)
        O.check(y, r[0:2]), O.check(dx, r[2:4]), O.check(dw, r[4:6])
    pos = pos.clamp(min=0)
    pos[5], pos[6] = 500, 2 ** 62
    y, _ = attention.qk_norm_rope(*zero[:2], wq, wk, cos, sin, pos)
    past = pos >= 500
    assert y[past][..., :32].isnan().all() and not y[past][..., 32:].isnan().any() and not y[~past].isnan().any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layouts(dtype):
    """Slices of a fused projection, heads before tokens, rows off 16 bytes, expanded gradients: the same bits."""
    T, Hq, Hk, D = 37, 6, 2, 64
    q, k, wq, wk, pos, gq, gk = _make(T, Hq, Hk, D, dtype, 5)
    cos, sin = _table(500, 32)

    def run(q, k, gq, gk):
        x = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
        y = attention.qk_norm_rope(*x, cos, sin, pos)
        return (*y, *torch.autograd.grad(y, x, (gq, gk)))

    want = run(q, k, gq, gk)
    fused = torch.cat([q, k, k], 1)
    odd = torch.empty(T * Hq * D + 1, dtype=dtype, device="cuda")[1:].view(T, Hq, D).copy_(q)
    turned = [t.permute(1, 2, 0).contiguous().permute(2, 0, 1) for t in (q, k, gq, gk)]
    heads = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, gq, gk)]
    for args in ((fused[:, :Hq], fused[:, Hq:Hq + Hk], gq, gk), (odd, k, gq, gk), turned, heads):
        assert all(torch.equal(a, b) for a, b in zip(run(*args), want))
    one = gq[:1, :1, :1]
    a, b = run(q, k, one.expand(T, Hq, D), gk), run(q, k, one.expand(T, Hq, D).contiguous(), gk)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_one_side_alone_and_same_result_every_run():
    q, k, wq, wk, pos, gq, gk = _make(900, 8, 2, 128, torch.float16, 6)
    cos, sin = _table(500, 64)

    def run():
        x = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
        y = attention.qk_norm_rope(*x, cos, sin, pos)
        return torch.autograd.grad(y, x, (gq, gk))

    want = run()
    assert all(torch.equal(a, b) for a, b in zip(run(), want))
    x = q.detach().requires_grad_()
    yq, _ = attention.qk_norm_rope(x, k, wq, wk, cos, sin, pos)
    assert torch.equal(torch.autograd.grad(yq, x, gq)[0], want[0])     # k's result unused: its gradient is nothing


def test_graph_replay_and_streams():
    q, k, wq, wk, pos, gq, gk = _make(64, 8, 2, 128, torch.bfloat16, 7)
    cos, sin = _table(500, 64)

    def run(q):
        x = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
        y = attention.qk_norm_rope(*x, cos, sin, pos)
        return (*(t.detach() for t in y), *torch.autograd.grad(y, x, (gq, gk)))

    q2 = q.flip(0).contiguous()
    want, want2 = run(q), run(q2)
    static = q.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(static)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = run(static)
    for source, w in ((q, want), (q2, want2)):
        static.copy_(source)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(r, w))


def test_no_tokens():
    cos, sin = _table(10, 32)
    x = [torch.zeros(0, h, 64, device="cuda", dtype=torch.float16, requires_grad=True) for h in (4, 2)]
    w = [torch.ones(64, device="cuda", dtype=torch.float16, requires_grad=True) for _ in range(2)]
    y = attention.qk_norm_rope(*x, *w, cos, sin, torch.zeros(0, dtype=torch.int64, device="cuda"))
    g = torch.autograd.grad(y, (*x, *w), [torch.zeros_like(t) for t in y])
    assert y[0].shape == (0, 4, 64) and (g[2] == 0).all() and (g[3] == 0).all()


def test_registered_operator():
    import emugen_b200.ops  # noqa: F401

    q, k, wq, wk, pos, _, _ = _make(9, 4, 2, 64, torch.bfloat16, 8)
    cos, sin = _table(500, 32)
    want = attention.qk_norm_rope(q, k, wq, wk, cos, sin, pos)
    got = torch.ops.emugen.qk_norm_rope(q, k, wq, wk, cos, sin, pos)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,D", [(37, 64), (5, 128), (700, 96)])
def test_without_eps(dtype, T, D):
    """eps 0: rows that are padding, and lanes without a row, add nothing to the weights' gradients."""
    q, k, wq, wk, pos, gq, gk = _make(T, 5, 3, D, dtype, 21)
    cos, sin = _table(500, 16)
    pos[1::4] = -1
    live = pos >= 0
    x = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    got = attention.qk_norm_rope(*x, cos, sin, pos, eps=0.0)
    grads = torch.autograd.grad(got, x, (gq, gk))
    for y, dx, dw, t, w, g in zip(got, grads[:2], grads[2:], (q, k), (wq, wk), (gq, gk)):
        r = O.norm_rope(t[live], w, cos, sin, pos[live], 0.0, False, g[live])
        assert (y[~live] == 0).all() and (dx[~live] == 0).all()
        O.check(y[live], r[0:2]), O.check(dx[live], r[2:4]), O.check(dw, r[4:6])


def test_offsets_past_32_bits():
    """Tensors of more than 2^31 elements: the last tokens as on their own."""
    T, H, D = 70000, 128, 256
    g = torch.Generator(device="cuda").manual_seed(3)
    q, gq = (torch.randn(T, H, D, device="cuda", dtype=torch.bfloat16, generator=g) for _ in range(2))
    k, gk = (torch.randn(T, 1, D, device="cuda", dtype=torch.bfloat16, generator=g) for _ in range(2))
    assert q.numel() > 2 ** 31
    w = torch.ones(D, device="cuda", dtype=torch.bfloat16)
    cos, sin = _table(500, 128)
    pos = torch.arange(T, device="cuda") % 500
    x = [t.requires_grad_() for t in (q, k)]
    y = attention.qk_norm_rope(*x, w, w, cos, sin, pos)
    grads = torch.autograd.grad(y, x, (gq, gk))
    for a, b, t, u in zip(y, grads, x, (gq, gk)):
        r = O.norm_rope(t[-50:].detach(), w, cos, sin, pos[-50:], 1e-6, False, u[-50:])
        O.check(a[-50:], r[0:2]), O.check(b[-50:], r[2:4])
