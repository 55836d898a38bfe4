"""The 8-bit quantiser, product and linear layer on the GPU against the 64-bit oracle (tests/fp8_oracle.py):
codes and scales bit for bit, products exactly where every sum is a small integer and within the derived
bound elsewhere."""
import numpy as np
import pytest
import torch

from emugen_b200 import _lib, fp8
from tests import fp8_oracle as O

pytestmark = pytest.mark.gpu
E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2


def _x(M, K, dtype, seed=0, special=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g) * torch.exp(2 * torch.randn(M, 1, generator=g))
    x[:, torch.rand(K, generator=g) < 0.02] *= 60
    if special:
        x[torch.rand(M, K, generator=g) < 0.01] = 0
        x[0] = 0                                   # a whole row, so whole blocks, of zeros
        if M > 3 and K > 7:
            x[1, 3], x[2, 5], x[3, 7], x[1, 0] = float("nan"), float("inf"), float("-inf"), -0.0
    return x.to(dtype)


def _check(x, block, dtype, q, s, qt=None, st=None):
    codes, scales = O.quant(x, block, dtype)
    assert (O.codes_of(q) == codes).all()
    assert (s.cpu().numpy() == scales).all()
    if qt is not None:
        codes, scales = O.quant(x.t(), block, dtype)
        assert (O.codes_of(qt) == codes).all()
        assert (st.cpu().numpy() == scales).all()


@pytest.mark.parametrize("M,K", [(1, 1), (1, 128), (3, 127), (5, 129), (130, 16), (127, 300), (257, 513), (64, 1111)])
@pytest.mark.parametrize("block", ["row", "tile"])
@pytest.mark.parametrize("dtype", [E4, E5])
@pytest.mark.parametrize("xt", [torch.bfloat16, torch.float16, torch.float32])
def test_quant_matches_the_oracle(M, K, block, dtype, xt):
    x = _x(M, K, xt, seed=M * 1000 + K)
    xc = x.cuda()
    _check(x, block, dtype, *fp8.quant_fp8(xc, block=block, dtype=dtype))
    _check(x, block, dtype, *fp8.quant_fp8(xc, block=block, dtype=dtype, transposed=True))


@pytest.mark.parametrize("dtype", [E4, E5])
def test_quant_borders(dtype):
    """Blocks whose quotients are exact ties, one unit beside ties (f32 inputs), in and below the normal range."""
    v = O.values(dtype)[:128]
    v = v[np.isfinite(v)]
    mid = ((v[1:] + v[:-1]) / 2).astype(np.float32)
    rows = []
    for scale in (1.0, 2.0 ** -40, 1.1, 0.7731, 3.0e-30, 2.0 ** 60 / 3):
        s = np.float32(scale)
        top = np.float32(O.MAX[dtype]) * s                      # amax: its scale is s again, or beside it
        got = np.float32(top / np.float32(O.MAX[dtype]))
        base = (mid.astype(np.float64) * got).astype(np.float32)
        for y in (base, np.nextafter(base, np.float32(np.inf)), np.nextafter(base, np.float32(0))):
            for part in np.array_split(y, -(-len(y) // 127)):
                row = np.zeros(128, np.float32)
                row[:len(part)] = part * np.where(np.arange(len(part)) % 2, -1, 1)
                row[127] = top
                rows.append(row)
    x = torch.from_numpy(np.stack(rows))
    _check(x, "row", dtype, *fp8.quant_fp8(x.cuda(), dtype=dtype))
    xb = x.to(torch.bfloat16)
    _check(xb, "row", dtype, *fp8.quant_fp8(xb.cuda(), dtype=dtype, transposed=True))


def test_quant_extreme_scales():
    x = torch.tensor([3e38, 1e-38, 1e-45, 2.0 ** -126, 0.0]).repeat_interleave(128).reshape(5, 128).clone()
    x[:, 1::2] *= -0.37
    _check(x, "row", E4, *fp8.quant_fp8(x.cuda()))
    _check(x, "row", E5, *fp8.quant_fp8(x.cuda(), dtype=E5))
    _check(x, "tile", E4, *fp8.quant_fp8(x.cuda(), block="tile"))


def test_quant_strides():
    """Row-strided, column-strided, misaligned and three-dimensional inputs."""
    base = _x(70, 700, torch.bfloat16, seed=5).cuda()
    for x in (base[:, :256], base[::2, 8:300], base[3:, 1:130], base.t(), base[:, ::2], base[:1].expand(5, 700)):
        for t in (False, True):
            _check(x.cpu(), "row", E4, *fp8.quant_fp8(x, transposed=t))
    x = base[:, :640].reshape(7, 10, 640)
    q, s = fp8.quant_fp8(x)
    assert q.shape == (70, 640) and s.shape == (70, 5)
    _check(x.reshape(70, 640).cpu(), "row", E4, q, s)


def test_quant_empty():
    for shape in ((0, 64), (3, 0), (0, 0)):
        q, s, qt, st = fp8.quant_fp8(torch.zeros(shape, dtype=torch.float16, device="cuda"), transposed=True)
        assert q.shape == shape and qt.shape == shape[::-1] and s.shape[0] == shape[0]


def test_quant_leaves_bytes_between_rows_alone():
    """The C entry: codes past K and rows past M keep what was there."""
    x = _x(5, 70, torch.bfloat16).cuda()
    q = torch.full((7, 96), 0xAB, dtype=torch.uint8, device="cuda")
    s = torch.full((1, 12), 7.0, device="cuda")
    qt = torch.full((72, 32), 0xCD, dtype=torch.uint8, device="cuda")
    st = torch.full((1, 80), 9.0, device="cuda")
    L = _lib.load()
    rc = L.emu_quant_fp8(x.data_ptr(), 1, 5, 70, 70, 0, 0, q.data_ptr(), 96, s.data_ptr(), 12, qt.data_ptr(), 32,
                         st.data_ptr(), 80, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    _check(x.cpu(), "row", E4, q[:5, :70].view(E4), s[:, :5].t(), qt[:70, :5].view(E4), st[:, :70].t())
    assert (q[:, 70:] == 0xAB).all() and (q[5:] == 0xAB).all() and (s[:, 5:] == 7).all()
    assert (qt[:, 5:] == 0xCD).all() and (qt[70:] == 0xCD).all() and (st[:, 70:] == 9).all()


def _operands(M, N, K, at, bt, rows, seed, exact):
    g = torch.Generator().manual_seed(seed)
    kb, nb = -(-K // 128), -(-N // 128)
    sb_rows = N if rows else nb
    if exact:   # small integers and powers of two: every partial sum is an integer below 2^24 units
        a = torch.randint(-2, 3, (M, K), generator=g).float()
        b = torch.randint(-2, 3, (N, K), generator=g).float()
        sa = torch.ldexp(torch.ones(M, kb), torch.randint(0, 3, (M, kb), generator=g))
        sb = torch.ldexp(torch.ones(sb_rows, kb), torch.randint(-2, 1, (sb_rows, kb), generator=g))
    else:
        a = torch.randn(M, K, generator=g) * O.MAX[at] / 4
        b = torch.randn(N, K, generator=g) * O.MAX[bt] / 4
        a, b = a.clamp(-O.MAX[at], O.MAX[at]), b.clamp(-O.MAX[bt], O.MAX[bt])
        sa = torch.rand(M, kb, generator=g) / O.MAX[at] * 4
        sb = torch.rand(sb_rows, kb, generator=g) / O.MAX[bt] * 4
    return a.to(at), b.to(bt), sa, sb


# one row to many, short and ragged K, one block to many, N below, at and past the tiles
SHAPES = [(1, 1, 1), (1, 128, 128), (1, 300, 4096), (2, 17, 33), (7, 1000, 130), (16, 128, 1024), (17, 129, 257), (33, 256, 2000),
          (64, 64, 64), (65, 130, 384), (100, 1500, 1111), (128, 128, 128), (129, 257, 129), (200, 96, 5000), (255, 511, 640),
          (300, 1000, 520), (513, 640, 256), (1024, 1024, 1024), (1300, 2304, 392),
          # large enough for the CTA pairs: ragged in every direction, one block of K, several tiles a pair
          (1111, 1501, 2000), (2049, 2300, 130), (4100, 4000, 260), (257, 20000, 512), (3000, 2900, 100)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("rows", [False, True])
def test_gemm_exact_integers(M, N, K, rows):
    """Small integers: every sum is exact in f32, so the f32 result has no error at all."""
    a, b, sa, sb = _operands(M, N, K, E4, E5 if rows else E4, rows, seed=M + N + K, exact=True)
    out = fp8.gemm_fp8(a.cuda(), b.cuda(), sa.cuda(), sb.cuda(), out_dtype=torch.float32)
    ref, mag = O.gemm(a, b, sa, sb)
    assert mag.max() * 4 < 2 ** 24
    assert (out.cpu().double().numpy() == ref).all()


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("rows", [False, True])
@pytest.mark.parametrize("at,bt,out_dtype", [(E4, E4, torch.bfloat16), (E5, E4, torch.float32), (E4, E5, torch.float16)])
def test_gemm_within_the_bound(M, N, K, rows, at, bt, out_dtype):
    a, b, sa, sb = _operands(M, N, K, at, bt, rows, seed=M * 3 + N + K, exact=False)
    out = fp8.gemm_fp8(a.cuda(), b.cuda(), sa.cuda(), sb.cuda(), out_dtype=out_dtype)
    ref, mag = O.gemm(a, b, sa, sb)
    assert out.shape == (M, N) and out.dtype == out_dtype
    err = np.abs(out.cpu().double().numpy() - ref)
    tol = O.gemm_tolerance(ref, mag, K, out_dtype)
    assert (err <= tol).all(), (err / tol).max()


def test_gemm_same_result_every_run():
    a, b, sa, sb = [t.cuda() for t in _operands(20, 700, 5000, E4, E4, False, 3, False)]
    first = fp8.gemm_fp8(a, b, sa, sb, out_dtype=torch.float32)
    for _ in range(5):
        assert torch.equal(first, fp8.gemm_fp8(a, b, sa, sb, out_dtype=torch.float32))


@pytest.mark.parametrize("M,N,K", [(5, 200, 300), (150, 300, 600), (700, 800, 640), (2000, 2100, 300)])
@pytest.mark.parametrize("rows", [False, True])
def test_gemm_nan_stays_in_its_row_and_column(M, N, K, rows):
    a, b, sa, sb = _operands(M, N, K, E4, E4, rows, 11, True)
    ref, _ = O.gemm(a, b, sa, sb)
    a.view(torch.uint8)[M // 2, K - 1] = 0x7F
    b.view(torch.uint8)[N - 1, 0] = 0xFF
    sa[M - 1, 0] = float("inf")
    out = fp8.gemm_fp8(a.cuda(), b.cuda(), sa.cuda(), sb.cuda(), out_dtype=torch.float32).cpu().double().numpy()
    bad = np.zeros((M, N), bool)
    bad[M // 2] = bad[:, N - 1] = True
    assert np.isnan(out[bad]).all()
    bad[M - 1] = True                               # an infinite scale: infinities and NaN, in its row alone
    assert not np.isfinite(out[M - 1]).any()
    assert (out[~bad] == ref[~bad]).all()


def test_gemm_bytes_past_k_and_rows_past_the_end_are_not_used():
    """Operands inside larger buffers full of NaN codes and infinite scales."""
    M, N, K = 70, 90, 200
    a, b, sa, sb = _operands(M, N, K, E4, E4, True, 4, True)
    ref, _ = O.gemm(a, b, sa, sb)

    def inside(t):
        big = torch.full((t.shape[0] + 5, 256), 0x7F, dtype=torch.uint8, device="cuda").view(t.dtype)
        big.view(torch.uint8)[:t.shape[0], :K] = t.view(torch.uint8).cuda()
        return big[:t.shape[0], :K]

    def scales(s):
        big = torch.full((s.shape[1], 160), float("inf"), device="cuda")
        big[:, :s.shape[0]] = s.t().cuda()
        return big.t()[:s.shape[0]]

    out = fp8.gemm_fp8(inside(a), inside(b), scales(sa), scales(sb), out_dtype=torch.float32)
    assert (out.cpu().double().numpy() == ref).all()


def test_gemm_other_layouts_are_copied():
    """Column-major operands, pitches that are no multiple of 16, contiguous scales, CPU tensors."""
    M, N, K = 37, 150, 259
    a, b, sa, sb = _operands(M, N, K, E4, E4, False, 8, True)
    ref, _ = O.gemm(a, b, sa, sb)
    ac, bc, sac, sbc = a.cuda(), b.cuda(), sa.cuda(), sb.cuda()
    at = ac.view(torch.uint8).t().contiguous().t().view(E4)
    odd = torch.zeros(M, K + 1, dtype=torch.uint8, device="cuda")
    odd[:, 1:] = ac.view(torch.uint8)
    for x in (ac, at, odd[:, 1:].view(E4)):
        for s in (sac, sac.t().contiguous().t(), torch.cat([sac, sac])[::2] * 0 + sac):
            out = fp8.gemm_fp8(x, bc, s, sbc.t().contiguous().t(), out_dtype=torch.float32)
            assert (out.cpu().double().numpy() == ref).all()
    out = fp8.gemm_fp8(a, b, sa, sb, out_dtype=torch.float32)
    assert not out.is_cuda and (out.double().numpy() == ref).all()


def test_gemm_output_rows_apart():
    """The C entry with ldo > N: what lies between the rows and behind the last stays."""
    for M, N, K in ((3, 130, 256), (200, 300, 256), (2000, 2101, 256), (2000, 2104, 256)):
        a, b, sa, sb = [t.cuda() for t in _operands(M, N, K, E4, E4, False, 2, True)]
        sa4 = torch.zeros(2, (M + 3) // 4 * 4, device="cuda")
        sa4[:, :M] = sa.t()
        out = torch.full((M + 2, N + 13), 5.0, dtype=torch.bfloat16, device="cuda")
        rc = _lib.load().emu_gemm_fp8(a.data_ptr(), K, 0, b.data_ptr(), K, 0, sa4.data_ptr(), sa4.shape[1], sb.data_ptr(), 2, 1,
                                      M, N, K, 1, out.data_ptr(), N + 13, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        want = fp8.gemm_fp8(a, b, sa, sb)
        assert torch.equal(out[:M, :N], want)
        assert (out[:, N:] == 5).all() and (out[M:] == 5).all()


def test_gemm_empty():
    z = torch.zeros(0, 64, dtype=torch.uint8, device="cuda").view(E4)
    b = torch.zeros(5, 64, dtype=torch.uint8, device="cuda").view(E4)
    s0, s5 = torch.zeros(0, 1, device="cuda"), torch.ones(5, 1, device="cuda")
    assert fp8.gemm_fp8(z, b, s0, s5).shape == (0, 5)
    assert fp8.gemm_fp8(b, z, s5, s0).shape == (5, 0)
    e = torch.zeros(5, 0, dtype=torch.uint8, device="cuda").view(E4)
    out = fp8.gemm_fp8(e, e, s5[:, :0], s5[:, :0])
    assert out.shape == (5, 5) and (out == 0).all()


def test_streams_and_graph():
    """On a side stream, two streams at once, and captured and replayed on new inputs."""
    sets = [[t.cuda() for t in _operands(m, n, 3000, E4, E4, False, m, True)] for m, n in ((3, 900), (40, 900), (300, 900), (2000, 2500))]
    want = [fp8.gemm_fp8(*s, out_dtype=torch.float32) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    outs = []
    for st, s in zip(streams, sets):
        with torch.cuda.stream(st):
            outs.append([fp8.gemm_fp8(*s, out_dtype=torch.float32) for _ in range(5)])
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(x, w) for x in o)
    x = torch.randn(64, 512, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(256, 512, device="cuda", dtype=torch.bfloat16)
    wq, ws = fp8.quant_fp8(w, block="tile")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, s, qt, st = fp8.quant_fp8(x, transposed=True)
        y = fp8.gemm_fp8(q, wq, s, ws)
    for seed in range(3):
        x.copy_(torch.randn(64, 512, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        q2, s2, qt2, st2 = fp8.quant_fp8(x, transposed=True)
        for got, ref in ((q, q2), (qt, qt2)):
            assert (O.codes_of(got) == O.codes_of(ref)).all()
        assert torch.equal(s, s2) and torch.equal(st, st2)
        assert torch.equal(y, fp8.gemm_fp8(q2, wq, s2, ws))


def _dequant(codes, scales, block, M, K):
    v = torch.from_numpy(O.values(E4)[codes])
    return v * torch.from_numpy(O.spread(scales, M, K, block == "row"))


@pytest.mark.parametrize("shape,N,dtype", [((1, 64), 32, torch.bfloat16), ((130, 200), 257, torch.float16), ((2, 5, 136), 70, torch.bfloat16),
                                            ((300, 520), 1000, torch.float32)])
def test_linear_forward_and_gradients(shape, N, dtype):
    """y, dx and dw against the formula in 64 bits on the oracle's codes."""
    K = shape[-1]
    g = torch.Generator().manual_seed(K)
    x, w = torch.randn(shape, generator=g).to(dtype), (torch.randn(N, K, generator=g) * K ** -0.5).to(dtype)
    dy = torch.randn(*shape[:-1], N, generator=g).to(dtype)
    xc, wc = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    y = fp8.linear_fp8(xc, wc)
    assert y.shape == dy.shape and y.dtype == dtype
    y.backward(dy.cuda())
    M = x[..., 0].numel()
    x2, g2 = x.reshape(M, K), dy.reshape(M, N)

    def deq(t, block):
        return _dequant(*O.quant(t, block, E4), block, *t.shape).numpy()

    cases = [(y.reshape(M, N), deq(x2, "row"), deq(w, "tile")), (xc.grad.reshape(M, K), deq(g2, "row"), deq(w, "tile").T),
             (wc.grad, deq(g2.t(), "row"), deq(x2.t(), "row"))]
    for got, p, q in cases:
        ref, mag = p @ q.T, np.abs(p) @ np.abs(q).T
        err = np.abs(got.detach().cpu().double().numpy() - ref)
        assert (err <= O.gemm_tolerance(ref, mag, p.shape[1], dtype)).all()


def test_linear_gradient_against_differences():
    """Where quantisation changes nothing (small integers under a scale that is a power of two), the layer
    is linear, and differences along any direction give the gradients exactly."""
    M, N, K = 40, 130, 256
    g = torch.Generator().manual_seed(1)

    def ints(*s):
        t = torch.randint(-8, 9, s, generator=g).float()
        t[:, ::128] = 7.0                   # 448 = 7 * 64: every row block's, column block's and tile's scale is 2^-6 ..
        return t
    x, w, dy = ints(M, K).clamp(-7, 7), ints(N, K).clamp(-7, 7), ints(M, N).clamp(-7, 7)
    x[0], dy[0] = 7.0, 7.0                  # .. in the transposed blocks too
    xc, wc = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    y = fp8.linear_fp8(xc, wc)
    assert torch.equal(y.cpu().double(), x.double() @ w.double().t())
    dx, dw = torch.autograd.grad(y, (xc, wc), dy.cuda())
    loss = lambda a, b: (fp8.linear_fp8(a, b).double() * dy.cuda().double()).sum().item()
    base = loss(x.cuda(), w.cuda())
    for i in range(6):
        r, c = (5 * i + 1) % M, (37 * i + 3) % K
        x2 = x.clone()
        x2[r, c] += -1 if x[r, c] > 0 else 1
        assert loss(x2.cuda(), w.cuda()) - base == dx[r, c].item() * (x2 - x)[r, c].item()
        r = (29 * i + 2) % N
        w2 = w.clone()
        w2[r, c] += -1 if w[r, c] > 0 else 1
        assert loss(x.cuda(), w2.cuda()) - base == dw[r, c].item() * (w2 - w)[r, c].item()


def test_linear_partial_gradients_and_expanded_gradient():
    x = torch.randn(33, 128, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(48, 128, device="cuda", dtype=torch.bfloat16)
    full = fp8.linear_fp8(x.clone().requires_grad_(), w)
    for nx, nw in ((True, False), (False, True)):
        a, b = x.clone().requires_grad_(nx), w.clone().requires_grad_(nw)
        y = fp8.linear_fp8(a, b)
        assert torch.equal(y, full)
        y.sum().backward()                  # the gradient comes as an expanded scalar
        assert (a.grad is not None) == nx and (b.grad is not None) == nw
    assert not fp8.linear_fp8(x, w).requires_grad
    with torch.no_grad():
        assert torch.equal(fp8.linear_fp8(x, w), full)
    one = fp8.linear_fp8(x[3], w)                       # a vector
    assert one.shape == (48,) and torch.equal(one, fp8.linear_fp8(x[3:4], w)[0])
    p, q = x.clone().requires_grad_(), w.clone().requires_grad_()
    with torch.no_grad():                               # nothing is kept where nothing is to be differentiated
        assert fp8.linear_fp8(p, q).grad_fn is None
    for shape, n in (((2, 3, 0), 5), ((2, 0, 8), 5), ((2, 3, 8), 0)):   # nothing to add up, no rows, no columns
        a = torch.ones(shape, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        b = torch.ones(n, shape[-1], device="cuda", dtype=torch.bfloat16, requires_grad=True)
        out = fp8.linear_fp8(a, b)
        assert out.shape == (*shape[:-1], n) and (out == 0).all()
        da, db = torch.autograd.grad(out, (a, b), torch.ones_like(out))
        assert da.shape == a.shape and db.shape == b.shape and (da == 0).all() and (db == 0).all()
    y = fp8.linear_fp8(p, q)                            # a second backward pass through the same graph
    g1 = torch.autograd.grad(y, (p, q), torch.ones_like(y), retain_graph=True)
    g2 = torch.autograd.grad(y, (p, q), torch.ones_like(y))
    assert all(torch.equal(s, t) for s, t in zip(g1, g2))
    e = torch.zeros(0, 128, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    v = w.clone().requires_grad_()
    fp8.linear_fp8(e, v).sum().backward()
    assert (v.grad == 0).all() and e.grad.shape == e.shape


def test_linear_training_step_captured():
    """Forward and backward in a graph, replayed on new inputs, equal the eager step."""
    x = torch.randn(96, 256, device="cuda", dtype=torch.bfloat16).requires_grad_()
    w = torch.randn(128, 256, device="cuda", dtype=torch.bfloat16).requires_grad_()
    dy = torch.randn(96, 128, device="cuda", dtype=torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(fp8.linear_fp8(x, w), (x, w), dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fp8.linear_fp8(x, w)
        dx, dw = torch.autograd.grad(y, (x, w), dy)
    with torch.no_grad():
        x.copy_(torch.randn_like(x))
    graph.replay()
    a, b = x.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
    y2 = fp8.linear_fp8(a, b)
    dx2, dw2 = torch.autograd.grad(y2, (a, b), dy)
    assert torch.equal(y, y2) and torch.equal(dx, dx2) and torch.equal(dw, dw2)


@pytest.mark.parametrize("M,N", [(8, 256), (300, 256), (2048, 2048)])   # skinny (split over K), skinny, CTA pairs
def test_wait_limit_is_reported(M, N):
    """A withheld ready signal: the bounded wait runs out, the kernel returns, the status tells, and the
    next product is right."""
    a, b, sa, sb = _operands(M, N, 512, E4, E4, False, 6, True)
    dev = [t.cuda() for t in (a, b, sa, sb)]
    _lib.device_status()
    old = _lib.set_wait_limit(1_000_000)
    try:
        _lib.load().emu_test_hold_first_ready(1)
        try:
            fp8.gemm_fp8(*dev, out_dtype=torch.float32)
        finally:
            _lib.load().emu_test_hold_first_ready(0)
        with pytest.raises(_lib.EmuError, match="8-bit product") as e:
            _lib.device_status()
        assert e.value.status == _lib.EMU_ERR_TIMEOUT
    finally:
        _lib.set_wait_limit(old)
    _lib.device_status()
    out = fp8.gemm_fp8(*dev, out_dtype=torch.float32)
    assert (out.cpu().double().numpy() == O.gemm(a, b, sa, sb)[0]).all()


@pytest.mark.parametrize("M,N,K", [(1, 65536, 4096), (30, 40000, 2000), (100, 20000, 4096), (140, 20000, 4000)])
@pytest.mark.parametrize("rows", [False, True])
def test_gemm_many_blocks_and_ctas_exact(M, N, K, rows):
    """More tiles than the SMs hold at once and many blocks of K each, the same call repeated: integers, so that a
    stage read before it has landed would show.  The reference product is torch's in f64, on the GPU."""
    a, b, sa, sb = [t.cuda() for t in _operands(M, N, K, E4, E4, rows, 17, True)]
    kb = sa.shape[1]
    full = lambda q, s: q.double() * s.double().repeat_interleave(128, 1)[:, :K]
    ref = full(a, sa) @ full(b, sb if rows else sb.repeat_interleave(128, 0)[:N]).t()
    for _ in range(4):
        out = fp8.gemm_fp8(a, b, sa, sb, out_dtype=torch.float32)
        assert torch.equal(out.double(), ref)


def test_registered_operators():
    import emugen_b200.ops  # noqa: F401

    x = _x(33, 200, torch.bfloat16, special=False).cuda()
    w = _x(70, 200, torch.bfloat16, seed=1, special=False).cuda()

    def f(x, w):
        q, s = torch.ops.emugen.quant_fp8(x)
        v, t = torch.ops.emugen.quant_fp8(w, "tile")
        return torch.ops.emugen.gemm_fp8(q, v, s, t) * 2

    want = fp8.linear_fp8(x, w) * 2
    assert torch.equal(f(x, w), want)
    assert torch.equal(torch.compile(f, backend="aot_eager", fullgraph=True)(x, w), want)


def test_beside_the_emulated_product_on_other_streams():
    """The kernels that own tensor memory, at once: the emulated product, the CTA pairs and the skinny kernel."""
    from emugen_b200 import nvfp4_global_scales, quant_nvfp4

    g = torch.Generator().manual_seed(2)
    p, r = torch.randn(1024, 1024, generator=g).half().cuda(), torch.randn(1024, 1024, generator=g).half().cuda()
    gp, gr, alpha = nvfp4_global_scales(p, r)
    (qp, sp), (qr, sr) = quant_nvfp4(p, gp), quant_nvfp4(r, gr)
    emulated = lambda: _lib.gemm(qp, qr, sp, sr, fmt=0, group_size=16, w_reduce=4, stage3_rounding=0, stage4_rounding=0,
                                 alpha=alpha, out_mode=2, path="tc")
    big = [t.cuda() for t in _operands(2048, 2048, 2048, E4, E4, False, 3, True)]
    few = [t.cuda() for t in _operands(40, 4000, 4096, E4, E4, True, 4, True)]
    calls = [emulated, lambda: fp8.gemm_fp8(*big, out_dtype=torch.float32), lambda: fp8.gemm_fp8(*few, out_dtype=torch.float32)]
    want = [f() for f in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    outs = [[] for _ in calls]
    for _ in range(8):
        for st, f, o in zip(streams, calls, outs):
            with torch.cuda.stream(st):
                o.append(f())
    torch.cuda.synchronize()
    _lib.device_status()
    for o, w in zip(outs, want):
        assert all(torch.equal(x, w) for x in o)
