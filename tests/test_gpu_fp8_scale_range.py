"""The 8-bit product with scales whose product leaves f32's range although the result does not: every kernel and
scale layout against 64 bits.  Codes are small integers (times a power of two) and scales powers of two, constant along K
for an output, so that every partial sum is exact and the f32 result has no error at all."""
import math

import pytest
import torch

from emugen_b200 import fp8
from tests import fp8_oracle as O

pytestmark = pytest.mark.gpu
E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2

# few rows, one part and split over K; 32 and 64 columns; more rows than one column tile; the CTA pairs
SHAPES = [(5, 20000, 4096), (5, 300, 4096), (30, 700, 4096), (60, 300, 1100), (100, 500, 4096), (600, 2000, 4096), (1024, 2048, 4096)]


def _codes(rows, K, dtype, unit, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(-2, 3, (rows, K), generator=g).float() * unit).to(dtype).cuda()


def _pow2(exponents):
    return torch.tensor([math.ldexp(1.0, e) for e in exponents], dtype=torch.float32)


def _row_scales(exponents, rows, kb):
    """[rows, kb] scales, the exponents in turn."""
    return _pow2(exponents)[torch.arange(rows) % len(exponents)][:, None].expand(rows, kb).contiguous().cuda()


def _check(a, b, sa, sb, rows):
    N, K = b.shape
    out = fp8.gemm_fp8(a, b, sa, sb, out_dtype=torch.float32)
    s = sb if rows else sb.repeat_interleave(128, 0)[:N]
    ref = (a.double() * sa[:, :1].double()) @ (b.double() * s[:, :1].double()).t()
    assert torch.equal(out, ref.float())
    return out


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("rows", [False, True])
@pytest.mark.parametrize("dtype,unit,ea,eb", [
    (E4, 128.0, [-75], [-76]),                                  # the scales' product is below f32's range
    (E4, 128.0, [-100], [-26]),                                 # at its smallest normal number
    (E5, 2.0 ** -16, [-126], [119]),                            # smallest codes: either scale alone would lose them
    (E5, 2.0 ** -16, [119], [-126]),
    (E5, 8192.0, [-126], [105]),                                # largest codes: one scale alone would overflow
    (E5, 8192.0, [105], [-126]),
    (E4, 128.0, [-126, 0, -75, 75], [-76, 0, 20]),              # rows of a warp far apart
    (E4, 1.0, [0, 110, -126], [-100, 0]),
])
def test_scales_far_from_one(M, N, K, rows, dtype, unit, ea, eb):
    kb = -(-K // 128)
    a, b = _codes(M, K, dtype, unit, M + K), _codes(N, K, dtype, unit, N)
    _check(a, b, _row_scales(ea, M, kb), _row_scales(eb, N if rows else -(-N // 128), kb), rows)


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("rows", [False, True])
@pytest.mark.parametrize("ea,eb", [(70, 60), (-126, 127), (127, 127)])
def test_blocks_that_sum_to_nothing(M, N, K, rows, ea, eb):
    """Finite scales and a block sum of zero give zero, whatever the scales' product."""
    kb = -(-K // 128)
    a = torch.ones(M, K)
    a[:, 1::2] = -1.0
    b = (1.0 + torch.arange(N) % 2)[:, None].expand(N, K)
    out = fp8.gemm_fp8(a.to(E4).cuda(), b.contiguous().to(E4).cuda(), _row_scales([ea], M, kb),
                       _row_scales([eb], N if rows else -(-N // 128), kb), out_dtype=torch.float32)
    assert (out == 0).all()


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("rows", [False, True])
def test_nan_and_infinite_scales_beside_far_ones(M, N, K, rows):
    """A NaN scale makes its row (or column) NaN and no other; an infinite one its row infinite or NaN."""
    kb = -(-K // 128)
    a, b = _codes(M, K, E4, 128.0, 5), _codes(N, K, E4, 128.0, 6)
    sa, sb = _row_scales([-75, 0], M, kb), _row_scales([-76, 1], N if rows else -(-N // 128), kb)
    want = _check(a, b, sa, sb, rows)
    sa[1, kb - 1], sa[3, 0] = float("nan"), float("inf")
    sb[-1, 0] = float("nan")
    out = fp8.gemm_fp8(a, b, sa, sb, out_dtype=torch.float32)
    bad = torch.zeros(M, N, dtype=torch.bool, device="cuda")
    bad[1] = True
    bad[:, N - 1 if rows else (N - 1) // 128 * 128:] = True
    assert out[bad].isnan().all()
    bad[3] = True
    assert not out[3].isfinite().any()
    assert torch.equal(out[~bad], want[~bad])


def test_linear_of_small_operands():
    """Operands of 1e-19: their scales' product is below f32's smallest number, the sums of 4096 products are not."""
    g = torch.Generator().manual_seed(3)
    for M, N in ((4, 256), (700, 2048)):
        x, w = torch.rand(M, 4096, generator=g) * 1e-19, torch.rand(N, 4096, generator=g) * 1e-19
        (xq, xs), (wq, ws) = fp8.quant_fp8(x.cuda()), fp8.quant_fp8(w.cuda(), block="tile")
        ref, mag = O.gemm(xq.cpu(), wq.cpu(), xs.cpu(), ws.cpu())
        y = fp8.linear_fp8(x.cuda(), w.cuda()).cpu().double().numpy()
        # O(1e-35) sums: each block's addition is also rounded to a multiple of 2^-149 where it is that small
        assert (abs(y - ref) <= O.gemm_tolerance(ref, mag, 4096, torch.float32) + 33 * 2.0 ** -150).all()
        assert (y > 0).all()


@pytest.mark.parametrize("M,N,K", [(2048, 2304, 2000), (1500, 2100, 4096), (4096, 4000, 1300)])
@pytest.mark.parametrize("rows", [False, True])
def test_cta_pairs_over_many_blocks_exact(M, N, K, rows):
    """More blocks of K than the rings of the CTA pairs' kernel hold, several tiles a pair, random scales: exact."""
    g = torch.Generator().manual_seed(M)
    kb = -(-K // 128)
    a, b = _codes(M, K, E4, 1.0, M), _codes(N, K, E5, 1.0, N)
    sa = torch.ldexp(torch.ones(M, kb), torch.randint(0, 3, (M, kb), generator=g)).cuda()
    n = N if rows else -(-N // 128)
    sb = torch.ldexp(torch.ones(n, kb), torch.randint(-2, 1, (n, kb), generator=g)).cuda()
    full = lambda q, s: q.double() * s.double().repeat_interleave(128, 1)[:, :K]
    ref = full(a, sa) @ full(b, sb if rows else sb.repeat_interleave(128, 0)[:N]).t()
    for _ in range(3):
        assert torch.equal(fp8.gemm_fp8(a, b, sa, sb, out_dtype=torch.float32).double(), ref)


@pytest.mark.parametrize("M,N,K", SHAPES + [(700, 2300, 4000)])
@pytest.mark.parametrize("rows", [False, True])
@pytest.mark.parametrize("kind", ["zeros", "zeros and largest", "small"])
def test_scales_that_change_along_k(M, N, K, rows, kind):
    """Blocks of zeros (the quantiser's smallest scale, or the largest one) among others in every order, the first block
    of a row among them, and rows whose blocks are all below the range: exact."""
    g = torch.Generator().manual_seed(M + N)
    kb, nb = -(-K // 128), N if rows else -(-N // 128)
    a, b = _codes(M, K, E4, 1.0 if kind != "small" else 128.0, 1), _codes(N, K, E4, 1.0 if kind != "small" else 128.0, 2)
    ea, eb = torch.randint(-1, 2, (M, kb), generator=g), torch.randint(-1, 2, (nb, kb), generator=g)
    if kind == "small":
        ea = ea * 0 - 126 + 2 * torch.randint(0, 2, (M, kb), generator=g)
        eb = eb * 0 - 18
    else:
        dead = torch.rand(M, kb, generator=g) < torch.rand(M, 1, generator=g)       # some rows all dead, some none
        dead[::7, 0] = True
        ea[dead] = -126
        if kind != "zeros":
            ea[dead & (torch.rand(M, kb, generator=g) < 0.1)] = 127
        a = (a.float() * (~dead).repeat_interleave(128, 1)[:, :K].cuda()).to(E4)
        dead = torch.rand(nb, kb, generator=g) < 0.05
        eb[dead] = -126
        d = dead if rows else dead.repeat_interleave(128, 0)[:N]
        b = (b.float() * (~d).repeat_interleave(128, 1)[:, :K].cuda()).to(E4)
    sa, sb = (torch.ldexp(torch.ones(e.shape), e).cuda() for e in (ea, eb))
    out = fp8.gemm_fp8(a, b, sa, sb, out_dtype=torch.float32)
    full = lambda q, s: q.double() * s.double().repeat_interleave(128, 1)[:, :K]
    ref = full(a, sa) @ full(b, sb if rows else sb.repeat_interleave(128, 0)[:N]).t()
    assert torch.equal(out, ref.float())
