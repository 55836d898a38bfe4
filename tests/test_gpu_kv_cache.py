"""The quantised key/value cache on the GPU: written bytes against the 64-bit oracle and the framework's own
quantisers, read-back against the formula, and what must stay untouched."""
import numpy as np
import pytest
import torch

from emugen_b200 import _lib, fp8, kvcache
from tests import fp8_oracle as O

pytestmark = pytest.mark.gpu
E2M1 = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)


def _kv(T, H, D, dtype, seed, special=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, D, generator=g) * torch.exp(2 * torch.randn(T, H, 1, generator=g))
    if T > 1:
        x[1] = 0
    if special:
        x[0, 0, 1], x[0, 0, 2], x[0, 0, 3] = float("nan"), float("inf"), -0.0
    return x.to(dtype)


def _unswizzle(sf, rows, cols):
    """Scale bytes [rows, cols] from the 128 x 4 swizzled buffer."""
    R, C = sf.shape
    t = sf.view(R // 128, C // 4, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(R, C)
    return t[:rows, :cols]


def _rows(x, fmt):
    """(codes, scales) of rows [n, D] as the cache should hold them."""
    n, D = x.shape
    if fmt == "fp8":
        c, s = O.quant(x, "row", torch.float8_e4m3fn)
        return torch.from_numpy(c), torch.from_numpy(s)
    q, sf = _lib.quant_mxfp4(x.cuda())
    return q.cpu(), _unswizzle(sf.cpu(), n, D // 32)


def _bytes(cache):
    if cache.dtype == torch.float8_e4m3fn:
        return torch.from_numpy(O.codes_of(cache))
    return cache.cpu()


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
@pytest.mark.parametrize("T,H,D,page", [(1, 1, 32, 1), (3, 2, 64, 16), (40, 8, 128, 16), (70, 3, 160, 48), (17, 1, 576, 64), (700, 2, 96, 7)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_write_and_read(fmt, T, H, D, page, dtype):
    pages = T // page + 3
    g = torch.Generator().manual_seed(T)
    k, v = _kv(T, H, D, dtype, 1), _kv(T, H, D, dtype, 2)
    cache = kvcache.make_kv_cache(pages, page, H, D, fmt)
    for t in cache:
        t.view(torch.uint8).fill_(0x11)
    before = [t.clone() for t in cache]
    slots = torch.randperm(pages * page, generator=g)[:T]
    pad = torch.rand(T, generator=g) < 0.1
    slots_in = torch.where(pad, torch.where(torch.arange(T) % 2 == 0, -1, pages * page), slots)
    # keys and values as slices of one projection
    qkv = torch.cat([torch.zeros(T, 1, D, dtype=dtype), k, v], 1).cuda()
    kvcache.write_kv_cache(qkv[:, 1:1 + H], qkv[:, 1 + H:], slots_in.cuda(), *cache)
    live = ~pad
    for x, codes, scales, cb, sb in ((k, cache[0], cache[2], before[0], before[2]), (v, cache[1], cache[3], before[1], before[3])):
        want_c, want_s = _rows(x[live].reshape(-1, D), fmt)
        got_c, got_s = _bytes(codes).reshape(pages * page, H, -1), scales.cpu().reshape(pages * page, H, -1)
        assert torch.equal(got_c[slots[live]].reshape(want_c.shape), want_c)
        assert torch.equal(got_s[slots[live]].reshape(want_s.shape), want_s)
        rest = torch.ones(pages * page, dtype=torch.bool)
        rest[slots[live]] = False
        assert torch.equal(got_c[rest], _bytes(cb).reshape(got_c.shape)[rest])
        assert torch.equal(got_s[rest], sb.cpu().reshape(got_s.shape)[rest])


def _expected(codes, scales, fmt, D, slot):
    """Rows [n, H, D] in f64 of these slots (slot -1: zeros)."""
    H = codes.shape[2]
    if fmt == "fp8":
        c = torch.from_numpy(O.decode(codes)).reshape(-1, H, D)
        s = scales.cpu().double().reshape(-1, H, scales.shape[-1]).repeat_interleave(128, -1)[..., :D]
    else:
        b = codes.cpu().reshape(-1, H, D // 2).long()
        c = E2M1[torch.stack([b & 15, b >> 4], -1).flatten(-2)]
        s = torch.pow(2.0, scales.cpu().double().reshape(-1, H, D // 32) - 127).repeat_interleave(32, -1)
    x = (c * s)[slot.clamp(min=0)]
    x[slot < 0] = 0
    return x


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
@pytest.mark.parametrize("lens,H,D,page", [([1], 1, 32, 1), ([0, 5, 0, 17, 1, 0], 2, 64, 16), ([100, 3, 64, 65], 3, 160, 64), ([33] * 40, 1, 128, 8), ([257], 8, 576, 48)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_read_ragged(fmt, lens, H, D, page, dtype):
    g = torch.Generator().manual_seed(sum(lens))
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 2
    cache = kvcache.make_kv_cache(pages, page, H, D, fmt)
    for t in cache[:2]:
        r = torch.randint(0, 256, t.shape, generator=g, dtype=torch.int32).to(torch.uint8)
        if fmt == "fp8":
            r = torch.where((r & 0x7F) == 0x7F, 0, r).to(torch.uint8)
        t.view(torch.uint8).copy_(r)
    for t in cache[2:]:
        t.copy_(torch.rand(t.shape, generator=g) if fmt == "fp8" else torch.randint(120, 132, t.shape, generator=g))
    perm = torch.randperm(pages, generator=g)
    table = torch.full((len(lens), max(need) + 1), -7, dtype=torch.int32)
    at, slot = 0, []
    for i, n in enumerate(lens):
        table[i, :need[i]] = perm[at:at + need[i]]
        at += need[i]
        pos = torch.arange(n)
        slot.append(table[i].long()[pos // page] * page + pos % page)
    if len(lens) > 3 and need[3] > 0:      # pages that do not exist
        table[3, 0] = pages if fmt == "fp8" else -1
        slot[3][:page] = -1
    slot = torch.cat(slot)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    total = int(cu[-1])
    out = [torch.full((total + 3, H, D), 9.0, dtype=dtype, device="cuda") for _ in range(2)]
    got = kvcache.read_kv_cache(*cache, table.cuda(), cu.cuda(), out=out)
    fresh = kvcache.read_kv_cache(*cache, table.cuda(), cu.cuda(), total=total, dtype=dtype)
    for o, f, c, s in zip(got, fresh, cache[:2], cache[2:]):
        assert (o[total:] == 9).all()
        assert torch.equal(o[:total], f)
        want = _expected(c, s, fmt, D, slot)
        # the product is at most 5 + 24 bits: one rounding to f32, one to the type
        tol = want.abs() * (torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -20) + 2.0 ** -24) + (2.0 ** -25 if dtype == torch.float16 else 0)
        assert ((f.cpu().double() - want).abs() <= tol).all()


def test_read_into_strided_rows_and_one_tensor():
    cache = kvcache.make_kv_cache(4, 8, 2, 64, values=False)
    k = _kv(20, 2, 64, torch.bfloat16, 3).cuda()
    kvcache.write_kv_cache(k, None, torch.arange(20, device="cuda"), cache[0], None, cache[2], None)
    table = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    cu = torch.tensor([0, 20], dtype=torch.int32, device="cuda")
    want, none = kvcache.read_kv_cache(cache[0], None, cache[2], None, table, cu, total=20)
    assert none is None
    for width, off in ((200, 8), (131, 1)):          # 16-byte and 2-byte aligned rows
        big = torch.full((21, width), 3.0, dtype=torch.bfloat16, device="cuda")
        view = big[:20, off:off + 128].unflatten(1, (2, 64))
        kvcache.read_kv_cache(cache[0], None, cache[2], None, table, cu, out=(view, None))
        assert torch.equal(view, want)
        assert (big[20] == 3).all() and (big[:, :off] == 3).all() and (big[:, off + 128:] == 3).all()


@pytest.mark.parametrize("T", [2, 50, 5000])
def test_same_slot_twice_keeps_the_last(T):
    g = torch.Generator().manual_seed(T)
    H, D, page = 2, 64, 16
    pages = max(1, T // 40)
    slots = torch.randint(0, pages * page, (T,), generator=g)
    slots[T // 2:][torch.rand(T - T // 2, generator=g) < 0.3] = -1
    k, v = _kv(T, H, D, torch.bfloat16, 4).cuda(), _kv(T, H, D, torch.bfloat16, 5).cuda()
    cache = kvcache.make_kv_cache(pages, page, H, D)
    kvcache.write_kv_cache(k, v, slots.cuda(), *cache)
    last = {int(s): i for i, s in enumerate(slots.tolist()) if s >= 0}
    one = kvcache.make_kv_cache(pages, page, H, D)
    at = torch.tensor(list(last.values())).cuda()
    kvcache.write_kv_cache(k[at], v[at], torch.tensor(list(last.keys())).cuda(), *one)
    for a, b in zip(cache, one):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_special_values():
    k = _kv(4, 2, 128, torch.bfloat16, 6, special=True)
    cache = kvcache.make_kv_cache(1, 4, 2, 128, values=False)
    kvcache.write_kv_cache(k.cuda(), None, torch.arange(4, device="cuda"), cache[0], None, cache[2], None)
    c, s = O.quant(k.reshape(-1, 128), "row", torch.float8_e4m3fn)
    assert (O.codes_of(cache[0]).reshape(-1, 128) == c).all() and (cache[2].cpu().numpy().reshape(-1, 1) == s).all()
    # bf16 and fp16 rows of subnormals, powers of two and the largest values, in 4 bits
    for dtype in (torch.bfloat16, torch.float16):
        f = torch.finfo(dtype)
        rows = torch.stack([torch.full((32,), v, dtype=torch.float64) for v in (f.tiny, f.tiny / 4, f.max, 6.0, 3.0, 1.0, 6.0625, 2.0 ** -14)])
        rows = (rows * torch.linspace(-1, 1, 32)).to(dtype).unsqueeze(1)
        m = kvcache.make_kv_cache(1, 8, 1, 32, "mxfp4", values=False)
        kvcache.write_kv_cache(rows.cuda(), None, torch.arange(8, device="cuda"), m[0], None, m[2], None)
        want_c, want_s = _rows(rows.reshape(8, 32), "mxfp4")
        assert torch.equal(m[0].cpu().reshape(8, 16), want_c) and torch.equal(m[2].cpu().reshape(8, 1), want_s)


def test_append_and_read_captured():
    """A decode step's write and read in one graph, replayed with new tokens, slots and lengths."""
    H, D, page, B = 4, 128, 16, 3
    cache = kvcache.make_kv_cache(12, page, H, D)
    table = torch.arange(12, dtype=torch.int32, device="cuda").reshape(3, 4)
    k = torch.zeros(B, H, D, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    slots = torch.zeros(B, dtype=torch.int64, device="cuda")
    cu = torch.zeros(B + 1, dtype=torch.int32, device="cuda")
    out = (torch.zeros(B * 4, H, D, dtype=torch.bfloat16, device="cuda"), torch.zeros(B * 4, H, D, dtype=torch.bfloat16, device="cuda"))
    slots.fill_(-1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kvcache.write_kv_cache(k, v, slots, *cache)
        kvcache.read_kv_cache(*cache, table, cu, out=out)
    seen = [[], []]
    for step in range(4):
        new = _kv(B, H, D, torch.bfloat16, 10 + step), _kv(B, H, D, torch.bfloat16, 20 + step)
        k.copy_(new[0])
        v.copy_(new[1])
        slots.copy_(table[:, 0].long() * page + step)
        cu.copy_(torch.arange(B + 1) * (step + 1))
        graph.replay()
        for i in range(2):
            q, s = fp8.quant_fp8(new[i].reshape(-1, D).cuda())
            seen[i].append((q.float() * s).reshape(B, H, D).to(torch.bfloat16))
            want = torch.stack(seen[i], 1).flatten(0, 1)
            assert torch.equal(out[i][:B * (step + 1)], want)


def test_far_slots():
    """Slots whose byte offsets pass 2^31 and 2^32."""
    H, D, page = 8, 512, 64
    pages = (5 << 30) // (H * D * page) + 1
    cache = (torch.empty(pages, page, H, D, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn), None,
             torch.empty(pages, page, H, 4, device="cuda"), None)
    slots = torch.tensor([0, (1 << 31) // (H * D) + 5, (1 << 32) // (H * D) + 77, pages * page - 1], device="cuda")
    k = _kv(4, H, D, torch.bfloat16, 8).cuda()
    kvcache.write_kv_cache(k, None, slots, cache[0], None, cache[2], None)
    table = (slots // page).to(torch.int32)[:, None]
    q, s = fp8.quant_fp8(k.reshape(-1, D))
    for i in range(4):
        n = int(slots[i] % page) + 1
        cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        got, _ = kvcache.read_kv_cache(cache[0], None, cache[2], None, table[i:i + 1], cu, total=n, dtype=torch.float32)
        want = (q.float() * s.repeat_interleave(128, 1)).reshape(4, H, D)[i]
        assert torch.equal(got[n - 1], want)


def test_refusals():
    cache = kvcache.make_kv_cache(2, 8, 2, 64)
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device="cuda")
    slots = torch.zeros(3, dtype=torch.int64, device="cuda")
    for bad, msg in [((k.float(), k.float(), slots), "float16 or bfloat16"), ((k[:, :1], k[:, :1], slots), "k must be"), ((k, k[:2], slots), "v must"),
                     ((k, k, slots.int()), "slots"), ((k, k, slots[:2]), "slots"), ((k, None, slots), "go together"), ((k.cpu(), k, slots), "device")]:
        with pytest.raises(RuntimeError, match=msg):
            kvcache.write_kv_cache(*bad, *cache)
    table = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    cu = torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad, kw, msg in [((table.long(), cu), dict(total=1), "block_table"), ((table, cu[:1]), dict(total=1), "cu_lens"), ((table, cu), {}, "needs total"),
                         ((table, cu), dict(total=1, dtype=torch.float64), "dtype must be"), ((table.cpu(), cu), dict(total=1), "device"),
                         ((table, cu), dict(out=(k, None)), "a tensor for each"), ((table, cu), dict(out=(k, k[:, :1])), "out must be"),
                         ((table, cu), dict(out=(k, k), total=2), "total must"), ((table, cu), dict(out=(k.transpose(1, 2).contiguous().transpose(1, 2),) * 2), "contiguous")]:
        with pytest.raises(RuntimeError, match=msg):
            kvcache.read_kv_cache(*cache, *bad, **kw)


def test_registered_operators():
    import emugen_b200.ops  # noqa: F401

    k, v = _kv(20, 2, 64, torch.bfloat16, 1).cuda(), _kv(20, 2, 64, torch.bfloat16, 2).cuda()
    a, b = kvcache.make_kv_cache(3, 8, 2, 64, "mxfp4"), kvcache.make_kv_cache(3, 8, 2, 64, "mxfp4")
    slots = torch.arange(20, device="cuda")
    table = torch.arange(3, dtype=torch.int32, device="cuda")[None]
    cu = torch.tensor([0, 20], dtype=torch.int32, device="cuda")
    torch.ops.emugen.write_kv_cache(k, v, slots, *a)
    kvcache.write_kv_cache(k, v, slots, *b)
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    for x, y in zip(torch.ops.emugen.read_kv_cache(*a, table, cu, 20), kvcache.read_kv_cache(*b, table, cu, total=20)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("H,D", [(3, 128), (1, 32), (5, 48), (7, 64), (1, 144)])
@pytest.mark.parametrize("T", [1, 2, 601, 1500])
@pytest.mark.parametrize("values", [False, True])
def test_odd_numbers_of_groups(H, D, T, values):
    """Lane groups of one warp that belong to different tokens, with and without a value cache."""
    k, v = _kv(T, H, D, torch.bfloat16, 1), _kv(T, H, D, torch.bfloat16, 2)
    c = kvcache.make_kv_cache(T // 16 + 1, 16, H, D, values=values)
    slots = torch.randperm((T // 16 + 1) * 16, generator=torch.Generator().manual_seed(T))[:T]
    kvcache.write_kv_cache(k.cuda(), v.cuda() if values else None, slots.cuda(), *c)
    for x, codes, scales in ((k, c[0], c[2]),) + (((v, c[1], c[3]),) if values else ()):
        want_c, want_s = _rows(x.reshape(-1, D), "fp8")
        assert torch.equal(_bytes(codes).reshape(-1, H, D)[slots].reshape(want_c.shape), want_c)
        assert torch.equal(scales.cpu().reshape(-1, H, scales.shape[-1])[slots].reshape(want_s.shape), want_s)


def test_slots_far_apart_and_many_times():
    """Slots a power of two apart (one bucket of a low-bits hash) and one slot for all tokens."""
    T, H, D = 900, 1, 32
    k = _kv(T, H, D, torch.bfloat16, 3).cuda()
    c = kvcache.make_kv_cache(T, 4096, H, D, values=False)
    kvcache.write_kv_cache(k, None, torch.arange(T, device="cuda") * 4096, c[0], None, c[2], None)
    want_c, want_s = _rows(k.cpu().reshape(T, D), "fp8")
    assert torch.equal(_bytes(c[0])[:, 0].reshape(T, D), want_c) and torch.equal(c[2].cpu()[:, 0].reshape(T, 1), want_s)
    kvcache.write_kv_cache(k, None, torch.full((T,), 7, device="cuda"), c[0], None, c[2], None)
    assert torch.equal(_bytes(c[0])[0, 7].reshape(1, D), want_c[-1:]) and c[2].cpu()[0, 7, 0, 0] == want_s[-1, 0]
