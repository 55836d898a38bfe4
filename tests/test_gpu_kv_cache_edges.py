"""The quantised cache at its edges: scale bytes at the ends of their range, products beside ties, padding past the
cache and repeated slots in long calls, a cache without pages."""
import pytest
import torch

from emugen_b200 import kvcache
from tests.test_gpu_kv_cache import E2M1, _kv

pytestmark = pytest.mark.gpu


def _read_all(cache, rows, dtype):
    pages = cache[0].shape[0]
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    cu = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    return kvcache.read_kv_cache(*cache, table, cu, total=rows, dtype=dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_mxfp4_scale_bytes_of_the_whole_range(dtype):
    """Every scale byte with every code: code * 2^(byte - 127) in f32 (byte 255, 2^128: infinity), rounded to the type."""
    cache = kvcache.make_kv_cache(4, 64, 1, 32, "mxfp4")
    code = torch.arange(32, dtype=torch.int32) % 16
    packed = (code[0::2] | (code[1::2] << 4)).to(torch.uint8)
    for c, s in ((cache[0], cache[2]), (cache[1], cache[3])):
        c.copy_(packed.expand(4, 64, 1, 16))
        s.copy_(torch.arange(256).to(torch.uint8).reshape(4, 64, 1, 1))
    scale = torch.pow(2.0, torch.arange(256, dtype=torch.float64) - 127)
    scale[255] = float("inf")
    want = (E2M1[code.long()][None] * scale[:, None]).float().to(dtype)       # exact in f32 up to its range's end
    assert want[0].double().abs().max() == (6 * 2.0 ** -127 if dtype != torch.float16 else 0)
    for got in _read_all(cache, 256, dtype):
        got = got.cpu()[:, 0]
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(7.0, 8.0, 9.0), want.nan_to_num(7.0, 8.0, 9.0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_fp8_products_are_rounded_to_f32_and_then_to_the_type(dtype):
    """Scales whose products with a code lie beside a tie of the type: the two roundings that are documented."""
    g = torch.Generator().manual_seed(1)
    D = 128
    cache = kvcache.make_kv_cache(16, 64, 1, D, values=False)
    bits = 8 if dtype == torch.bfloat16 else 11
    tie = torch.randint(2 ** bits, 2 ** (bits + 1), (1024,), generator=g) | 1           # bits + 1 bits, the last one set
    code = torch.randint(1, 16, (1024, D), generator=g).float() / 8
    scale = (tie.double() * 2.0 ** -bits / code[:, 0].double()).float()                 # code * scale next to the tie
    scale = torch.where(torch.arange(1024) % 3 == 0, torch.nextafter(scale, torch.tensor(2.0)), scale)
    cache[0].view(torch.uint8).copy_(code.to(torch.float8_e4m3fn).view(torch.uint8).reshape(16, 64, 1, D))
    cache[2].copy_(scale.reshape(16, 64, 1, 1))
    got, _ = _read_all((cache[0], None, cache[2], None), 1024, dtype)
    f32 = code * scale[:, None]
    assert torch.equal(got.cpu()[:, 0], f32.to(dtype))
    once = code.double() * scale.double()[:, None]                                      # at most half a step of the type and of f32
    assert ((got.cpu()[:, 0].double() - once).abs() <= once * (torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -24) + 2.0 ** -24)).all()


def _written(k, slots, pages, page):
    """The cache after one call with each slot's last row (k: every token's)."""
    n = pages * page
    last = torch.full((n,), -1, dtype=torch.int64)
    live = (slots >= 0) & (slots < n)
    at = torch.arange(len(slots))[live]
    last.scatter_reduce_(0, slots[live], at, "amax")
    where = torch.arange(n)[last >= 0]
    cache = kvcache.make_kv_cache(pages, page, *k.shape[1:], values=False)
    for w in where.split(100):                       # short calls of distinct slots
        kvcache.write_kv_cache(k[last[w].cuda()], None, w.cuda(), cache[0], None, cache[2], None)
    return cache


@pytest.mark.parametrize("T,pages,padding", [(160000, 80, -1), (160000, 80, 80 * 16), (160000, 1, 1 << 40), (5000, 20, 20 * 16), (700, 3, 3 * 16)])
def test_long_calls_with_repeated_slots_and_padding(T, pages, padding):
    """More tokens than 1024 for each SM, every slot many times over, a third of the tokens padding before or past the cache."""
    g = torch.Generator().manual_seed(T)
    k = _kv(T, 1, 32, torch.bfloat16, 7).cuda()
    slots = torch.randint(0, pages * 16, (T,), generator=g)
    slots[torch.rand(T, generator=g) < 0.33] = padding
    cache = kvcache.make_kv_cache(pages, 16, 1, 32, values=False)
    kvcache.write_kv_cache(k, None, slots.cuda(), cache[0], None, cache[2], None)
    want = _written(k, slots, pages, 16)
    assert torch.equal(cache[0].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(cache[2], want[2])


def _us(f, n=5):
    f()
    best = float("inf")
    for _ in range(n):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        f()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b) * 1e3)
    return best


@pytest.mark.parametrize("slot", [1 << 40, 5])
def test_padding_and_repeated_slots_cost_no_more_than_rows(slot):
    """A call whose tokens are all padding past the cache, or all of one slot, is not slower than one that writes them
    all (a factor of two for the clock): they write next to nothing."""
    T = 131072
    k = _kv(T, 8, 128, torch.bfloat16, 9).cuda()
    cache = kvcache.make_kv_cache(T // 64, 64, 8, 128, values=False)
    many = torch.randperm(T, generator=torch.Generator().manual_seed(2)).cuda()
    one = torch.full((T,), slot, dtype=torch.int64, device="cuda")
    write = lambda s: kvcache.write_kv_cache(k, None, s, cache[0], None, cache[2], None)
    assert _us(lambda: write(one)) <= 2 * _us(lambda: write(many))


def test_a_cache_without_pages_reads_as_zeros():
    for fmt in ("fp8", "mxfp4"):
        cache = [t[:0] for t in kvcache.make_kv_cache(1, 16, 2, 64, fmt)]
        table = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
        cu = torch.tensor([0, 3, 8], dtype=torch.int32, device="cuda")
        out = [torch.full((9, 2, 64), 5.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        kvcache.read_kv_cache(*cache, table, cu, out=out)
        for o in out:
            assert (o[:8] == 0).all() and (o[8] == 5).all()
        kvcache.write_kv_cache(*[torch.ones(3, 2, 64, dtype=torch.bfloat16, device="cuda")] * 2, torch.arange(3, device="cuda"), *cache)
