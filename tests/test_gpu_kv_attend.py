"""Attention of one token for each sequence over the quantised cache, against 64 bits on the rows as they are stored."""
import pytest
import torch

from emugen_b200 import attention, kvcache
from tests import attention_oracle as O

pytestmark = pytest.mark.gpu
E2M1 = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)


def _stored(codes, scales, fmt):
    """Every slot's rows as 64-bit values [slots, heads, head_size]."""
    if fmt == "fp8":
        x = codes.cpu().float().double().flatten(0, 1)
        return x * scales.cpu().double().flatten(0, 1).repeat_interleave(128, -1)[..., :x.shape[-1]]
    b = codes.cpu().flatten(0, 1)
    x = E2M1[torch.stack([b & 15, b >> 4], -1).flatten(-2).long()]
    s = scales.cpu().flatten(0, 1).double()
    f = torch.where(s == 255, torch.inf, torch.pow(2.0, s - 127))
    return x * f.repeat_interleave(32, -1)


def _make(lens, Hq, Hk, D, page, fmt, dtype, seed, spread=1.0):
    """(q, cache, table, lens): random rows written through the cache's own writer at shuffled pages."""
    g = torch.Generator().manual_seed(seed)
    need = [(n + page - 1) // page for n in lens]
    pages = sum(need) + 2
    cache = kvcache.make_kv_cache(pages, page, Hk, D, fmt)
    perm = torch.randperm(pages, generator=g)
    table = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += n
    slots = torch.cat([table[i].long()[torch.arange(n) // page] * page + torch.arange(n) % page for i, n in enumerate(lens)] + [torch.zeros(0, dtype=torch.int64)])
    T = len(slots)
    for t in cache:                                   # what was never written holds the worst
        t.view(torch.uint8).fill_(0xFF)
    if T:
        k, v = ((torch.randn(T, Hk, D, generator=g) * torch.exp(spread * torch.randn(T, Hk, 1, generator=g))).to(dtype).cuda() for _ in range(2))
        kvcache.write_kv_cache(k, v, slots.cuda(), *cache)
    q = torch.randn(len(lens), Hq, D, generator=g).to(dtype).cuda()
    return q, cache, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()


def _want(q, cache, table, lens, fmt, scale, page):
    k, v = (_stored(cache[i], cache[i + 2], fmt) for i in (0, 1))
    pages = cache[0].shape[0]
    block = 128 if fmt == "fp8" else 32
    ks, vs, low, cu = [], [], [], [0]
    for b, n in enumerate(lens.tolist()):
        n = max(0, min(n, table.shape[1] * page))
        pos = torch.arange(n)
        pg = table[b].cpu().long()[pos // page] if n else pos
        ok = (pg >= 0) & (pg < pages)
        at = (pg * page + pos % page)[ok]
        ks.append(k[at]), vs.append(v[at]), cu.append(cu[-1] + len(at))
        # A weight p * scale is put to 2^6 times its share of at most twice the largest scale of the values' block (some p
        # is 1 or more) and rounded to fp16: half a subnormal step, 2^-25, is 2^-31 of that scale, times the code.
        s = cache[3].cpu().flatten(0, 1)[at].double() if fmt == "fp8" else torch.pow(2.0, cache[3].cpu().flatten(0, 1)[at].double() - 127)
        s = s.nan_to_num(0, 0, 0)
        code = v[at].abs() / s.repeat_interleave(block, -1)[..., :v.shape[-1]].clamp(min=1e-300)
        top = s.amax(0, keepdim=True) if len(at) else s
        low.append((code * top.repeat_interleave(block, -1)[..., :v.shape[-1]] * 2.0 ** -31).nan_to_num(0, 0, 0))
    kk, vv = torch.cat(ks).cuda(), torch.cat(vs).cuda()
    r = O.attention(q, kk, vv, list(range(len(lens) + 1)), cu, False, scale, p_step=2.0 ** -11, v_low=torch.cat(low).cuda())
    return r["out"], (r["lse"][0].t(), r["lse"][1].t())


def _check(lens, Hq, Hk, D, page, fmt, dtype, seed=0, scale=None, spread=1.0):
    q, cache, table, n = _make(lens, Hq, Hk, D, page, fmt, dtype, seed, spread)
    out, lse = kvcache.attend_kv_cache(q, *cache, table, n, scale=scale, return_lse=True)
    o, l = _want(q, cache, table, n, fmt, D ** -0.5 if scale is None else scale, page)
    O.check(out, o, "out")
    O.check(lse, l, "lse")


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,page", [([1], 1), ([0], 16), ([5, 0, 17, 64], 16), ([300], 7), ([15, 16, 17, 31, 32, 33], 16), ([1000, 3], 48), ([129] * 9, 128), ([2500, 1, 0, 70], 64)])
def test_lengths_and_pages(fmt, dtype, lens, page):
    _check(lens, 8, 2, 64, page, fmt, dtype, seed=len(lens))


@pytest.mark.parametrize("fmt,D", [("fp8", d) for d in (16, 32, 48, 64, 80, 112, 128, 144, 192, 240, 256)] + [("mxfp4", d) for d in (32, 64, 96, 128, 160, 224, 256)])
@pytest.mark.parametrize("Hq,Hk", [(1, 1), (7, 1), (8, 8), (24, 2), (40, 1), (64, 2)])
def test_head_sizes_and_groups(fmt, D, Hq, Hk):
    _check([100, 37], Hq, Hk, D, 16, fmt, torch.bfloat16 if D % 64 else torch.float16, seed=D + Hq)


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
@pytest.mark.parametrize("lens", [[20000], [9000, 40, 3000, 1], [64] * 200])
def test_long_and_many(fmt, lens):
    _check(lens, 8, 2, 128, 16, fmt, torch.bfloat16, seed=3)


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
@pytest.mark.parametrize("Hq,Hk", [(8, 4), (96, 4), (12, 12), (18, 6), (32, 8), (10, 10)])
@pytest.mark.parametrize("lens", [[3000, 0, 70, 1], [64] * 90], ids=["ragged", "many"])
def test_neighbouring_heads_side_by_side(fmt, Hq, Hk, lens):
    """Slots with long rows, whose heads go to CTAs in sets of 2 or 4; some sets' runs end inside sequences."""
    _check(lens, Hq, Hk, 256, 16, fmt, torch.bfloat16, seed=Hq)


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
@pytest.mark.parametrize("spread,scale", [(4.0, None), (0.1, 3.0), (1.0, 1e-3)])
def test_scales_far_apart_and_peaked_scores(fmt, spread, scale):
    _check([700, 33], 8, 2, 64, 16, fmt, torch.float16 if spread < 2 else torch.bfloat16, seed=4, spread=spread, scale=scale)


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
def test_pages_that_do_not_exist_are_not_seen(fmt):
    q, cache, table, lens = _make([200, 90, 64], 4, 2, 64, 16, fmt, torch.bfloat16, 6)
    pages = cache[0].shape[0]
    table[0, 3], table[0, 12], table[1, 0], table[1, 5] = -1, pages, 2 ** 31 - 1, -2 ** 31
    table[2] = -1
    lens[0] = 10 ** 9                                 # longer than the table: all of it
    out, lse = kvcache.attend_kv_cache(q, *cache, table, lens, return_lse=True)
    o, l = _want(q, cache, table, lens, fmt, 64 ** -0.5, 16)
    O.check(out, o), O.check(lse, l)
    assert (out[2] == 0).all() and (lse[2] == float("-inf")).all()
    lens[:] = torch.tensor([-5, 0, -2 ** 31], dtype=torch.int32)
    assert (kvcache.attend_kv_cache(q, *cache, table, lens) == 0).all()
    empty = kvcache.make_kv_cache(1, 16, 2, 64, fmt)
    none = [t[:0] for t in empty]
    assert (kvcache.attend_kv_cache(q, *none, table, lens.fill_(40)) == 0).all()
    assert (kvcache.attend_kv_cache(q, *cache, table[:, :0], lens) == 0).all()


def test_nan_rows_spread_to_their_sequence_alone():
    q, cache, table, lens = _make([100, 100], 4, 2, 64, 16, "fp8", torch.bfloat16, 7)
    slot = int(table[0, 2]) * 16 + 3
    cache[1].view(torch.uint8).flatten(0, 1)[slot, 1, 9] = 0x7F
    out = kvcache.attend_kv_cache(q, *cache, table, lens)
    nan = out.isnan()
    assert nan[0, 2:, 9].all() and int(nan.sum()) == 2
    cache[0].view(torch.uint8).flatten(0, 1)[slot, 0, 9] = 0x7F
    nan = kvcache.attend_kv_cache(q, *cache, table, lens).isnan()
    assert nan[0, :2].all() and int(nan.sum()) == 2 * 64 + 2


def test_queries_of_any_size():
    """Queries near bf16's largest and smallest values: they are not put into a narrower type as they are."""
    for factor, scale in ((1e30, 1e-31), (1e-30, 1e29)):
        q, cache, table, lens = _make([77], 4, 2, 64, 16, "fp8", torch.bfloat16, 8)
        q = (q.float() * factor).to(torch.bfloat16)
        q[0, 0, :5] = 0
        q[0, 1] = 0
        out = kvcache.attend_kv_cache(q, *cache, table, lens, scale=scale)
        O.check(out, _want(q, cache, table, lens, "fp8", scale, 16)[0])


def test_layouts():
    q, cache, table, lens = _make([50, 260, 3], 8, 2, 64, 16, "fp8", torch.bfloat16, 9)
    want = kvcache.attend_kv_cache(q, *cache, table, lens)
    fused = torch.cat([q, q], 1)
    wide = torch.cat([table, table], 1)
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(q.shape).copy_(q)
    for qq, t in ((fused[:, 8:], table), (q.transpose(0, 1).contiguous().transpose(0, 1), table), (q.permute(2, 0, 1).contiguous().permute(1, 2, 0), table),
                  (odd, table), (q, wide[:, :table.shape[1]]), (q, table.t().contiguous().t())):
        assert torch.equal(kvcache.attend_kv_cache(qq, *cache, t, lens), want)
    shared = table[:1].expand(3, -1)                   # three continuations of one prompt
    n = lens.clone().fill_(40)
    a = kvcache.attend_kv_cache(q, *cache, shared, n)
    assert torch.equal(a, kvcache.attend_kv_cache(q, *cache, shared.contiguous(), n))


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
def test_far_slots(fmt):
    """Codes more than 2^31 bytes into the cache."""
    D, Hk, page = 256, 16, 64
    row = Hk * (D if fmt == "fp8" else D // 2)
    pages = (2 ** 31 // row + 4096) // page
    cache = kvcache.make_kv_cache(pages, page, Hk, D, fmt)
    n = 100
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(n, Hk, D, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    slots = pages * page - 1 - torch.arange(n)
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32)
    kvcache.write_kv_cache(k, v, slots.cuda(), *cache)
    q = torch.randn(1, 32, D, generator=g).to(torch.bfloat16).cuda()
    lens = torch.tensor([2 * page], dtype=torch.int32).cuda()
    out = kvcache.attend_kv_cache(q, *cache, table.cuda(), lens)
    two = [t[-2:].contiguous() for t in cache]
    small = torch.tensor([[1, 0]], dtype=torch.int32).cuda()
    assert torch.equal(out, kvcache.attend_kv_cache(q, *two, small, lens))
    O.check(out, _want(q, two, small, lens, fmt, D ** -0.5, page)[0])


def test_same_result_every_run_streams_and_graph_replay():
    q, cache, table, lens = _make([5000, 100, 1, 0, 900], 16, 2, 128, 16, "fp8", torch.bfloat16, 10)
    want = kvcache.attend_kv_cache(q, *cache, table, lens)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(kvcache.attend_kv_cache(q, *cache, table, lens))
    torch.cuda.synchronize()
    assert all(torch.equal(t, want) for t in got)
    graphs = []
    for _ in range(2):                                # two graphs that may share their workspace's memory
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r = kvcache.attend_kv_cache(q, *cache, table, lens)
        graphs.append((graph, r))
    for _ in range(2):
        for graph, r in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(r, want)
    lens.copy_(torch.tensor([4000, 0, 1, 0, 901 // 2], dtype=torch.int32))     # the graph reads the lengths as they are
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], kvcache.attend_kv_cache(q, *cache, table, lens))


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
def test_a_prompt_and_the_tokens_after_it(fmt):
    """A run of the operators as they are used: the prompt's queries and keys normalised and turned, attended to and
    written to the cache; then token by token norms, cache write, attention over the cache."""
    Hq, Hk, D, page, dtype = 8, 2, 64, 16, torch.bfloat16
    lens = [37, 5, 64]
    steps = 3
    g = torch.Generator().manual_seed(11)
    half = D // 2
    angle = torch.arange(256, dtype=torch.float64)[:, None] * torch.pow(10000.0, -torch.arange(half, dtype=torch.float64) / half)
    cos, sin = torch.cos(angle).float().cuda(), torch.sin(angle).float().cuda()
    wq, wk = ((1 + 0.2 * torch.randn(D, generator=g)).to(dtype).cuda() for _ in range(2))
    cols = 8
    table = torch.randperm(3 * cols, generator=g).to(torch.int32).view(3, cols).cuda()
    cache = kvcache.make_kv_cache(3 * cols, page, Hk, D, fmt)

    def slots(seq, pos):
        return table.long()[seq, pos // page] * page + pos % page

    seq = torch.cat([torch.full((n,), i) for i, n in enumerate(lens)]).cuda()
    pos = torch.cat([torch.arange(n) for n in lens]).cuda()
    qkv = torch.randn(len(pos), Hq + 2 * Hk, D, generator=g).to(dtype).cuda()
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:]
    yq, yk = attention.qk_norm_rope(q, k, wq, wk, cos, sin, pos)
    O.check(yk, O.norm_rope(k, wk, cos, sin, pos, 1e-6, False))
    cu = torch.tensor([0, 37, 42, 106], dtype=torch.int32).cuda()
    out = attention.packed_attention(yq, yk, v, cu)
    O.check(out, O.attention(yq, yk, v, cu.tolist(), cu.tolist(), True, D ** -0.5)["out"])
    kvcache.write_kv_cache(yk, v, slots(seq, pos), *cache)
    # the prompt's attention over its cached rows, read back
    ck, cv = kvcache.read_kv_cache(*cache, table, cu, total=len(pos), dtype=dtype)
    out = attention.packed_attention(yq, ck, cv, cu)
    O.check(out, O.attention(yq, ck, cv, cu.tolist(), cu.tolist(), True, D ** -0.5)["out"])
    n = torch.tensor(lens, dtype=torch.int32).cuda()
    for _ in range(steps):
        qkv = torch.randn(3, Hq + 2 * Hk, D, generator=g).to(dtype).cuda()
        at = n.long()
        yq, yk = attention.qk_norm_rope(qkv[:, :Hq], qkv[:, Hq:Hq + Hk], wq, wk, cos, sin, at)
        kvcache.write_kv_cache(yk, qkv[:, Hq + Hk:], slots(torch.arange(3).cuda(), at), *cache)
        n = n + 1
        got = kvcache.attend_kv_cache(yq, *cache, table, n)
        O.check(got, _want(yq, cache, table, n, fmt, D ** -0.5, page)[0])


def test_registered_operator():
    import emugen_b200.ops  # noqa: F401

    q, cache, table, lens = _make([50, 20], 4, 2, 64, 16, "fp8", torch.bfloat16, 12)
    assert torch.equal(torch.ops.emugen.attend_kv_cache(q, *cache, table, lens), kvcache.attend_kv_cache(q, *cache, table, lens))


def test_refusals_of_arguments():
    cache = kvcache.make_kv_cache(2, 4, 2, 64)
    q = torch.zeros(3, 4, 64, dtype=torch.float16, device="cuda")
    table, lens = torch.zeros(3, 1, dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
    for args, msg in [((q.float(), *cache, table, lens), "float16 or bfloat16"), ((q[:, :3], *cache, table, lens), "multiple of 2"),
                      ((q[..., :32], *cache, table, lens), "must be"), ((q, *cache, table.long(), lens), "block_table"), ((q, *cache, table[:2], lens), "block_table"),
                      ((q, *cache, table, lens.long()), "lens"), ((q, *cache, table, lens[:2]), "lens"), ((q.cpu(), *cache, table, lens), "device"),
                      ((q, *cache, table, lens.cpu()), "device")]:
        with pytest.raises(RuntimeError, match=msg):
            kvcache.attend_kv_cache(*args)
    big = kvcache.make_kv_cache(2, 4, 1, 272)
    with pytest.raises(RuntimeError, match="at most 256"):
        kvcache.attend_kv_cache(torch.zeros(3, 4, 272, dtype=torch.float16, device="cuda"), *big, table, lens)
    with pytest.raises(RuntimeError, match="scale"):
        kvcache.attend_kv_cache(q, *cache, table, lens, scale=0.0)
