"""Cases for the 8-bit block-scaled operators: the quantiser, the matrix product, the linear layer with
its backward pass, and the quantised key/value cache (write, read back).

``run`` computes a case in plain torch operations, or -- where ``own`` is set -- through the framework's
entry points.  ``exact`` restates every operator in 64 bits, written apart from the plain form.
"""
import math

import torch

own = False

DEV = "cuda"
F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
F8_MAX = {"e4m3": 448.0, "e5m2": 57344.0}
F8_BITS = {"e4m3": (3, -6), "e5m2": (2, -14)}      # stored significand bits, exponent of the smallest normal
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
ESZ = {"bf16": 2, "f16": 2, "f32": 4}
TINY = 2.0 ** -126


def listed():
    return [
        # the activations of eight decode tokens: latency
        {"name": "quant_row_8x4096", "op": "quant", "M": 8, "K": 4096, "dtype": "bf16", "fp8": "e4m3", "block": "row",
         "transposed": False},
        # a training layer's activations, quantised along the rows (forward) and down the columns (weight gradient)
        {"name": "quant_row_t_8192x8192", "op": "quant", "M": 8192, "K": 8192, "dtype": "bf16", "fp8": "e4m3",
         "block": "row", "transposed": True},
        # a weight of odd sizes in 128 x 128 tiles with its transpose (input gradient)
        {"name": "quant_tile_t_1411x4099", "op": "quant", "M": 1411, "K": 4099, "dtype": "f16", "fp8": "e4m3",
         "block": "tile", "transposed": True},
        # one decode token against a vocabulary projection: all of it is reading the weight
        {"name": "gemm_1x128256x4096", "op": "gemm", "M": 1, "N": 128256, "K": 4096, "a": "e4m3", "b": "e4m3",
         "block": "tile", "out": "bf16"},
        # a decode batch against an up projection
        {"name": "gemm_32x14336x4096", "op": "gemm", "M": 32, "N": 14336, "K": 4096, "a": "e4m3", "b": "e4m3",
         "block": "tile", "out": "bf16"},
        # a weight gradient's form (both operands scaled along their rows, e5m2 gradient) at ragged sizes
        {"name": "gemm_777x1500x1111", "op": "gemm", "M": 777, "N": 1500, "K": 1111, "a": "e5m2", "b": "e4m3",
         "block": "row", "out": "f32"},
        # a prompt's or a training batch's product: bound by the tensor cores
        {"name": "gemm_8192x8192x8192", "op": "gemm", "M": 8192, "N": 8192, "K": 8192, "a": "e4m3", "b": "e4m3",
         "block": "tile", "out": "bf16"},
        # a linear layer, forward and backward, over a batch of 4096 tokens
        {"name": "linear_4096x4096x4096", "op": "linear", "M": 4096, "N": 4096, "K": 4096, "dtype": "bf16"},
        # the same at small ragged sizes
        {"name": "linear_301x1000x520", "op": "linear", "M": 301, "N": 1000, "K": 520, "dtype": "bf16"},
        # a decode step's keys and values of 32 sequences into an 8-bit cache: latency
        {"name": "kv_write_32", "op": "kv_write", "T": 32, "H": 8, "D": 128, "page": 16, "pages": 256, "dtype": "bf16",
         "fmt": "fp8"},
        # a prompt's keys and values appended to a 4-bit cache and the whole of the sequences read back
        {"name": "kv_append_read_mxfp4", "op": "kv_append_read", "T": 8192, "B": 9, "total": 40000, "H": 8, "D": 128,
         "page": 64, "dtype": "bf16", "fmt": "mxfp4"},
        # the cached contexts of a batch of long sequences read back for a prefix's attention
        {"name": "kv_read_131072", "op": "kv_read", "B": 32, "total": 131072, "H": 8, "D": 128, "page": 16,
         "dtype": "bf16", "fmt": "fp8"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quant", "gemm", "gemm", "linear", "kv_write", "kv_append_read", "kv_read"])
    if op == "quant":
        m, k = _log(rng, 1, 8192), _log(rng, 16, 8192)
        return {"op": op, "M": m, "K": k, "dtype": rng.choice(["bf16", "f16", "f32"]), "fp8": rng.choice(["e4m3", "e5m2"]),
                "block": rng.choice(["row", "tile"]), "transposed": rng.random() < 0.5}
    if op == "gemm":
        return {"op": op, "M": _log(rng, 1, 8192), "N": _log(rng, 8, 8192), "K": _log(rng, 32, 8192),
                "a": rng.choice(["e4m3", "e4m3", "e5m2"]), "b": rng.choice(["e4m3", "e4m3", "e5m2"]),
                "block": rng.choice(["tile", "tile", "row"]), "out": rng.choice(["bf16", "f16", "f32"])}
    if op == "linear":
        return {"op": op, "M": _log(rng, 1, 4096), "N": _log(rng, 32, 4096), "K": _log(rng, 32, 4096),
                "dtype": rng.choice(["bf16", "f16"])}
    fmt = rng.choice(["fp8", "mxfp4"])
    d = 32 * rng.randint(1, 16)
    h = rng.randint(1, 16)
    page = rng.choice([1, 8, 16, 48, 64, 128])
    most = 131072 * 8 * 128 // (h * d)
    if op == "kv_write":
        t = _log(rng, 1, min(16384, most // 8))
        return {"op": op, "T": t, "H": h, "D": d, "page": page, "pages": t // page + rng.randint(2, 64),
                "dtype": rng.choice(["bf16", "f16"]), "fmt": "fp8"}
    b = _log(rng, 1, 128)
    total = max(b, _log(rng, 16, min(131072, most // 2)))
    if op == "kv_read":
        return {"op": op, "B": b, "total": total, "H": h, "D": d, "page": page, "dtype": rng.choice(["bf16", "f16", "f32"]),
                "fmt": fmt}
    return {"op": op, "T": _log(rng, b, max(b + 1, total // 2)), "B": b, "total": total, "H": h, "D": d, "page": page,
            "dtype": rng.choice(["bf16", "f16"]), "fmt": fmt}


# ------------------------------------------------------------------------------------- inputs

def _activations(g, m, k, dtype):
    """Rows of unit scale with a few outlier channels and a few silent ones."""
    x = torch.randn(m, k, generator=g, device=DEV)
    f = torch.rand(k, generator=g, device=DEV)
    x *= torch.where(f < 0.01, 40.0, torch.where(f > 0.99, 0.0, 1.0))
    return x.to(DT[dtype])


def _f8_matrix(g, m, k, kind):
    """Codes as the quantiser leaves them: rows start on 16 bytes, the largest magnitudes near the type's."""
    pitch = (k + 15) // 16 * 16
    x = torch.randn(m, pitch, generator=g, device=DEV) * (F8_MAX[kind] / 4)
    return x.clamp_(-F8_MAX[kind], F8_MAX[kind]).to(F8[kind])[:, :k]


def _scales(g, rows, kb, kind):
    """Scales as the quantiser leaves them: [rows, blocks], stored block after block; values of about one."""
    pitch = (rows + 3) // 4 * 4
    s = torch.exp(torch.randn(kb, pitch, generator=g, device=DEV) * 0.5) * (4 / F8_MAX[kind])
    return s.t()[:rows]


def _cache_geometry(g, lens, page):
    """A shuffled block table for sequences of these lengths, and the number of pages."""
    need = [(n + page - 1) // page for n in lens]
    pages = sum(need) + 3
    perm = torch.randperm(pages, generator=g, device=DEV).to(torch.int32).cpu()
    table = torch.full((len(lens), max(max(need), 1)), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += n
    return table, pages


def _split(seed, total, parts):
    """total into `parts` positive lengths, unevenly."""
    r = torch.Generator().manual_seed(seed)
    w = torch.rand(parts, generator=r).pow(2) + 0.01
    n = (w / w.sum() * (total - parts)).floor().long() + 1
    n[0] += total - int(n.sum())
    return [int(v) for v in n]


def _cache(g, pages, page, h, d, fmt):
    """A cache that holds earlier tokens."""
    def part():
        if fmt == "fp8":
            x = (torch.randn(pages, page, h, d, generator=g, device=DEV) * 110).clamp_(-448, 448)
            s = torch.rand(pages, page, h, (d + 127) // 128, generator=g, device=DEV) * 0.02 + 1e-3
            return x.to(torch.float8_e4m3fn), s
        x = torch.randint(0, 256, (pages, page, h, d // 2), generator=g, device=DEV, dtype=torch.uint8)
        s = torch.randint(120, 130, (pages, page, h, d // 32), generator=g, device=DEV, dtype=torch.uint8)
        return x, s
    (k, ks), (v, vs) = part(), part()
    return {"k_cache": k, "v_cache": v, "k_scale": ks, "v_scale": vs}


def _new_kv(g, t, h, d, dtype):
    """Keys and values as slices of a fused projection's output (two query heads for each of theirs)."""
    qkv = torch.randn(t, 4 * h, d, generator=g, device=DEV)
    qkv *= torch.exp(torch.randn(1, 4 * h, d, generator=g, device=DEV) * 0.5)
    qkv = qkv.to(DT[dtype])
    return qkv[:, 2 * h:3 * h], qkv[:, 3 * h:]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    op = case["op"]
    st = {"case": case}
    if op == "quant":
        st["x"] = _activations(g, case["M"], case["K"], case["dtype"])
    elif op == "gemm":
        m, n, k = case["M"], case["N"], case["K"]
        kb = (k + 127) // 128
        st["a"], st["b"] = _f8_matrix(g, m, k, case["a"]), _f8_matrix(g, n, k, case["b"])
        st["sa"] = _scales(g, m, kb, case["a"])
        st["sb"] = _scales(g, n if case["block"] == "row" else (n + 127) // 128, kb, case["b"])
        if case["block"] == "tile":
            st["sb"] = st["sb"].contiguous()
    elif op == "linear":
        m, n, k = case["M"], case["N"], case["K"]
        st["x"] = _activations(g, m, k, case["dtype"]).requires_grad_()
        st["w"] = (torch.randn(n, k, generator=g, device=DEV) * k ** -0.5).to(DT[case["dtype"]]).requires_grad_()
        st["dy"] = torch.randn(m, n, generator=g, device=DEV).to(DT[case["dtype"]])
    elif op == "kv_write":
        t, h, d = case["T"], case["H"], case["D"]
        st.update(_cache(g, case["pages"], case["page"], h, d, case["fmt"]))
        st["k"], st["v"] = _new_kv(g, t, h, d, case["dtype"])
        slots = torch.randperm(case["pages"] * case["page"], generator=g, device=DEV)[:t]
        # one token in thirty is padding
        st["slots"] = torch.where(torch.rand(t, generator=g, device=DEV) < 1 / 30, -1, slots)
    else:
        b, total, h, d, page = case["B"], case["total"], case["H"], case["D"], case["page"]
        lens = _split(seed, total, b)
        table, pages = _cache_geometry(g, lens, page)
        st.update(_cache(g, pages, page, h, d, case["fmt"]))
        cu = torch.tensor([0] + lens, dtype=torch.int64).cumsum(0)
        if op == "kv_append_read":
            # the last tokens of each sequence are new
            t = case["T"]
            fresh = [min(n, max(1, n * t // total)) for n in lens]
            slots = []
            for i, (n, f) in enumerate(zip(lens, fresh)):
                pos = torch.arange(n - f, n)
                slots.append(table[i].long()[pos // page] * page + pos % page)
            st["slots"] = torch.cat(slots).to(DEV)
            st["k"], st["v"] = _new_kv(g, len(st["slots"]), h, d, case["dtype"])
        st["table"], st["cu"] = table.to(DEV), cu.to(torch.int32).to(DEV)
    return st


# ------------------------------------------------------------------------------------- the plain forms

def _round_f8(y, kind):
    """y (64 bits) to the nearest value of the 8-bit type, ties to even, as that type."""
    bits, low = F8_BITS[kind]
    _, e = torch.frexp(y)
    step = torch.ldexp(torch.ones_like(y), (e - 1).clamp(min=low) - bits)
    r = (torch.round(y / step) * step).clamp(-F8_MAX[kind], F8_MAX[kind])
    return r.float().to(F8[kind])


def _pad_to(x, rows, cols):
    out = x.new_zeros(rows, cols)
    out[:x.shape[0], :x.shape[1]] = x
    return out


def _plain_quant(x, block, kind):
    m, k = x.shape
    kb, mb = (k + 127) // 128, (m + 127) // 128
    # the group maxima in 32 bits, the quotients (values next to a border) in 64; the scale is rounded once to 32
    if block == "row":
        p = _pad_to(x.float(), m, kb * 128).view(m, kb, 128)
        s = (p.abs().amax(-1).double() / F8_MAX[kind]).float().clamp(min=TINY)
        q = p.double() / s.double()[..., None]
    else:
        p = _pad_to(x.float(), mb * 128, kb * 128).view(mb, 128, kb, 128)
        s = (p.abs().amax((1, 3)).double() / F8_MAX[kind]).float().clamp(min=TINY)
        q = p.double() / s.double()[:, None, :, None]
    return _round_f8(q.reshape(-1, kb * 128)[:m, :k], kind), s


def _spread(s, rows, cols, block):
    """Scales of the blocks as one factor for each element."""
    s = s.repeat_interleave(128, 1)[:, :cols]
    return s if block == "row" else s.repeat_interleave(128, 0)[:rows]


def _plain_gemm(a, b, sa, sb, block, out):
    x = a.float() * _spread(sa, a.shape[0], a.shape[1], "row")
    w = b.float() * _spread(sb, b.shape[0], b.shape[1], block)
    return (x @ w.t()).to(out)


def _plain_linear(x, w, dy):
    xq, xs = _plain_quant(x, "row", "e4m3")
    wq, ws = _plain_quant(w, "tile", "e4m3")
    y = _plain_gemm(xq, wq, xs, ws, "tile", x.dtype)
    gq, gs = _plain_quant(dy, "row", "e4m3")
    dx = _plain_gemm(gq, wq.t(), gs, ws.t(), "tile", x.dtype)
    gt, gts = _plain_quant(dy.t(), "row", "e4m3")
    xt, xts = _plain_quant(x.t(), "row", "e4m3")
    return y, dx, _plain_gemm(gt, xt, gts, xts, "row", w.dtype)


E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _plain_mxfp4(x):
    """[..., D] -> packed codes [..., D/2] and exponent codes [..., D/32]; the scale is the smallest power of
    two that is not below the largest magnitude over 6."""
    p = x.float().unflatten(-1, (-1, 32))
    top = p.abs().amax(-1)
    f, e = torch.frexp(top)
    # top / 6 = f * 2^e / 6 with f in [1/2, 1): at most 2^(e - 3) where f <= 3/4, else at most 2^(e - 2)
    e = torch.where(f <= 0.75, e - 3, e - 2).clamp(-127, 127)
    code = torch.where(top > 0, e + 127, 0).to(torch.uint8)
    y = torch.ldexp(p, -torch.where(top > 0, e, 0)[..., None])
    a = y.abs()
    # steps of 1/2 up to 2, of 1 up to 4, of 2 above; ties to even
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = (torch.round(a / step) * step).clamp(max=6.0)
    mag = torch.where(a <= 2, a * 2, torch.where(a <= 4, a + 2, a / 2 + 4)).to(torch.uint8)
    q = (mag | (torch.signbit(y).to(torch.uint8) << 3)).flatten(-2)
    return q[..., 0::2] | (q[..., 1::2] << 4), code


def _plain_write(st, name):
    case = st["case"]
    x, slots = st[name], st["slots"]
    cache, scale = st[name + "_cache"], st[name + "_scale"]
    keep = slots >= 0
    x, slots = x[keep], slots[keep]
    t, h, d = x.shape
    if case["fmt"] == "fp8":
        q, s = _plain_quant(x.reshape(t * h, d), "row", "e4m3")
        cache.view(torch.uint8).view(-1, h, d)[slots] = q.view(torch.uint8).view(t, h, d)
        scale.view(-1, h, scale.shape[-1])[slots] = s.view(t, h, -1)
    else:
        q, s = _plain_mxfp4(x)
        cache.view(-1, h, d // 2)[slots] = q
        scale.view(-1, h, d // 32)[slots] = s


def _rows_of(st):
    """The slot of each row that is read."""
    case, cu = st["case"], st["cu"].long()
    r = torch.arange(case["total"], device=DEV)
    b = torch.searchsorted(cu, r, right=True) - 1
    pos = r - cu[b]
    return st["table"].long()[b, pos // case["page"]] * case["page"] + pos % case["page"]


def _plain_read(st, name):
    case = st["case"]
    h, d = case["H"], case["D"]
    rows = _rows_of(st)
    q = st[name + "_cache"].view(torch.uint8).flatten(0, 1)[rows]
    s = st[name + "_scale"].flatten(0, 1)[rows]
    if case["fmt"] == "fp8":
        x = q.view(torch.float8_e4m3fn).float() * s.repeat_interleave(128, -1)[..., :d]
    else:
        codes = torch.stack([q & 15, q >> 4], -1).flatten(-2).long()
        v = torch.tensor(E2M1, device=DEV)
        x = torch.cat([v, -v])[codes] * torch.ldexp(torch.ones_like(s, dtype=torch.float32), s.int() - 127).repeat_interleave(32, -1)
    return x.view(-1, h, d).to(DT[case["dtype"]])


# ------------------------------------------------------------------------------------- one pass

def run(st):
    case = st["case"]
    op = case["op"]
    if own:
        return _run_own(st, case, op)
    if op == "quant":
        q, s = _plain_quant(st["x"], case["block"], case["fp8"])
        if not case["transposed"]:
            return q, s
        qt, s_t = _plain_quant(st["x"].t(), case["block"], case["fp8"])
        return q, s, qt, s_t
    if op == "gemm":
        return _plain_gemm(st["a"], st["b"], st["sa"], st["sb"], case["block"], DT[case["out"]])
    if op == "linear":
        return _plain_linear(st["x"].detach(), st["w"].detach(), st["dy"])
    if op in ("kv_write", "kv_append_read"):
        _plain_write(st, "k")
        _plain_write(st, "v")
        if op == "kv_write":
            return st["k_cache"], st["k_scale"], st["v_cache"], st["v_scale"]
    return _plain_read(st, "k"), _plain_read(st, "v")


def _run_own(st, case, op):
    from emugen_b200 import fp8, kvcache

    if op == "quant":
        return fp8.quant_fp8(st["x"], block=case["block"], dtype=F8[case["fp8"]], transposed=case["transposed"])
    if op == "gemm":
        return fp8.gemm_fp8(st["a"], st["b"], st["sa"], st["sb"], out_dtype=DT[case["out"]])
    if op == "linear":
        y = fp8.linear_fp8(st["x"], st["w"])
        dx, dw = torch.autograd.grad(y, (st["x"], st["w"]), st["dy"])
        return y, dx, dw
    cache = (st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"])
    if op in ("kv_write", "kv_append_read"):
        kvcache.write_kv_cache(st["k"], st["v"], st["slots"], *cache)
        if op == "kv_write":
            return st["k_cache"], st["k_scale"], st["v_cache"], st["v_scale"]
    return kvcache.read_kv_cache(*cache, st["table"], st["cu"], total=case["total"], dtype=DT[case["dtype"]])


# ------------------------------------------------------------------------------------- work

def work(case):
    op = case["op"]
    if op == "quant":
        m, k = case["M"], case["K"]
        kb, mb = (k + 127) // 128, (m + 127) // 128
        one = m * k + 4 * (m if case["block"] == "row" else mb) * kb
        two = m * k + 4 * (k if case["block"] == "row" else kb) * mb
        return {"bytes": m * k * ESZ[case["dtype"]] + one + (two if case["transposed"] else 0), "flops": 4 * m * k}
    if op == "gemm":
        m, n, k = case["M"], case["N"], case["K"]
        kb = (k + 127) // 128
        return {"bytes": (m + n) * k + m * n * ESZ[case["out"]] + 4 * kb * (m + (n if case["block"] == "row" else (n + 127) // 128)),
                "flops": 2 * m * n * k}
    if op == "linear":
        m, n, k = case["M"], case["N"], case["K"]
        # x, w and dy read once; y, dx and dw written once
        return {"bytes": 2 * ESZ[case["dtype"]] * (m * k + n * k + m * n), "flops": 6 * m * n * k}
    h, d = case["H"], case["D"]
    row = 2 * h * (d + 4 * ((d + 127) // 128) if case["fmt"] == "fp8" else d // 2 + d // 32)
    wide = 2 * h * d * ESZ[case["dtype"]]
    if op == "kv_write":
        return {"bytes": case["T"] * (wide + row + 8), "flops": case["T"] * 2 * h * d * 4}
    total, b = case["total"], case["B"]
    table = 4 * (total // case["page"] + 2 * b)
    w = {"bytes": total * (wide + row) + table, "flops": total * 2 * h * d}
    if op == "kv_append_read":
        w["bytes"] += case["T"] * (wide + row + 8)
        w["flops"] += case["T"] * 2 * h * d * 4
    return w


# ------------------------------------------------------------------------------------- in 64 bits

def _grid(kind):
    """The type's non-negative values in order: the value's place is its code."""
    bits, low = F8_BITS[kind]
    v = [i * 2.0 ** (low - bits) for i in range(2 ** bits)]
    e = low
    while v[-1] < F8_MAX[kind]:
        v += [(1 + i * 2.0 ** -bits) * 2.0 ** e for i in range(2 ** bits)]
        e += 1
    v = [x for x in v if x <= F8_MAX[kind]]
    return torch.tensor(v, dtype=torch.float64, device=DEV)


def _nearest(y, grid):
    """The grid's value nearest to y; halfway, the one with the even code."""
    mid = (grid[1:] + grid[:-1]) / 2
    a = y.abs().contiguous()
    lo = torch.searchsorted(mid, a)                   # values below or at the border
    hi = torch.searchsorted(mid, a, right=True)       # values at the border go up
    code = torch.where(lo % 2 == 0, lo, hi)
    return torch.copysign(grid[code], y)


def _exact_quant(x, block, kind):
    """Blocks one column of blocks at a time."""
    m, k = x.shape
    x = x.double()
    grid = _grid(kind)
    values, scales = [], []
    for c in range(0, k, 128):
        part = x[:, c:c + 128]
        top = part.abs().max(1).values
        if block == "tile":
            top = torch.stack([t.max() for t in top.split(128)])
        s = torch.clamp((top / F8_MAX[kind]).to(torch.float32).double(), min=TINY)
        scales.append(s)
        each = s if block == "row" else s.repeat_interleave(128)[:m]
        values.append(_nearest(part / each[:, None], grid))
    return torch.cat(values, 1), torch.stack(scales, 1)


def _exact_product(a, sa, b, sb, out=None):
    """Sum over the blocks of K of scale times scale times the block's product."""
    m, n, k = a.shape[0], b.shape[0], a.shape[1]
    acc = torch.zeros(m, n, dtype=torch.float64, device=DEV)
    rows_b = torch.arange(n, device=DEV)
    if sb.shape[0] != n:
        rows_b = rows_b // 128
    for i, c in enumerate(range(0, k, 128)):
        left = a[:, c:c + 128].double() * sa[:, i:i + 1].double()
        right = b[:, c:c + 128].double() * sb[rows_b, i:i + 1].double()
        acc.addmm_(left, right.t())
    return acc


def _exact_mx(x):
    """(values, exponent codes) of groups of 32."""
    grid = torch.tensor(E2M1, dtype=torch.float64, device=DEV)
    g = x.double().unflatten(-1, (-1, 32))
    top = g.abs().max(-1).values
    e = torch.ceil(torch.log2(torch.where(top > 0, top, 1.0) / 6 * (1 - 1e-12))).clamp(-127, 127)
    scale = torch.pow(2.0, e)
    y = torch.where(top[..., None] > 0, g / scale[..., None], g)
    return _nearest(y, grid) * scale[..., None], torch.where(top > 0, e + 127, 0)


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "quant":
        out = _exact_quant(st["x"], case["block"], case["fp8"])
        return out + _exact_quant(st["x"].t(), case["block"], case["fp8"]) if case["transposed"] else out
    if op == "gemm":
        return _exact_product(st["a"], st["sa"], st["b"], st["sb"])
    if op == "linear":
        x, w, dy = st["x"].detach(), st["w"].detach(), st["dy"]
        (xq, xs), (wq, ws), (gq, gs) = _exact_quant(x, "row", "e4m3"), _exact_quant(w, "tile", "e4m3"), _exact_quant(dy, "row", "e4m3")
        (gt, gts), (xt, xts) = _exact_quant(dy.t(), "row", "e4m3"), _exact_quant(x.t(), "row", "e4m3")
        return (_exact_product(xq, xs, wq, ws), _exact_product(gq, gs, wq.t(), ws.t()), _exact_product(gt, gts, xt, xts))
    h, d, page = case["H"], case["D"], case["page"]
    done = {}
    for name in ("k", "v"):
        cache, scale = st[name + "_cache"], st[name + "_scale"]
        if case["fmt"] == "fp8":
            q = cache.float().double().view(-1, h, d)
            s = scale.double().view(-1, h, scale.shape[-1]).clone()
        else:
            byte = cache.view(-1, h, d // 2).int()
            code = torch.stack([byte % 16, byte // 16], -1).flatten(-2)
            grid = torch.tensor(E2M1, dtype=torch.float64, device=DEV)
            s = torch.pow(2.0, scale.view(-1, h, d // 32).double() - 127)
            q = torch.where(code >= 8, -1.0, 1.0) * grid[code % 8]
            q, s = (q.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2), None
        if op != "kv_read":
            live = st["slots"] >= 0
            x, at = st[name][live], st["slots"][live]
            if case["fmt"] == "fp8":
                qn, sn = _exact_quant(x.reshape(-1, d), "row", "e4m3")
                q[at], s[at] = qn.view(-1, h, d), sn.view(-1, h, sn.shape[-1])
            else:
                q[at] = _exact_mx(x)[0].flatten(-2)
        done[name] = (q, s)
    if op == "kv_write":
        return tuple(t.view(*st[n].shape) for n, t in zip(("k_cache", "k_scale", "v_cache", "v_scale"), done["k"] + done["v"]))
    rows = []
    table, cu = st["table"].tolist(), st["cu"].tolist()
    for b in range(len(cu) - 1):
        n = cu[b + 1] - cu[b]
        pos = torch.arange(n)
        rows.append(torch.tensor(table[b])[pos // page].long() * page + pos % page)
    rows = torch.cat(rows).to(DEV)
    out = []
    for name in ("k", "v"):
        q, s = done[name]
        x = q[rows]
        if s is not None:
            x = x * s[rows].repeat_interleave(128, -1)[..., :d]
        out.append(x)
    return tuple(out)
