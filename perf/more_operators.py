"""Cases for the attention operators: the norms of queries and keys with the position rotation, attention over
packed prompts with its gradients, and attention of one new token over the quantised key/value cache.

``run`` computes a case in plain torch operations, or -- where ``own`` is set -- through the framework's
entry points.  ``exact`` restates every operator in 64 bits, written apart from the plain form.
"""
import math
import random

import torch

own = False

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
ESZ = {"bf16": 2, "f16": 2, "f32": 4}
TABLE = 32768            # positions of the rotation's table
MOST_PAIRS = 4 * 10 ** 9  # (query, key, head) triples of the largest case


def listed():
    return [
        # a decode step of 32 sequences: latency
        {"name": "norm_rope_32", "op": "norm_rope", "T": 32, "Hq": 32, "Hk": 8, "D": 128, "R": 128, "dtype": "bf16",
         "interleaved": False, "train": False},
        # a long prompt's queries and keys on their way to the attention
        {"name": "norm_rope_16384", "op": "norm_rope", "T": 16384, "Hq": 32, "Hk": 8, "D": 128, "R": 128, "dtype": "bf16",
         "interleaved": False, "train": False},
        # a training batch of odd size, pairs side by side and half of each head rotated: forward and backward
        {"name": "norm_rope_train_8191", "op": "norm_rope", "T": 8191, "Hq": 24, "Hk": 6, "D": 96, "R": 48, "dtype": "f16",
         "interleaved": True, "train": True},
        # a handful of short prompts packed together: latency
        {"name": "attention_333", "op": "attention", "Tq": 333, "Tk": 333, "B": 7, "Hq": 8, "Hk": 2, "D": 128, "dtype": "f16",
         "causal": True, "train": False},
        # one long prompt: bound by the tensor cores
        {"name": "attention_16384", "op": "attention", "Tq": 16384, "Tk": 16384, "B": 1, "Hq": 32, "Hk": 8, "D": 128,
         "dtype": "bf16", "causal": True, "train": False},
        # further pieces of prompts against their cached beginnings, odd lengths, a head size between the tiles'; where a
        # sequence has fewer keys than queries its first rows see none
        {"name": "attention_prefix_2051x20011", "op": "attention", "Tq": 2051, "Tk": 20011, "B": 9, "Hq": 20, "Hk": 4, "D": 80,
         "dtype": "bf16", "causal": True, "train": False},
        # a training step of documents packed into one row: forward and backward
        {"name": "attention_train_8192", "op": "attention", "Tq": 8192, "Tk": 8192, "B": 3, "Hq": 32, "Hk": 8, "D": 128,
         "dtype": "bf16", "causal": True, "train": True},
        # an encoder's batch of short ragged texts, without a mask: forward and backward
        {"name": "attention_train_3001", "op": "attention", "Tq": 3001, "Tk": 3001, "B": 24, "Hq": 12, "Hk": 12, "D": 64,
         "dtype": "f16", "causal": False, "train": True},
        # one user's next token: latency
        {"name": "kv_attend_1x8192", "op": "kv_attend", "B": 1, "total": 8192, "Hq": 32, "Hk": 8, "D": 128, "page": 16,
         "dtype": "bf16", "fmt": "fp8"},
        # a full server's decode step: bound by reading the cache
        {"name": "kv_attend_64x262144", "op": "kv_attend", "B": 64, "total": 262144, "Hq": 32, "Hk": 8, "D": 128, "page": 16,
         "dtype": "bf16", "fmt": "fp8"},
        # a few very long contexts on one key head
        {"name": "kv_attend_4x400001", "op": "kv_attend", "B": 4, "total": 400001, "Hq": 16, "Hk": 1, "D": 128, "page": 64,
         "dtype": "bf16", "fmt": "fp8"},
        # ragged contexts in a 4-bit cache, an odd number of query heads for each key head, pages that end inside tiles
        {"name": "kv_attend_mxfp4_33x100003", "op": "kv_attend", "B": 33, "total": 100003, "Hq": 28, "Hk": 4, "D": 64,
         "page": 48, "dtype": "f16", "fmt": "mxfp4"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_rope", "attention", "attention", "kv_attend", "kv_attend"])
    hk = rng.randint(1, 8)
    group = rng.randint(1, 8)
    if op == "norm_rope":
        d = 8 * rng.randint(4, 32)
        interleaved = rng.random() < 0.5
        most = 16384 * 40 * 128 // ((group + 1) * hk * d)
        train = rng.random() < 0.5
        return {"op": op, "T": _log(rng, 1, max(2, most // (4 if train else 1))), "Hq": group * hk, "Hk": hk, "D": d,
                "R": 2 * rng.randint(1, d // 2) if interleaved else 16 * rng.randint(1, d // 16),
                "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "interleaved": interleaved, "train": train}
    if op == "attention":
        d = 8 * rng.randint(4, 16)
        train = rng.random() < 0.5
        # as if one sequence had it all, and twice as much for the gradients' products
        most = MOST_PAIRS / (3 if train else 1) / (group * hk)
        tq = _log(rng, 1, min(16384, int(math.sqrt(most))))
        tk = tq if rng.random() < 0.6 else _log(rng, 1, min(65536, int(most / tq)))
        return {"op": op, "Tq": tq, "Tk": tk, "B": _log(rng, 1, min(32, tq)), "Hq": group * hk, "Hk": hk, "D": d,
                "dtype": rng.choice(["bf16", "f16"]), "causal": rng.random() < 0.7, "train": train}
    fmt = rng.choice(["fp8", "mxfp4"])
    d = 32 * rng.randint(1, 4) if fmt == "mxfp4" else 16 * rng.randint(2, 8)
    b = _log(rng, 1, 128)
    most = 262144 * 8 * 128 // (hk * d)
    return {"op": op, "B": b, "total": max(b, _log(rng, 16, min(524288, most))), "Hq": group * hk, "Hk": hk, "D": d,
            "page": rng.choice([1, 8, 16, 48, 64, 128]), "dtype": rng.choice(["bf16", "f16"]), "fmt": fmt}


# ------------------------------------------------------------------------------------- inputs

def _lengths(total, parts, salt):
    """total into `parts` uneven lengths, some of them zero where there are many; the same for every seed."""
    r = random.Random(total * 1009 + parts * 31 + salt)
    w = [0.0 if parts > 4 and r.random() < 0.06 else r.random() ** 2 + 0.01 for _ in range(parts)]
    w[0] = max(w[0], 0.3)
    n = [int(total * x / sum(w)) for x in w]
    n[0] += total - sum(n)
    return n


def _sequences(case):
    """(lengths of queries, lengths of keys) of an attention case."""
    q = _lengths(case["Tq"], case["B"], 1)
    return q, (q if case["Tk"] == case["Tq"] else _lengths(case["Tk"], case["B"], 2))


def _cumulative(n):
    return torch.tensor([0] + n, dtype=torch.int64).cumsum(0).to(torch.int32).to(DEV)


def _heads(g, t, h, d, dtype):
    """Rows of heads at about unit scale, channels of uneven size."""
    x = torch.randn(t, h, d, generator=g, device=DEV)
    return (x * torch.exp(torch.randn(1, h, d, generator=g, device=DEV) * 0.3)).to(DT[dtype])


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    op, h, hk, d = case["op"], case["Hq"], case["Hk"], case["D"]
    st = {"case": case}
    if op == "norm_rope":
        t = case["T"]
        qkv = _heads(g, t, h + 2 * hk, d, case["dtype"])         # a fused projection's output
        st["q"], st["k"] = qkv[:, :h], qkv[:, h:h + hk]
        for n in ("wq", "wk"):
            st[n] = (1 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(DT[case["dtype"]])
        angle = torch.arange(TABLE, device=DEV, dtype=torch.float64)[:, None] * torch.pow(
            10000.0, -torch.arange(0, case["R"], 2, device=DEV, dtype=torch.float64) / case["R"])
        st["cos"], st["sin"] = torch.cos(angle).float(), torch.sin(angle).float()
        st["pos"] = torch.randint(0, TABLE, (t,), generator=g, device=DEV)
        if case["train"]:
            for n in ("q", "k", "wq", "wk"):
                st[n] = st[n].detach().requires_grad_()
            st["dq"], st["dk"] = _heads(g, t, h, d, case["dtype"]), _heads(g, t, hk, d, case["dtype"])
    elif op == "attention":
        nq, nk = _sequences(case)
        st["q"] = _heads(g, case["Tq"], h, d, case["dtype"])
        st["k"], st["v"] = (_heads(g, case["Tk"], hk, d, case["dtype"]) for _ in range(2))
        st["nq"], st["nk"] = nq, nk                              # on the host for the plain form alone
        st["cu_q"], st["cu_k"] = _cumulative(nq), _cumulative(nk)
        if case["train"]:
            for n in ("q", "k", "v"):
                st[n].requires_grad_()
            st["do"] = _heads(g, case["Tq"], h, d, case["dtype"])
    else:
        n = _lengths(case["total"], case["B"], 3)
        page, fmt = case["page"], case["fmt"]
        need = [(x + page - 1) // page for x in n]
        pages = sum(need) + 3
        perm = torch.randperm(pages, generator=g, device=DEV).to(torch.int32).cpu()
        table = torch.full((len(n), max(max(need), 1)), -1, dtype=torch.int32)
        at = 0
        for i, x in enumerate(need):
            table[i, :x] = perm[at:at + x]
            at += x
        for name in ("k", "v"):
            if fmt == "fp8":
                x = (torch.randn(pages, page, hk, d, generator=g, device=DEV) * 110).clamp_(-448, 448)
                st[name + "_cache"] = x.to(torch.float8_e4m3fn)
                st[name + "_scale"] = torch.rand(pages, page, hk, (d + 127) // 128, generator=g, device=DEV) * 0.01 + 1e-3
            else:
                st[name + "_cache"] = torch.randint(0, 256, (pages, page, hk, d // 2), generator=g, device=DEV, dtype=torch.uint8)
                st[name + "_scale"] = torch.randint(122, 127, (pages, page, hk, d // 32), generator=g, device=DEV, dtype=torch.uint8)
        st["q"] = _heads(g, case["B"], h, d, case["dtype"])
        st["n"] = n                                              # on the host for the plain form alone
        st["table"], st["lens"] = table.to(DEV), torch.tensor(n, dtype=torch.int32, device=DEV)
    return st


# ------------------------------------------------------------------------------------- the plain forms

def _rotate(x, cos, sin, r, interleaved, back=False):
    """The first r elements of each head turned by their position's angles (back: the other way)."""
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    c, s = cos[:, None], (-sin if back else sin)[:, None]
    y = x.clone()
    if interleaved:
        y[..., 0:r:2], y[..., 1:r:2] = a * c - b * s, b * c + a * s
    else:
        y[..., :r // 2], y[..., r // 2:r] = a * c - b * s, b * c + a * s
    return y


def _plain_norm_rope(x, w, dy, st):
    case = st["case"]
    cos, sin = st["cos"][st["pos"]], st["sin"][st["pos"]]
    f = x.detach().float()
    inv = torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-6)
    wf = w.detach().float()
    y = _rotate(f * inv * wf, cos, sin, case["R"], case["interleaved"]).to(x.dtype)
    if dy is None:
        return y, None, None
    dz = _rotate(dy.float(), cos, sin, case["R"], case["interleaved"], back=True)
    n = f * inv
    gw = dz * wf
    dx = inv * (gw - n * (gw * n).mean(-1, keepdim=True))
    # a long sum: in 64 bits
    return y, dx.to(x.dtype), (dz * n).sum((0, 1), dtype=torch.float64).to(w.dtype)


def _mask(nq, nk, causal):
    """True where a key is seen: the last query stands on the last key."""
    if not causal:
        return torch.ones(nq, nk, dtype=torch.bool, device=DEV)
    return torch.arange(nk, device=DEV)[None] <= torch.arange(nq, device=DEV)[:, None] + (nk - nq)


def _weights(s, seen):
    """Softmax over the keys that are seen; zeros where there are none."""
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    return p / p.sum(-1, keepdim=True).clamp(min=1e-30)


def _plain_attention(st):
    case = st["case"]
    h, hk, d = case["Hq"], case["Hk"], case["D"]
    grp, scale = h // hk, d ** -0.5
    q, k, v = (st[n].detach().float() for n in "qkv")
    out = torch.zeros_like(q)
    train = case["train"]
    if train:
        do = st["do"].float()
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    a = b = 0
    for nq, nk in zip(st["nq"], st["nk"]):
        rq, rk = slice(a, a + nq), slice(b, b + nk)
        a, b = a + nq, b + nk
        if nq == 0 or nk == 0:
            continue
        seen = _mask(nq, nk, case["causal"])
        for j in range(hk):
            hs = slice(j * grp, (j + 1) * grp)
            qs, ks, vs = q[rq, hs].transpose(0, 1), k[rk, j], v[rk, j]
            p = _weights(qs @ ks.t() * scale, seen)
            out[rq, hs] = (p @ vs).transpose(0, 1)
            if train:
                g = do[rq, hs].transpose(0, 1)
                dv[rk, j] = torch.einsum("hij,hid->jd", p, g)
                dp = g @ vs.t()
                ds = p * (dp - (dp * p).sum(-1, keepdim=True))
                dq[rq, hs] = (ds @ ks * scale).transpose(0, 1)
                dk[rk, j] = torch.einsum("hij,hid->jd", ds, qs) * scale
    t = st["q"].dtype
    return (out.to(t), dq.to(t), dk.to(t), dv.to(t)) if train else out.to(t)


E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _plain_rows(st, name, rows):
    """The cached rows at these slots in 32 bits."""
    case = st["case"]
    q = st[name + "_cache"].view(torch.uint8).flatten(0, 1)[rows]
    s = st[name + "_scale"].flatten(0, 1)[rows]
    if case["fmt"] == "fp8":
        return q.view(torch.float8_e4m3fn).float() * s.repeat_interleave(128, -1)[..., :case["D"]]
    codes = torch.stack([q & 15, q >> 4], -1).flatten(-2).long()
    value = torch.tensor(E2M1, device=DEV)
    factor = torch.ldexp(torch.ones_like(s, dtype=torch.float32), s.int() - 127)
    return torch.cat([value, -value])[codes] * factor.repeat_interleave(32, -1)


def _plain_attend(st):
    case = st["case"]
    h, hk, d, page = case["Hq"], case["Hk"], case["D"], case["page"]
    q = st["q"].float().view(-1, hk, h // hk, d)
    out = torch.zeros_like(q)
    for b, n in enumerate(st["n"]):
        if n == 0:
            continue
        pos = torch.arange(n, device=DEV)
        rows = st["table"][b].long()[pos // page] * page + pos % page
        k, v = _plain_rows(st, "k", rows), _plain_rows(st, "v", rows)
        s = q[b] @ k.permute(1, 2, 0) * d ** -0.5
        p = torch.exp(s - s.amax(-1, keepdim=True))
        out[b] = (p / p.sum(-1, keepdim=True)) @ v.transpose(0, 1)
    return out.view(-1, h, d).to(st["q"].dtype)


# ------------------------------------------------------------------------------------- one pass

def run(st):
    case = st["case"]
    op = case["op"]
    if own:
        return _run_own(st, case, op)
    if op == "norm_rope":
        yq, dq, dwq = _plain_norm_rope(st["q"], st["wq"], st.get("dq"), st)
        yk, dk, dwk = _plain_norm_rope(st["k"], st["wk"], st.get("dk"), st)
        return (yq, yk, dq, dk, dwq, dwk) if case["train"] else (yq, yk)
    return _plain_attention(st) if op == "attention" else _plain_attend(st)


def _run_own(st, case, op):
    from emugen_b200 import attention, kvcache

    if op == "norm_rope":
        x = (st["q"], st["k"], st["wq"], st["wk"])
        yq, yk = attention.qk_norm_rope(*x, st["cos"], st["sin"], st["pos"], eps=1e-6, interleaved=case["interleaved"])
        if not case["train"]:
            return yq, yk
        return (yq, yk, *torch.autograd.grad((yq, yk), x, (st["dq"], st["dk"])))
    if op == "attention":
        out = attention.packed_attention(st["q"], st["k"], st["v"], st["cu_q"], st["cu_k"], causal=case["causal"])
        if not case["train"]:
            return out
        return (out, *torch.autograd.grad(out, (st["q"], st["k"], st["v"]), st["do"]))
    return kvcache.attend_kv_cache(st["q"], st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"], st["table"], st["lens"])


# ------------------------------------------------------------------------------------- work

def _pairs(nq, nk, causal):
    """(query, key) pairs that are seen."""
    if not causal:
        return nq * nk
    first = nk - nq + 1                              # keys that the first query sees, were there negative counts
    if first >= 0:
        return nq * (first + nk) // 2
    return nk * (nk + 1) // 2


def work(case):
    op, h, hk, d = case["op"], case["Hq"], case["Hk"], case["D"]
    if op == "norm_rope":
        n, e = case["T"] * (h + hk) * d, ESZ[case["dtype"]]
        table = min(case["T"], TABLE) * case["R"] * 4 + case["T"] * 8
        if case["train"]:
            # forward x to y; backward dy and x to dx
            return {"bytes": 4 * n * e + table + 4 * d * e, "flops": 20 * n}
        return {"bytes": 2 * n * e + table + 2 * d * e, "flops": 7 * n}
    if op == "attention":
        pairs = sum(_pairs(a, b, case["causal"]) for a, b in zip(*_sequences(case)))
        q, kv = case["Tq"] * h * d * 2, case["Tk"] * hk * d * 2
        if case["train"]:
            # q, do, k and v in; out, dq, dk and dv out
            return {"bytes": 4 * q + 4 * kv, "flops": 14 * d * h * pairs}
        return {"bytes": 2 * q + 2 * kv, "flops": 4 * d * h * pairs}
    row = 2 * hk * (d + 4 * ((d + 127) // 128) if case["fmt"] == "fp8" else d // 2 + d // 32)
    return {"bytes": case["total"] * row + 4 * case["B"] * h * d + 4 * (case["total"] // case["page"] + 2 * case["B"]),
            "flops": 4 * d * h * case["total"]}


# ------------------------------------------------------------------------------------- in 64 bits

def _exact_turned(x, w, st):
    """x / rms(x) * w with its pairs as complex numbers times exp(i angle), as a function that torch differentiates."""
    case = st["case"]
    r = case["R"]
    y = x * w / torch.sqrt((x * x).sum(-1, keepdim=True) / case["D"] + 1e-6)
    turn = torch.complex(st["cos"].double(), st["sin"].double())[st["pos"]][:, None, :]
    head, tail = y[..., :r], y[..., r:]
    if case["interleaved"]:
        z = torch.view_as_complex(head.unflatten(-1, (r // 2, 2)).contiguous()) * turn
        return torch.cat([torch.view_as_real(z).flatten(-2), tail], -1)
    z = torch.complex(head[..., :r // 2].contiguous(), head[..., r // 2:].contiguous()) * turn
    return torch.cat([z.real, z.imag, tail], -1)


def _exact_attention(st):
    """Head by head, the queries in blocks; the softmax through its logarithm."""
    case = st["case"]
    h, hk, d = case["Hq"], case["Hk"], case["D"]
    q, k, v = (st[n].detach().double() for n in "qkv")
    train = case["train"]
    out = torch.zeros_like(q)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    cq, ck = st["cu_q"].tolist(), st["cu_k"].tolist()
    for s in range(case["B"]):
        nq, nk = cq[s + 1] - cq[s], ck[s + 1] - ck[s]
        if not nk:
            continue
        for i0 in range(0, nq, 4096):
            i1 = min(nq, i0 + 4096)
            last = torch.arange(i0, i1, device=DEV) + nk - nq if case["causal"] else torch.full((i1 - i0,), nk - 1, device=DEV)
            hidden = torch.arange(nk, device=DEV).expand(i1 - i0, nk) > last[:, None]
            some = (last >= 0).double()[:, None]
            for x in range(h):
                kk, vv = k[ck[s]:ck[s + 1], x * hk // h], v[ck[s]:ck[s + 1], x * hk // h]
                qq = q[cq[s] + i0:cq[s] + i1, x]
                z = torch.where(hidden, -1e300, torch.mm(qq, kk.t()) / math.sqrt(d))
                p = torch.exp(z - torch.logsumexp(z, 1, keepdim=True)) * some
                o = torch.mm(p, vv)
                out[cq[s] + i0:cq[s] + i1, x] = o
                if train:
                    g = st["do"][cq[s] + i0:cq[s] + i1, x].double()
                    dv[ck[s]:ck[s + 1], x * hk // h] += torch.mm(p.t(), g)
                    ds = p * (torch.mm(g, vv.t()) - (g * o).sum(1, keepdim=True)) / math.sqrt(d)
                    dq[cq[s] + i0:cq[s] + i1, x] = torch.mm(ds, kk)
                    dk[ck[s]:ck[s + 1], x * hk // h] += torch.mm(ds.t(), qq)
    return (out, dq, dk, dv) if train else out


def _exact_cache(st, name, at):
    case = st["case"]
    hk, d = case["Hk"], case["D"]
    if case["fmt"] == "fp8":
        x = st[name + "_cache"].view(-1, hk, d)[at].to(torch.float32).double()
        s = st[name + "_scale"].view(-1, hk, (d + 127) // 128)[at].double()
        return x * s[..., torch.arange(d, device=DEV) // 128]
    byte = st[name + "_cache"].view(-1, hk, d // 2)[at].int()
    code = torch.stack([byte % 16, byte // 16], -1).flatten(-2)
    x = torch.where(code >= 8, -1.0, 1.0) * torch.tensor(E2M1, dtype=torch.float64, device=DEV)[code % 8]
    s = torch.pow(2.0, st[name + "_scale"].view(-1, hk, d // 32)[at].double() - 127)
    return x * s[..., torch.arange(d, device=DEV) // 32]


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "norm_rope":
        leaf = [st[n].detach().double().requires_grad_(case["train"]) for n in ("q", "k", "wq", "wk")]
        yq, yk = _exact_turned(leaf[0], leaf[2], st), _exact_turned(leaf[1], leaf[3], st)
        if not case["train"]:
            return yq, yk
        grads = torch.autograd.grad((yq, yk), leaf, (st["dq"].double(), st["dk"].double()))
        return (yq.detach(), yk.detach(), *grads)
    if op == "attention":
        return _exact_attention(st)
    h, hk, d, page = case["Hq"], case["Hk"], case["D"], case["page"]
    out = torch.zeros(case["B"], h, d, dtype=torch.float64, device=DEV)
    table, lens = st["table"].cpu(), st["lens"].tolist()
    for b, n in enumerate(lens):
        if n:
            pages = torch.arange(n) // page
            at = (table[b][pages].long() * page + torch.arange(n) - pages * page).to(DEV)
            k, v = _exact_cache(st, "k", at), _exact_cache(st, "v", at)
            for x in range(h):
                z = torch.mv(k[:, x * hk // h], st["q"][b, x].double()) / math.sqrt(d)
                out[b, x] = torch.mv(v[:, x * hk // h].t(), torch.softmax(z, 0))
    return out
