"""Attention and its neighbours in 64 bits, each result with the largest error that its roundings allow.

With u = half a step of the tensors' 16-bit type and f = 2^-23 for each f32 operation of a chain:
  scores      |error| <= f (D + 4) scale sum |q_d k_d|                  (a D-term sum, the scale, log2 e)
  p           relative: twice the row's largest score error (numerator and sum) + u (its rounding) + f * 64
  ds          p (dp - delta) relative as p, + u; dp and delta as sums of D terms, delta of the output before its rounding (with a rest of it that was
              rounded in its turn: u^2, or half a subnormal step)
Sums over n terms add f n times the sum of magnitudes.  16-bit results: u relative, and half a subnormal step."""
import math

import torch

F = 2.0 ** -23
# A weight exp(s) below f32's smallest normal number, 2^-126, is made 0 (and bf16 has the same smallest one): with the
# rounding at that border, a weight may be off by 2^-125 whatever its size.
LOWEST = 2.0 ** -125


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the smallest subnormal step."""
    return {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[dtype]


def attention(q, k, v, cu_q, cu_k, causal, scale, do=None, p_step=None, v_low=None):
    """{name: (value, tolerance)} for out, lse and, with do, dq, dk, dv; a head and a sequence at a time.  Hidden keys and
    values are left out of the sums altogether.  p_step: half a step of the type that the weights are rounded to; v_low
    (v's shape): the error of one key's share of the output where its weight is below that type's normal numbers."""
    dev = q.device
    u, D = half_step(q.dtype), q.shape[2]
    pu = u if p_step is None else p_step
    low = tiny(q.dtype)
    Hq, Hk = q.shape[1], k.shape[1]
    z = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=dev)
    out, out_t = z(q), z(q)
    lse = torch.full((Hq, q.shape[0]), -math.inf, dtype=torch.float64, device=dev)
    lse_t = torch.zeros_like(lse)
    dq, dq_t, dk, dk_t, dv, dv_t = z(q), z(q), z(k), z(k), z(k), z(k)
    Q, K, V = q.detach().double(), k.detach().double(), v.detach().double()
    for s in range(len(cu_q) - 1):
        i0, i1, j0, j1 = cu_q[s], cu_q[s + 1], cu_k[s], cu_k[s + 1]
        nq, nk = i1 - i0, j1 - j0
        if not nq or not nk:
            continue
        seen = torch.ones(nq, nk, dtype=torch.bool, device=dev)
        if causal:
            seen = torch.arange(nk, device=dev)[None] <= torch.arange(nq, device=dev)[:, None] + nk - nq
        some = seen.any(1)
        n = nk + 64
        for h in range(Hq):
            g = h * Hk // Hq
            a, b, c = Q[i0:i1, h], K[j0:j1, g], V[j0:j1, g]
            x = a @ b.t() * scale
            x_err = (F * (D + 4) * scale * (a.abs() @ b.abs().t()))
            x = torch.where(seen, x, -math.inf)
            x_err = torch.where(seen, x_err, 0.0)
            m = torch.where(some, x.amax(1), 0.0)
            e = torch.exp(x - m[:, None])
            total = torch.where(some, e.sum(1), 1.0)
            p = e / total[:, None]
            rel = 2 * x_err.amax(1, keepdim=True) + F * 64 + F * 4 * (x - m[:, None]).abs().nan_to_num(0, 0, 0).clamp(max=200)
            lse[h, i0:i1] = torch.where(some, m + torch.log(total), -math.inf)
            lse_t[h, i0:i1] = torch.where(some, x_err.amax(1) + F * 32 + F * 8 * lse[h, i0:i1].abs().nan_to_num(0, 0, 0), 0.0)
            # rows of values that only hidden queries meet may hold anything: they enter as zeros beside p = 0
            used = seen.any(0)
            c0 = torch.where(used[:, None], c, 0.0)
            o = p @ c0
            p_err = p * (rel + pu) + ((2.0 ** -31 if q.dtype == torch.float16 else 0.0) + LOWEST) * seen
            o_t = (p_err + F * n * p) @ c0.abs() + u * o.abs() + low
            if v_low is not None:
                o_t = o_t + seen.double() @ v_low[j0:j1, g]
            out[i0:i1, h], out_t[i0:i1, h] = o, o_t
            if do is None:
                continue
            w = do[i0:i1, h].double()
            # the same on the queries' side: rows that see no key may hold anything
            w = torch.where(some[:, None], w, 0.0)
            a0, b0 = torch.where(some[:, None], a, 0.0), torch.where(used[:, None], b, 0.0)
            b_err = rel + 2 * lse_t[h, i0:i1, None] + F * 4 * lse[h, i0:i1, None].abs().nan_to_num(0, 0, 0)
            dv[j0:j1, g] += p.t() @ w
            dv_t[j0:j1, g] += (p * (b_err + u + F * (nq + 64)) + LOWEST * seen).t() @ w.abs()
            dp = w @ c0.t()
            delta = (w * o).sum(1, keepdim=True)
            dp_err = F * (D + 4) * (w.abs() @ c0.abs().t()) + F * (D + 4) * (w * o).abs().sum(1, keepdim=True) + (w.abs() * (o_t - u * o.abs() + u * u * o.abs())).sum(1, keepdim=True)
            ds = p * (dp - delta)
            # (fp16: held to 2^-24 of a bound on |dp - delta| times 2^-15)
            bound = 2 * w.norm(dim=1).amax() * c0.norm(dim=1).amax()
            ds_err = ds.abs() * (b_err + u) + p * dp_err + LOWEST * (1 + (dp - delta).abs()) * seen + (bound * 2.0 ** -36 if q.dtype == torch.float16 else 0.0) * seen
            dq[i0:i1, h] = ds @ b0 * scale
            dq_t[i0:i1, h] = (ds_err + F * n * ds.abs()) @ b0.abs() * scale
            dk[j0:j1, g] += ds.t() @ a0 * scale
            dk_t[j0:j1, g] += (ds_err + F * (nq * Hq // Hk + 64) * ds.abs()).t() @ a0.abs() * scale
    r = {"out": (out, out_t), "lse": (lse, lse_t)}
    if do is not None:
        r["dq"], r["dk"], r["dv"] = ((x, t + u * x.abs() + low) for x, t in ((dq, dq_t), (dk, dk_t), (dv, dv_t)))
    return r


def check(got, want, name=""):
    value, tol = want
    got = got.detach().double()
    assert got.shape == value.shape, name
    same = (got == value) | (got.isnan() & value.isnan())
    bad = ~same & ~((got - value).abs() <= tol)
    if bad.any():
        i = tuple(int(x) for x in bad.nonzero()[0])
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} off, first at {i}: {float(got[i])} for {float(value[i])}, "
                             f"tolerance {float(tol[i])}")


def norm_rope(x, w, cos, sin, pos, eps, interleaved, dy=None):
    """(y, tolerance) and, with dy, also (dx, tolerance), (dw, tolerance)."""
    u, low = half_step(x.dtype), tiny(x.dtype)
    D, half = x.shape[2], cos.shape[1]
    X = x.detach().double()
    W = torch.ones(D, dtype=torch.float64, device=x.device) if w is None else w.detach().double()
    inv = 1 / torch.sqrt((X * X).mean(-1, keepdim=True) + eps)
    n = X * inv
    c = torch.ones(x.shape[0], 1, D, dtype=torch.float64, device=x.device)
    s = torch.zeros_like(c)
    other = torch.arange(D, device=x.device)
    i = torch.arange(half, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    at = pos.clamp(min=0)
    known = (at < cos.shape[0])[:, None]
    C = torch.where(known, cos.double()[at.clamp(max=cos.shape[0] - 1)], math.nan) if half else cos.double()[:0]
    S = torch.where(known, sin.double()[at.clamp(max=cos.shape[0] - 1)], math.nan) if half else C
    if half:
        c[:, 0, a], c[:, 0, b], s[:, 0, a], s[:, 0, b] = C, C, -S, S
        other[a], other[b] = b, a
    pad = (pos < 0)[:, None, None]
    z = n * W
    y = torch.where(pad, 0.0, z * c + z[..., other] * s)
    # about D / 8 + 40 f32 roundings in the mean, the root and the products
    f = F * (D / 8 + 40)
    y_t = f * ((z * c).abs() + (z[..., other] * s).abs()) + u * y.abs() + low
    if dy is None:
        return y, y_t.nan_to_num(0)
    G = dy.double()
    dz = G * c - G[..., other] * s
    dz_m = (G * c).abs() + (G[..., other] * s).abs()
    g = dz * W
    mean = (g * n).mean(-1, keepdim=True)
    dx = torch.where(pad, 0.0, inv * (g - n * mean))
    dx_t = f * inv * (dz_m * W.abs() + n.abs() * (dz_m * W.abs() * n.abs()).mean(-1, keepdim=True)) + u * dx.abs() + low
    live = ~pad
    dw = torch.where(live, dz * n, 0.0).sum((0, 1))
    rows = x.shape[0] * x.shape[1]
    dw_t = (f + F * (rows ** 0.5 + 300)) * torch.where(live, dz_m * n.abs(), 0.0).sum((0, 1)) + u * dw.abs() + low
    return y, y_t.nan_to_num(0), dx, dx_t.nan_to_num(0), dw, dw_t.nan_to_num(0)
