"""Attention's entry points without a GPU: every refusal is made on the host before any CUDA call."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwd

from emugen_b200 import _lib, attention, kvcache

P = 256   # a 256-byte aligned address that no call below gets to read


def _args(cls, base, kw):
    names = [f[0] for f in cls._fields_]
    return cls(**{n: kw.pop(n, base.get(n, 0)) for n in names})


def _norm_rope(back=False, **kw):
    base = dict(q=P, k=P, q_token_stride=256, q_head_stride=128, k_token_stride=256, k_head_stride=128, q_weight=P, k_weight=P, cos=P,
                sin=P, positions=P, tokens=3, table_rows=10, heads_q=2, heads_k=2, head_size=128, half=64, dtype=1, eps=1e-6)
    args = _args(_lib.EmuNormRopeArgs, base, kw)
    L = _lib.load()
    if back:
        a = dict(gq=P, gk=P, s0=256, s1=128, s2=256, s3=128, dq=P, dk=P, dqw=P, dkw=P, work=P, size=L.emu_qk_norm_rope_workspace_size(128))
        a.update(kw)
        st = L.emu_qk_norm_rope_backward(ctypes.byref(args), *a.values(), None)
    else:
        a = dict(qo=P, ko=P)
        a.update(kw)
        st = L.emu_qk_norm_rope(ctypes.byref(args), *a.values(), None)
    return st, L.emu_last_error().decode()


@pytest.mark.parametrize("kw,status,msg", [
    (dict(tokens=-1), 1, "negative size"), (dict(dtype=3), 1, "dtype"), (dict(heads_q=0), 8, "heads"), (dict(heads_k=0), 8, "heads"),
    (dict(head_size=12), 8, "multiple of 8"), (dict(head_size=264), 8, "up to 256"), (dict(half=65), 1, "half"), (dict(half=12), 1, "half"),
    (dict(q=None), 1, "NULL"), (dict(k=None), 1, "NULL"), (dict(positions=None), 1, "NULL"), (dict(cos=None), 1, "NULL"), (dict(qo=None), 1, "NULL"),
    (dict(q=P + 1), 1, "aligned"), (dict(q_weight=P + 1), 1, "aligned"), (dict(positions=P + 4), 1, "aligned"), (dict(ko=P + 8), 1, "16-byte"),
    (dict(eps=-1.0), 1, "eps"),
])
def test_norm_rope_refusals(kw, status, msg):
    st, got = _norm_rope(**kw)
    assert st == status and msg in got


@pytest.mark.parametrize("kw,msg", [
    (dict(tokens=-1), "negative size"), (dict(gq=None), "NULL"), (dict(dk=None), "NULL"), (dict(work=None), "NULL"), (dict(gk=P + 1), "aligned"),
    (dict(dq=P + 8), "16-byte"), (dict(dqw=P + 1), "aligned"), (dict(work=P + 4), "16-byte"), (dict(size=8), "workspace needs"),
])
def test_norm_rope_backward_refusals(kw, msg):
    st, got = _norm_rope(back=True, **kw)
    assert st == 1 and msg in got


def _attention(back=False, **kw):
    base = dict(q=P, k=P, v=P, q_token_stride=512, q_head_stride=128, k_token_stride=256, k_head_stride=128, v_token_stride=256,
                v_head_stride=128, cu_q=P, cu_k=P, total_q=5, total_k=7, sequences=2, heads_q=4, heads_k=2, head_size=128, dtype=1,
                causal=1, scale=0.1)
    args = _args(_lib.EmuAttentionArgs, base, kw)
    L = _lib.load()
    if back:
        a = dict(out=P, low=P, lse=P, do=P, s0=512, s1=128, dq=P, dk=P, dv=P, work=P,
                 size=L.emu_attention_backward_workspace_size(ctypes.byref(args)))
        a.update(kw)
        st = L.emu_attention_backward(ctypes.byref(args), *a.values(), None)
    else:
        a = dict(out=P, low=P, lse=P)
        a.update(kw)
        st = L.emu_attention(ctypes.byref(args), *a.values(), None)
    return st, L.emu_last_error().decode()


ATTENTION = [
    (dict(total_q=-1), 1, "negative size"), (dict(sequences=-1), 1, "negative size"), (dict(dtype=2), 1, "dtype"), (dict(heads_k=0), 8, "heads"),
    (dict(heads_q=65536, heads_k=1), 8, "heads"), (dict(heads_k=3), 1, "multiple of heads_k"), (dict(head_size=4), 8, "multiple of 8"),
    (dict(head_size=136), 8, "up to 128"), (dict(scale=0.0), 1, "scale"), (dict(scale=-1.0), 1, "scale"), (dict(scale=float("inf")), 1, "scale"),
    (dict(scale=float("nan")), 1, "scale"), (dict(total_k=1 << 31), 8, "rows"), (dict(sequences=1 << 40), 8, "sequences"),
    (dict(cu_q=None), 1, "cu_q"), (dict(cu_k=P + 2), 1, "4-byte"), (dict(q=None), 1, "NULL"), (dict(v=None), 1, "NULL"), (dict(k=P + 8), 1, "16-byte"),
    (dict(q_token_stride=130), 1, "multiples of 8"), (dict(k_head_stride=0), 1, "multiples of 8"), (dict(v_token_stride=1 << 40), 1, "strides"),
    (dict(out=None), 1, "NULL"), (dict(low=P + 8), 1, "16-byte"), (dict(lse=P + 2), 1, "4-byte"),
]


@pytest.mark.parametrize("kw,status,msg", ATTENTION)
@pytest.mark.parametrize("back", [False, True])
def test_attention_refusals(kw, status, msg, back):
    st, got = _attention(back, **dict(kw))
    assert st == status and msg in got


@pytest.mark.parametrize("kw,msg", [
    (dict(do=None), "NULL"), (dict(lse=None), "NULL"), (dict(work=None), "NULL"), (dict(do=P + 8), "16-byte"), (dict(work=P + 16), "256-byte"),
    (dict(dq=P + 8), "16-byte"), (dict(dv=P + 2), "16-byte"), (dict(s0=12), "multiples of 8"), (dict(s1=0), "multiples of 8"), (dict(size=256), "workspace needs"),
])
def test_attention_backward_refusals(kw, msg):
    st, got = _attention(True, **kw)
    assert st == 1 and msg in got


def _attend(**kw):
    L = _lib.load()
    a = dict(q=P, s0=512, s1=128, dtype=1, B=3, Hq=4, H=2, D=128, scale=0.1, fmt=0, kc=P, vc=P, ks=P, vs=P, pages=4, page=8, table=P, cols=2,
             ts=2, lens=P, out=P, lse=P, work=P, size=L.emu_kv_attend_workspace_size(3, 4, 2, 128))
    a.update(kw)
    st = L.emu_kv_attend(*a.values(), None)
    return st, L.emu_last_error().decode()


@pytest.mark.parametrize("kw,status,msg", [
    (dict(B=-1), 1, "negative size"), (dict(pages=-1), 1, "negative size"), (dict(page=0), 1, "page_size"), (dict(dtype=2), 1, "dtype"),
    (dict(fmt=2), 1, "cache format"), (dict(D=40), 3, "multiple of 16"), (dict(fmt=1, D=48), 3, "multiple of 32"), (dict(D=272), 8, "256"),
    (dict(Hq=3), 1, "multiple"), (dict(Hq=0), 1, "multiple"), (dict(scale=0.0), 1, "scale"), (dict(scale=float("nan")), 1, "scale"),
    (dict(B=1 << 40), 8, "2^31"), (dict(pages=1 << 45), 8, "slots"), (dict(q=None), 1, "NULL"), (dict(lens=None), 1, "NULL"), (dict(table=None), 1, "NULL"),
    (dict(vc=None), 1, "NULL"), (dict(ks=None), 1, "NULL"), (dict(ts=1), 1, "table_stride"), (dict(q=P + 1), 1, "aligned"), (dict(out=P + 8), 1, "16-byte"),
    (dict(lens=P + 2), 1, "aligned"), (dict(kc=P + 8), 1, "16-byte"), (dict(vs=P + 2), 1, "4-byte"), (dict(size=0), 1, "workspace needs"),
    (dict(work=P + 16), 1, "256-byte"),
])
def test_attend_refusals(kw, status, msg):
    st, got = _attend(**kw)
    assert st == status and msg in got


def test_empty_calls_succeed_without_pointers():
    assert _norm_rope(tokens=0, q=None, k=None, qo=None, ko=None)[0] == 0
    assert _attention(total_q=0, q=None, out=None)[0] == 0
    assert _attention(True, total_q=0, total_k=0, q=None, k=None, v=None, out=None)[0] == 0
    assert _attend(B=0, q=None, lens=None, out=None)[0] == 0


def _pair(T=3, Hq=4, Hk=2, D=64, dtype=torch.bfloat16):
    return torch.zeros(T, Hq, D, dtype=dtype), torch.zeros(T, Hk, D, dtype=dtype)


def test_python_norm_rope_refusals():
    q, k = _pair()
    w, c, p = torch.ones(64, dtype=q.dtype), torch.zeros(9, 32), torch.zeros(3, dtype=torch.int64)
    for args, kw, msg in [((q[0], k, w, w, c, c, p), {}, "tokens, heads"), ((q, k[:2], w, w, c, c, p), {}, "same tokens"),
                          ((q, k.half(), w, w, c, c, p), {}, "share one"), ((q[..., :60], k[..., :60], None, None, c, c, p), {}, "multiple of 8"),
                          ((q[:, :0], k, w, w, c, c, p), {}, "heads"), ((q, k, w.float(), w, c, c, p), {}, "q_weight"), ((q, k, w, w[:8], c, c, p), {}, "k_weight"),
                          ((q, k, w, w, c.double(), c, p), {}, "float32"), ((q, k, w, w, c, c[:, :16], p), {}, "float32"),
                          ((q, k, w, w, c[:, :20], c[:, :20], p), {}, "half"), ((q, k, w, w, torch.zeros(9, 33), torch.zeros(9, 33), p), dict(interleaved=True), "half"),
                          ((q, k, w, w, c, c, p.int()), {}, "positions"), ((q, k, w, w, c, c, p[:2]), {}, "positions"),
                          ((q, k, w, w, c.clone().requires_grad_(), c, p), {}, "no gradient"), ((q, k, w, w, c, c, p), {}, "CUDA")]:
        with pytest.raises(RuntimeError, match=msg):
            attention.qk_norm_rope(*args, **kw)
    with pytest.raises(ValueError, match="eps"):
        attention.qk_norm_rope(q, k, w, w, c, c, p, eps=-1.0)


def test_python_attention_refusals():
    q, k = _pair()
    cu = torch.tensor([0, 3], dtype=torch.int32)
    for args, msg in [((q[0], k, k, cu), "must be"), ((q, k, k[:, :1], cu), "must be"), ((q, k, k.half(), cu), "share one"),
                      ((q.float(), k.float(), k.float(), cu), "share one"), ((*(t[..., :12] for t in (q, k, k)), cu), "multiple of 8"),
                      ((q[:, :3], k, k, cu), "multiple of key heads"), ((q[:2], k, k, cu), "cu_k is needed"), ((q, k, k, cu.long()), "cu_q"),
                      ((q, k, k, cu[None]), "cu_q"), ((q, k, k, cu, torch.tensor([0, 1, 3], dtype=torch.int32)), "cu_k"), ((q, k, k, cu), "CUDA")]:
        with pytest.raises(RuntimeError, match=msg):
            attention.packed_attention(*args)
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="scale"):
            attention.packed_attention(q, k, k, cu, scale=scale)


def test_python_attend_refusals():
    cache = kvcache.make_kv_cache(2, 4, 2, 64, device="cpu")
    q, table, lens = torch.zeros(3, 4, 64, dtype=torch.float16), torch.zeros(3, 1, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="keys and values"):
        kvcache.attend_kv_cache(q, cache[0], None, cache[2], None, table, lens)
    with pytest.raises(RuntimeError, match="CUDA"):
        kvcache.attend_kv_cache(q, *cache, table, lens)


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("no_grad", [False, True])
def test_a_tangent_is_refused(which, no_grad):
    ops = list(_pair(dtype=torch.float16))
    cu, c, p = torch.tensor([0, 3], dtype=torch.int32), torch.zeros(9, 32), torch.zeros(3, dtype=torch.int64)
    with fwd.dual_level():
        ops[which] = fwd.make_dual(ops[which], torch.ones_like(ops[which]))
        with torch.set_grad_enabled(not no_grad):
            with pytest.raises(RuntimeError, match="forward-mode"):
                attention.packed_attention(ops[0], ops[1], ops[1], cu)
            with pytest.raises(RuntimeError, match="forward-mode"):
                attention.qk_norm_rope(*ops, None, None, c, c, p)
        # without a tangent the calls go on to their other checks
        with pytest.raises(RuntimeError, match="CUDA"):
            attention.packed_attention(*(t.clone() for t in (*_pair(), _pair()[1])), cu)
