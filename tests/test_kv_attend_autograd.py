"""attend_kv_cache has no gradient: what asks for one is refused, not answered without it."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from emugen_b200 import kvcache


def _inputs(device, fmt="fp8"):
    cache = kvcache.make_kv_cache(2, 16, 2, 64, fmt, device=device)
    q = torch.zeros(3, 4, 64, dtype=torch.float16, device=device)
    return q, cache, torch.zeros(3, 1, dtype=torch.int32, device=device), torch.ones(3, dtype=torch.int32, device=device)


@pytest.mark.parametrize("which", ["q", "k_scale", "v_scale"])
def test_what_wants_a_gradient_is_refused(which):
    q, cache, table, lens = _inputs("cpu")
    {"q": q, "k_scale": cache[2], "v_scale": cache[3]}[which].requires_grad_()
    with pytest.raises(RuntimeError, match="not differentiable"):
        kvcache.attend_kv_cache(q, *cache, table, lens)
    # without gradients the call goes on to its other checks
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
        kvcache.attend_kv_cache(q, *cache, table, lens)


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
@pytest.mark.parametrize("no_grad", [False, True])
def test_a_tangent_is_refused(fmt, no_grad):
    q, cache, table, lens = _inputs("cpu", fmt)
    with fwd.dual_level(), torch.set_grad_enabled(not no_grad):
        with pytest.raises(RuntimeError, match="forward-mode"):
            kvcache.attend_kv_cache(fwd.make_dual(q, torch.ones_like(q)), *cache, table, lens)
        with pytest.raises(RuntimeError, match="CUDA"):
            kvcache.attend_kv_cache(q, *cache, table, lens)


@pytest.mark.gpu
def test_without_gradients_it_is_as_before():
    import emugen_b200.ops  # noqa: F401

    q, cache, table, lens = _inputs("cuda")
    q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(1)))
    k = torch.randn(1, 2, 64, generator=torch.Generator().manual_seed(2)).half().cuda()
    kvcache.write_kv_cache(k, k, torch.zeros(1, dtype=torch.int64, device="cuda"), *cache)
    want = kvcache.attend_kv_cache(q, *cache, table, lens)
    assert want.any()
    q.requires_grad_()
    with torch.no_grad():
        assert torch.equal(kvcache.attend_kv_cache(q, *cache, table, lens), want)
    assert torch.equal(kvcache.attend_kv_cache(q.detach(), *cache, table, lens), want)
    # the registered operator answers, and refuses the backward pass
    out = torch.ops.emugen.attend_kv_cache(q, *cache, table, lens)
    assert torch.equal(out, want)
    if out.requires_grad:
        with pytest.raises(RuntimeError):
            out.float().sum().backward()
