"""linear_fp8 has no forward-mode derivative: a dual input is refused, never answered without its tangent.  (The
refusal comes before the device is looked at, so it shows without a GPU.)"""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from emugen_b200 import fp8


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("no_grad", [False, True])
def test_a_tangent_is_refused(which, no_grad):
    ops = [torch.ones(3, 128), torch.ones(5, 128)]
    with fwd.dual_level():
        ops[which] = fwd.make_dual(ops[which], torch.ones_like(ops[which]))
        with torch.set_grad_enabled(not no_grad), pytest.raises(RuntimeError, match="forward-mode"):
            fp8.linear_fp8(*ops)
        # without a tangent the call goes on to its other checks
        with pytest.raises(RuntimeError, match="CUDA"):
            fp8.linear_fp8(torch.ones(3, 128), torch.ones(5, 128))
