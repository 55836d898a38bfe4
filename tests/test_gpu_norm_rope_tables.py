"""Norms with rotation where the table's rows do not start on 16 bytes, or the tensors' do not: how they are read changes no bit."""
import pytest
import torch

from emugen_b200 import attention
from tests.test_gpu_norm_rope import _check, _make, _table

pytestmark = pytest.mark.gpu


def _off(t):
    """t in memory that starts one element past a 16-byte boundary."""
    return torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape).copy_(t)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D,half,interleaved", [(96, 18, True), (96, 30, True), (64, 1, True), (40, 7, True), (128, 64, True), (64, 32, False), (256, 8, False)])
@pytest.mark.parametrize("T", [1, 333])
def test_rows_and_table_are_read_each_for_itself(dtype, D, half, interleaved, T):
    q, k, wq, wk, pos, gq, gk = _make(T, 6, 2, D, dtype, D + half)
    cos, sin = _table(500, half)
    _check(q, k, wq, wk, cos, sin, pos, gq, gk, interleaved)

    def run(q, k, wq, wk, cos, sin, gq, gk):
        x = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
        y = attention.qk_norm_rope(*x, cos, sin, pos, interleaved=interleaved)
        return (*y, *torch.autograd.grad(y, x, (gq, gk)))

    want = run(q, k, wq, wk, cos, sin, gq, gk)
    for i in range(8):
        args = [q, k, wq, wk, cos, sin, gq, gk]
        args[i] = _off(args[i])
        assert all(torch.equal(a, b) for a, b in zip(run(*args), want)), i
