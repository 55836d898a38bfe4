"""Two kernels whose waits run out before one status call: both records are taken, so that the next status call
speaks for later calls alone.  No GPU fault: the ready signals are withheld through the test hook and the waits are short."""
import pytest
import torch

from emugen_b200 import _lib, fp8
from tests.test_gpu_failure import _case, _gemm
from tests.test_gpu_fp8 import E4, _operands

pytestmark = pytest.mark.gpu


def test_one_status_call_takes_every_kernel_s_record():
    case = _case()
    ops = [t.cuda() for t in _operands(8, 256, 512, E4, E4, False, 6, True)]
    want = fp8.gemm_fp8(*ops, out_dtype=torch.float32)
    _lib.device_status()
    prev = _lib.set_wait_limit(1 << 20)
    _lib.load().emu_test_hold_first_ready(1)
    try:
        _gemm(*case)
        fp8.gemm_fp8(*ops, out_dtype=torch.float32)
    finally:
        _lib.load().emu_test_hold_first_ready(0)
        _lib.set_wait_limit(prev)
    with pytest.raises(_lib.EmuError) as err:
        _lib.device_status()
    assert err.value.status == _lib.EMU_ERR_TIMEOUT
    _lib.device_status()                                   # nothing left from before
    assert torch.equal(fp8.gemm_fp8(*ops, out_dtype=torch.float32), want)
    _lib.device_status()
