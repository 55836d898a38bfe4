"""The registered 8-bit operators give the tracer the device that they answer on: the quantiser's codes and scales are on
the GPU whatever x is on, the product's output is on the CPU only where every operand is."""
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import emugen_b200.ops  # noqa: F401


def test_fake_outputs_are_on_the_device_of_the_real_ones():
    with FakeTensorMode():
        for dev in ("cpu", "cuda"):
            for block in ("row", "tile"):
                q, s = torch.ops.emugen.quant_fp8(torch.empty(7, 200, dtype=torch.bfloat16, device=dev), block)
                assert q.device.type == s.device.type == "cuda"
        a, sa = torch.empty(7, 200, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.empty(7, 2)
        assert torch.ops.emugen.gemm_fp8(a, a, sa, sa).device.type == "cpu"
        assert torch.ops.emugen.gemm_fp8(a, a, sa, sa.cuda()).device.type == "cuda"
