"""Caps that are no 32-bit numbers, or whose double or reciprocal is none, are refused before anything reaches a device."""
import pytest
import torch

from kungfu_b200 import ops
from kungfu_b200.ops import KernelError


@pytest.mark.parametrize("cap", [1e39, 3e38, 1e-46, 1e-40, -1e-46])
def test_caps_out_of_range(cap):
    z = torch.zeros
    with pytest.raises(KernelError, match="softcap"):
        ops.head_logprobs(z(4, 8), z(20, 8), z(4, dtype=torch.int32), z(4), softcap=cap)
    with pytest.raises(KernelError, match="CUDA"):             # the ends of the range get as far as the device
        ops.head_logprobs(z(4, 8), z(20, 8), z(4, dtype=torch.int32), z(4), softcap=2.0 ** -126 if cap < 1 else 2.0 ** 126)
