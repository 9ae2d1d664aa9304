"""Operands of attention over shared prefixes whose address its kernels cannot read 16 bytes at a time."""

from __future__ import annotations

import pytest
import torch
from test_attention_shared_gpu import DEV, Step, _call

from rapid_llm_b200.ops import kernels

pytestmark = pytest.mark.gpu


def moved(tensor):
    """The same numbers one element further: contiguous, and off the boundary."""
    room = torch.empty(tensor.numel() + 16 // tensor.element_size(), dtype=tensor.dtype, device=DEV)
    there = room[1 : 1 + tensor.numel()].view(tensor.shape)
    there.copy_(tensor)
    assert there.is_contiguous() and there.data_ptr() % 16
    return there


@pytest.mark.parametrize("dtype,dim", [(torch.float32, 64), (torch.bfloat16, 64), (torch.bfloat16, 128)])
@pytest.mark.parametrize("name", ["q", "cache", "part_out"])
def test_operands_off_the_boundary(dtype, dim, name):
    step = Step([64], [(0, 3, 1), (0, 5, 1), (0, 1, 1)], heads=8, kv_heads=2, dim=dim, page=16, dtype=dtype)
    with pytest.raises(kernels.KernelError, match="16-byte aligned"):
        _call(step, **{name: lambda a: moved(a[name])})
