"""Refusals of the projection with adapters, before anything is launched."""

import pytest
import torch

from tinyvllm_b200.ops import kernels, linear_adapted


def good(m=3, k=16, n=24, adapters=2, rank=4, dtype=torch.bfloat16):
    return dict(x=torch.zeros(m, k, dtype=dtype), weight=torch.zeros(n, k, dtype=dtype), down=torch.zeros(adapters, rank, k, dtype=dtype),
                up=torch.zeros(adapters, n, rank, dtype=dtype), ids=torch.zeros(m, dtype=torch.int32), scales=torch.ones(adapters))


@pytest.mark.parametrize("changed", [{}, dict(scales=None), dict(out_dtype=torch.float32), dict(out=torch.zeros(3, 24)),
                                     dict(out=torch.zeros(3, 24, dtype=torch.bfloat16)), good(m=0), good(dtype=torch.float32)])
def test_a_good_call_gets_as_far_as_the_device(changed):
    with pytest.raises(kernels.KernelError, match="CUDA tensors only"):
        linear_adapted(**(good() | changed))


BF16 = torch.bfloat16


@pytest.mark.parametrize("changed", [
    dict(x=torch.zeros(3, 17, dtype=BF16)), dict(x=torch.zeros(16, dtype=BF16)), dict(x=torch.zeros(3, 16)),
    dict(x=torch.zeros(16, 3, dtype=BF16).t()), dict(weight=torch.zeros(24, 16)), good(dtype=torch.float16), good(k=0),
    dict(down=torch.zeros(2, 4, 16)), dict(down=torch.zeros(2, 4, 15, dtype=BF16)), dict(down=torch.zeros(4, 16, dtype=BF16)),
    dict(down=torch.zeros(2, 16, 4, dtype=BF16).transpose(1, 2)), dict(up=torch.zeros(2, 24, 5, dtype=BF16)),
    dict(up=torch.zeros(3, 24, 4, dtype=BF16)), dict(up=torch.zeros(2, 4, 24, dtype=BF16).transpose(1, 2)), good(adapters=0),
    good(rank=0), good(rank=257), dict(ids=torch.zeros(3)), dict(ids=torch.zeros(2, dtype=torch.int32)),
    dict(ids=torch.zeros(6, dtype=torch.int32)[::2]), dict(scales=torch.ones(3)), dict(scales=torch.ones(2, dtype=BF16)),
    dict(out_dtype=torch.float16), dict(out=torch.zeros(3, 25, dtype=BF16)), dict(out=torch.zeros(3, 24, dtype=torch.float64)),
    dict(out=torch.zeros(24, 3, dtype=BF16).t()), dict(out=torch.zeros(3, 24), out_dtype=BF16),
    dict(out=torch.zeros(1, 24, dtype=BF16).expand(3, 24)),
])
def test_refusals(changed):
    with pytest.raises(kernels.KernelError) as refusal:
        linear_adapted(**(good() | changed))
    assert "CUDA tensors only" not in str(refusal.value)


@pytest.mark.parametrize("name", ["x", "weight", "down", "up", "scales"])
def test_operands_that_want_gradients_are_refused(name):
    arguments = good()
    arguments[name].requires_grad_(True)
    with pytest.raises(kernels.KernelError, match="backward"):
        linear_adapted(**arguments)
    with torch.no_grad(), pytest.raises(kernels.KernelError, match="CUDA tensors only"):
        linear_adapted(**arguments)


def test_a_result_over_an_operand_is_refused():
    arguments = good(n=16)
    for name in ("x", "weight"):
        with pytest.raises(kernels.KernelError, match="memory of its own"):
            linear_adapted(**arguments, out=arguments[name][:3])
