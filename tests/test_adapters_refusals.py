"""What the adapters' kernels do not take is refused before the projection runs."""

import pytest
import torch

from test_adapters import good
from tinyvllm_b200.ops import kernels, linear_adapted


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_more_rows_than_the_kernels_take(dtype):
    most = kernels.ADAPTERS_MAX_ROWS
    for m, reason in ((most, "CUDA tensors only"), (most + 1, f"up to {most} rows")):
        arguments = good(dtype=dtype) | dict(x=torch.zeros(1, 16, dtype=dtype).expand(m, 16), ids=torch.zeros(m, dtype=torch.int32))
        with pytest.raises(kernels.KernelError, match=reason):
            linear_adapted(**arguments)
