"""Calls of the attention over keys in common that have to be refused on the host: what a kernel would read out of line."""

import pytest
import torch

from test_attention_shared import BF16, call, good
from tinyvllm_b200.ops import kernels


@pytest.mark.parametrize("page", [1, 4, 8, 16, 48, 256])
@pytest.mark.parametrize("name", ["key_cache", "value_cache"])
@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("offset", [1, 2, 8])
def test_caches_off_the_16_bytes(offset, dtype, name, page):
    """Contiguous views in the middle of a buffer: the kernels read 16 bytes at a time, tensor maps start on 16."""
    arguments = good(dtype=dtype)
    for cache in ("key_cache", "value_cache"):
        arguments[cache] = torch.zeros(5, 2, page, 64, dtype=dtype)
    buffer = torch.zeros(5 * 2 * page * 64 + 8, dtype=dtype)
    assert buffer.data_ptr() % 16 == 0
    arguments[name] = buffer[offset:offset + 5 * 2 * page * 64].view(5, 2, page, 64)
    assert arguments[name].is_contiguous()
    aligned = offset * buffer.element_size() % 16 == 0
    with pytest.raises(kernels.KernelError, match="CUDA tensors only" if aligned else "16 bytes"):
        call(arguments)


@pytest.mark.parametrize("scale", [1e-46, 1e-39, 2.4e38, 3.4e38, 1e39, 1e300])
def test_scales_that_float32_does_not_have(scale):
    """1e-46 would be 0 (times -inf for a masked score: NaN), 2.4e38 infinite times log2(e), 1e39 infinite."""
    with pytest.raises(kernels.KernelError, match="scale"):
        call(good() | dict(scale=scale))


@pytest.mark.parametrize("scale", [2.0**-126, 1e-30, 1.0, 2.0**127])
def test_scales_that_it_has(scale):
    with pytest.raises(kernels.KernelError, match="CUDA tensors only"):
        call(good() | dict(scale=scale))


@pytest.mark.parametrize("name", ["q", "key_cache", "value_cache", "out"])
def test_operands_that_want_gradients(name):
    arguments = good() | dict(out=torch.zeros(3, 256, dtype=BF16))
    arguments[name].requires_grad_(True)
    with pytest.raises(kernels.KernelError, match="backward"):
        call(arguments)
    with torch.no_grad(), pytest.raises(kernels.KernelError, match="CUDA tensors only"):
        call(arguments)
