"""Refusals of the attention over keys in common, before anything is launched."""

import pytest
import torch

from tinyvllm_b200.ops import kernels

BF16, I32 = torch.bfloat16, torch.int32


def good(tokens=3, num_q=4, num_kv=2, head_dim=64, dtype=BF16):
    return dict(q=torch.zeros(tokens, num_q * head_dim, dtype=dtype), q_token_stride=num_q * head_dim,
                key_cache=torch.zeros(5, num_kv, 16, head_dim, dtype=dtype), value_cache=torch.zeros(5, num_kv, 16, head_dim, dtype=dtype),
                block_tables=torch.zeros(3, 2, dtype=I32), token_row=torch.zeros(tokens, dtype=I32),
                positions=torch.zeros(tokens, dtype=I32), group_starts=torch.zeros(2, dtype=I32), shared_lens=torch.zeros(1, dtype=I32),
                num_q=num_q, num_kv=num_kv, head_dim=head_dim, scale=0.125)


def call(arguments):
    return kernels.attention_shared(**arguments)


@pytest.mark.parametrize("changed", [{}, dict(max_shared=16, max_own=0), dict(out=torch.zeros(3, 256, dtype=BF16)), good(tokens=0),
                                     good(dtype=torch.float32), good(head_dim=128), good(head_dim=256, num_q=2),
                                     dict(group_starts=torch.zeros(1, dtype=I32), shared_lens=torch.zeros(0, dtype=I32))])
def test_a_good_call_gets_as_far_as_the_device(changed):
    with pytest.raises(kernels.KernelError, match="CUDA tensors only"):
        call(good() | changed)


@pytest.mark.parametrize("changed", [
    good(head_dim=32), good(head_dim=96), good(num_q=3), dict(num_kv=0), good(dtype=torch.float16),
    dict(key_cache=torch.zeros(5, 2, 16, 64)), dict(key_cache=torch.zeros(5, 16, 2, 64, dtype=BF16)),
    dict(value_cache=torch.zeros(4, 2, 16, 64, dtype=BF16)), dict(value_cache=torch.zeros(5, 2, 16, 64)),
    dict(key_cache=torch.zeros(5, 16, 2, 64, dtype=BF16).transpose(1, 2)), dict(positions=torch.zeros(3)),
    dict(positions=torch.zeros(1, 3, dtype=I32)), dict(token_row=torch.zeros(2, dtype=I32)), dict(token_row=torch.zeros(3, dtype=torch.int64)),
    dict(block_tables=torch.zeros(6, dtype=I32)), dict(block_tables=torch.zeros(3, 2)), dict(block_tables=torch.zeros(2, 3, dtype=I32).t()),
    dict(group_starts=torch.zeros(3, dtype=I32)), dict(shared_lens=torch.zeros(1)), dict(shared_lens=torch.zeros(1, 1, dtype=I32)),
    dict(q_token_stride=128), dict(q_token_stride=260), dict(q_token_stride=264), dict(q=torch.zeros(3, 512, dtype=BF16)[:, ::2]),
    dict(q=torch.zeros(3 * 256 + 8, dtype=BF16)[1:769].view(3, 256)), dict(max_shared=-1), dict(max_own=-1), dict(max_shared=2**31), dict(max_own=2**31), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
    dict(out=torch.zeros(3, 256)), dict(out=torch.zeros(3, 255, dtype=BF16)), dict(out=torch.zeros(256, 3, dtype=BF16).t()),
    dict(out=torch.zeros(1, 256, dtype=BF16).expand(3, 256)),
])
def test_refusals(changed):
    with pytest.raises(kernels.KernelError) as refusal:
        call(good() | changed)
    assert "CUDA tensors only" not in str(refusal.value)


@pytest.mark.parametrize("of", ["q", "key_cache", "value_cache"])
def test_a_result_in_memory_that_is_read(of):
    arguments = good()
    memory = arguments[of].view(-1)
    with pytest.raises(kernels.KernelError, match="memory of its own"):
        call(arguments | dict(out=memory[: 3 * 256].view(3, 256)))
