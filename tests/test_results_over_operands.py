"""Results in memory that the same call reads are refused on the host, whatever the types of the two are."""

import pytest
import torch

import test_logit_rules
from tinyvllm_b200.ops import kernels


def over(other, like):
    """``like``'s shape and type in memory that begins with the last four bytes of ``other`` (which moves there)."""
    size = other.numel() * other.element_size()
    memory = torch.zeros(size + like.numel() * like.element_size() + 64, dtype=torch.uint8)
    moved = memory[:size].view(other.dtype).view(other.shape).copy_(other)
    start = size - 4
    return moved, memory[start:start + like.numel() * like.element_size()].view(like.dtype).view(like.shape)


@pytest.mark.parametrize("name", ["slots", "penalties", "lengths", "history", "bias_tokens", "bias_values", "masks", "mask_rows"])
def test_rules(name):
    arguments = test_logit_rules.good()
    arguments[name], out = over(arguments[name], arguments["logits"])
    for logits in (arguments["logits"], out):              # elsewhere, and in place
        with pytest.raises(kernels.KernelError, match="memory of its own"):
            test_logit_rules.call(dict(arguments, logits=logits, out=out))


@pytest.mark.parametrize("written, read", [("history", "tokens"), ("history", "slots"), ("lengths", "tokens"), ("lengths", "slots"),
                                           ("history", "lengths")])
def test_appended_tokens(written, read):
    arguments = dict(tokens=torch.zeros(2, dtype=torch.int32), slots=torch.zeros(2, dtype=torch.int32),
                     lengths=torch.zeros(3, 2, dtype=torch.int32), history=torch.zeros(3, 5, dtype=torch.int32))
    arguments[read], arguments[written] = over(arguments[read], arguments[written])
    with pytest.raises(kernels.KernelError, match="memory of their own"):
        kernels.append_tokens(arguments.pop("tokens"), **arguments)


@pytest.mark.parametrize("name", ["x", "weight", "down", "up", "ids", "scales"])
def test_adapters(name):
    import test_adapters as adapters

    arguments = adapters.good()
    arguments[name], out = over(arguments[name], torch.zeros(3, 24, dtype=torch.bfloat16))
    with pytest.raises(kernels.KernelError, match="memory of its own"):
        adapters.linear_adapted(**arguments, out=out)


@pytest.mark.parametrize("name", ["q", "key_cache", "value_cache", "block_tables", "token_row", "positions", "group_starts", "shared_lens"])
def test_attention_over_keys_in_common(name):
    import test_attention_shared as shared

    arguments = shared.good()
    arguments[name], out = over(arguments[name], torch.zeros(3, 256, dtype=torch.bfloat16))
    with pytest.raises(kernels.KernelError, match="memory of its own"):
        shared.call(arguments | dict(out=out))
