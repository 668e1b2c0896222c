"""Rules on logits whose gradients are wanted are refused: the kernel has no backward pass."""

import pytest
import torch

from test_logit_rules import call, good
from tinyvllm_b200 import SamplingParams
from tinyvllm_b200.ops import kernels
from tinyvllm_b200.sampling import LogitRules, Sampler


@pytest.mark.parametrize("name", ["logits", "penalties", "bias_values", "out"])
def test_operands_that_want_gradients(name):
    arguments = good() | dict(out=torch.zeros(2, 70))
    arguments[name].requires_grad_(True)
    with pytest.raises(kernels.KernelError, match="backward"):
        call(arguments)
    with torch.no_grad(), pytest.raises(kernels.KernelError, match="CUDA tensors only"):
        call(arguments)


def test_the_rules_of_slots_refuse_them_too():
    rules = LogitRules(vocab=8, slots=1, room=4, device="cpu")
    logits = torch.zeros(1, 8, requires_grad=True)
    with pytest.raises(kernels.KernelError, match="backward"):
        rules.apply(logits, torch.zeros(1, dtype=torch.int32))
    with pytest.raises(kernels.KernelError, match="backward"):
        Sampler().sample(logits, [SamplingParams()], [0], rules=rules, slots=[0])


def test_whether_there_are_rules_follows_a_changed_copy():
    import copy
    import dataclasses
    import pickle

    bare = SamplingParams(temperature=0.5)
    ruled = dataclasses.replace(bare, frequency_penalty=0.5)
    assert not bare.has_rules and ruled.has_rules and not dataclasses.replace(ruled, frequency_penalty=0.0).has_rules
    for again in (copy.copy(ruled), copy.deepcopy(ruled), pickle.loads(pickle.dumps(ruled))):
        assert again == ruled and again.has_rules
