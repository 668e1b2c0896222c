"""Rules on logits on the host: parameters, mask words, refusals of the kernel's face (checked before anything is launched)."""

import pytest
import torch

from tinyvllm_b200 import SamplingParams
from tinyvllm_b200.ops import kernels
from tinyvllm_b200.sampling import LogitRules, Sampler
from tinyvllm_b200.sampling.rules import pack_mask


def test_parameters_without_rules_are_as_before():
    params = SamplingParams(temperature=0.5)
    assert not params.has_rules
    assert (params.repetition_penalty, params.presence_penalty, params.frequency_penalty) == (1.0, 0.0, 0.0)
    assert params.logit_bias == () and params.allowed_token_ids is None


@pytest.mark.parametrize("rule", [dict(repetition_penalty=1.2), dict(presence_penalty=-0.5), dict(frequency_penalty=1),
                                  dict(logit_bias={3: -1.5}), dict(logit_bias=[(3, 1), (3, 2.0)]), dict(allowed_token_ids=[0])])
def test_each_rule_counts(rule):
    assert SamplingParams(**rule).has_rules
    hash(SamplingParams(**rule))


@pytest.mark.parametrize("rule", [dict(repetition_penalty=0.0), dict(repetition_penalty=-1.0), dict(repetition_penalty=float("inf")),
                                  dict(presence_penalty=float("nan")), dict(frequency_penalty=float("inf")),
                                  dict(logit_bias=[(-1, 0.5)]), dict(logit_bias=[(1, float("inf"))]), dict(logit_bias=[(1.0, 0.5)]),
                                  dict(logit_bias=[(1, 2, 3)]), dict(logit_bias={i: 1.0 for i in range(1025)}),
                                  dict(allowed_token_ids=[]), dict(allowed_token_ids=[-1]), dict(allowed_token_ids=[1.5])])
def test_bad_rules_are_refused(rule):
    with pytest.raises(ValueError):
        SamplingParams(**rule)


@pytest.mark.parametrize("rule", [dict(repetition_penalty=1e300), dict(repetition_penalty=1e-300), dict(presence_penalty=-1e39),
                                  dict(frequency_penalty=10**400), dict(logit_bias={1: 3.5e38})])
def test_numbers_that_float32_does_not_have_are_refused(rule):
    with pytest.raises(ValueError, match="float32"):
        SamplingParams(**rule)


@pytest.mark.parametrize("rule", [dict(repetition_penalty="1"), dict(presence_penalty=None), dict(frequency_penalty=True)])
def test_rules_of_another_type_are_refused(rule):
    with pytest.raises(TypeError):
        SamplingParams(**rule)


@pytest.mark.parametrize("vocab", [1, 31, 32, 33, 97])
def test_mask_words(vocab):
    allowed = sorted({0, vocab // 2, vocab - 1})
    words = pack_mask(allowed, vocab)
    assert words.dtype == torch.int32 and words.shape == (-(-vocab // 32),)
    assert [v for v in range(vocab) if int(words[v // 32]) >> (v % 32) & 1] == allowed


def test_slots_keep_rules_and_tokens():
    rules = LogitRules(vocab=50, slots=3, room=6, device="cpu")
    rules.set(1, SamplingParams(repetition_penalty=1.5, logit_bias=[(7, 2.0)], allowed_token_ids=[7, 9]), [1, 2, 3], [4])
    rules.set(2, SamplingParams(presence_penalty=0.5), list(range(10)))          # more than there is room for
    assert rules.lengths.tolist() == [[0, 0], [4, 3], [6, 6]]
    assert rules.history[1, :4].tolist() == [1, 2, 3, 4] and rules.history[2].tolist() == [0, 1, 2, 3, 4, 5]
    assert rules.bias_tokens[1, 0].item() == 7 and (rules.bias_tokens[2] == -1).all()
    assert rules.mask_rows.tolist() == [-1, 1, -1]
    rules.set(1, SamplingParams(logit_bias={i: float(i) for i in range(40)}), [5])    # wider rows, no mask any more
    assert rules.bias_tokens[1, :40].tolist() == list(range(40)) and (rules.bias_tokens[1, 40:] == -1).all()
    assert rules.mask_rows.tolist() == [-1, -1, -1] and rules.lengths[1].tolist() == [1, 1]
    for bad in (dict(logit_bias=[(50, 1.0)]), dict(allowed_token_ids=[50])):
        with pytest.raises(ValueError, match="vocabulary"):
            rules.set(0, SamplingParams(**bad), [1])
    with pytest.raises(ValueError, match="slots"):
        rules.set(3, SamplingParams(), [1])


def good(rows=2, vocab=70, slots=3, room=5, biases=4):
    return dict(logits=torch.zeros(rows, vocab), slots=torch.zeros(rows, dtype=torch.int32), penalties=torch.ones(slots, 3),
                lengths=torch.zeros(slots, 2, dtype=torch.int32), history=torch.zeros(slots, room, dtype=torch.int32),
                bias_tokens=torch.zeros(slots, biases, dtype=torch.int32), bias_values=torch.zeros(slots, biases),
                masks=torch.zeros(2, 3, dtype=torch.int32), mask_rows=torch.zeros(slots, dtype=torch.int32))


def call(arguments):
    arguments = dict(arguments)
    return kernels.logit_rules(arguments.pop("logits"), **arguments)


def test_a_good_call_gets_as_far_as_the_device():
    with pytest.raises(kernels.KernelError, match="CUDA tensors only"):
        call(good())
    with pytest.raises(kernels.KernelError, match="CUDA tensors only"):
        call(dict(good(), out=torch.zeros(2, 70)))
    arguments = good()
    with pytest.raises(kernels.KernelError, match="CUDA tensors only"):
        call(dict(arguments, out=arguments["logits"]))


@pytest.mark.parametrize("name, value", [
    ("logits", torch.zeros(70)), ("logits", torch.zeros(70, 2).t()), ("logits", torch.zeros(2, 70, dtype=torch.float16)),
    ("slots", torch.zeros(2)), ("slots", torch.zeros(3, dtype=torch.int32)), ("slots", torch.zeros(4, dtype=torch.int32)[::2]),
    ("penalties", torch.ones(3, 2)), ("penalties", torch.ones(3, 3, dtype=torch.float64)), ("lengths", torch.zeros(3, 2)),
    ("lengths", torch.zeros(2, 2, dtype=torch.int32)), ("history", torch.zeros(3, 5, dtype=torch.int64)),
    ("history", torch.zeros(15, dtype=torch.int32)), ("history", torch.zeros(5, 3, dtype=torch.int32).t()),
    ("bias_values", None), ("bias_tokens", None), ("bias_values", torch.zeros(3, 5)),
    ("bias_tokens", torch.zeros(3, 4, dtype=torch.int64)), ("masks", None), ("mask_rows", None),
    ("masks", torch.zeros(2, 2, dtype=torch.int32)), ("masks", torch.zeros(2, 3, dtype=torch.bool)),
    ("mask_rows", torch.zeros(2, dtype=torch.int32)), ("out", torch.zeros(2, 71)), ("out", torch.zeros(2, 70, dtype=torch.bfloat16)),
    ("out", torch.zeros(1, 70).expand(2, 70)),
])
def test_refusals(name, value):
    with pytest.raises(kernels.KernelError) as refusal:
        call(dict(good(), **{name: value}))
    assert "CUDA tensors only" not in str(refusal.value)


def test_too_many_biases_and_shifted_results_are_refused():
    arguments = good(biases=1025)
    with pytest.raises(kernels.KernelError, match="1024"):
        call(arguments)
    memory = torch.zeros(3, 70)
    with pytest.raises(kernels.KernelError, match="memory of its own"):
        call(dict(good(), logits=memory[:2], out=memory[1:]))


def test_append_refusals():
    def append(**changed):
        arguments = dict(tokens=torch.zeros(2, dtype=torch.int32), slots=torch.zeros(2, dtype=torch.int32),
                         lengths=torch.zeros(3, 2, dtype=torch.int32), history=torch.zeros(3, 5, dtype=torch.int32)) | changed
        return kernels.append_tokens(arguments.pop("tokens"), **arguments)

    with pytest.raises(kernels.KernelError, match="CUDA tensors only"):
        append()
    many = torch.zeros(kernels.APPEND_MAX_ROWS + 1, dtype=torch.int32)
    for changed in (dict(tokens=torch.zeros(2)), dict(tokens=torch.zeros(3, dtype=torch.int32)), dict(tokens=many, slots=many),
                    dict(lengths=torch.zeros(2, 2, dtype=torch.int32)), dict(history=torch.zeros(3, 5))):
        with pytest.raises(kernels.KernelError) as refusal:
            append(**changed)
        assert "CUDA tensors only" not in str(refusal.value)


def test_the_sampler_wants_a_slot_a_row():
    rules = LogitRules(vocab=8, slots=1, room=4, device="cpu")
    with pytest.raises(ValueError, match="slots"):
        Sampler().sample(torch.zeros(2, 8), [SamplingParams()] * 2, [0, 0], rules=rules, slots=[0])
    with pytest.raises(ValueError, match="8 tokens"):
        rules.apply(torch.zeros(2, 9), torch.zeros(2, dtype=torch.int32))
