"""Rules that are part of a recorded step: the graph has the addresses of what they keep, so nothing of it may be replaced."""

import pytest
import torch

from tinyvllm_b200 import SamplingParams
from tinyvllm_b200.ops import kernels
from tinyvllm_b200.sampling import LogitRules

KEPT = ("penalties", "lengths", "history", "bias_tokens", "bias_values", "masks", "mask_rows")


@pytest.fixture
def recording(monkeypatch):
    """``apply`` with the kernel left out, inside a capture."""
    monkeypatch.setattr(kernels, "logit_rules", lambda logits, **rest: logits)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    return lambda rules: rules.apply(torch.zeros(1, rules.vocab), torch.zeros(1, dtype=torch.int32))


def addresses(rules):
    return [None if t is None else t.data_ptr() for t in (getattr(rules, name) for name in KEPT)]


def test_room_made_at_once(recording):
    rules = LogitRules(vocab=50, slots=3, room=6, device="cpu", biases=40, masks=True)
    assert rules.bias_tokens.shape == (3, 40) and (rules.bias_tokens == -1).all() and rules.mask_rows.tolist() == [-1] * 3
    before = addresses(rules)
    recording(rules)
    rules.set(0, SamplingParams(logit_bias={i: 1.0 for i in range(40)}, allowed_token_ids=[1, 2]), [1])
    rules.set(1, SamplingParams(repetition_penalty=2.0), [1, 2])
    assert addresses(rules) == before
    with pytest.raises(ValueError, match="recorded.*40 biases"):
        rules.set(2, SamplingParams(logit_bias={i: 1.0 for i in range(41)}), [1])
    assert addresses(rules) == before and rules.lengths[2].tolist() == [0, 0]          # a refused request changes nothing


@pytest.mark.parametrize("rule", [dict(logit_bias={1: 1.0}), dict(allowed_token_ids=[1])])
def test_a_request_that_needs_more_than_was_recorded_is_refused(recording, rule):
    rules = LogitRules(vocab=50, slots=2, room=6, device="cpu")
    rules.set(0, SamplingParams(presence_penalty=1.0), [1])
    recording(rules)
    before = addresses(rules)
    with pytest.raises(ValueError, match="recorded"):
        rules.set(1, SamplingParams(**rule), [1])
    assert addresses(rules) == before
    rules.set(1, SamplingParams(frequency_penalty=1.0), [3, 4])
    assert addresses(rules) == before


def test_rules_that_no_graph_has_still_grow():
    rules = LogitRules(vocab=50, slots=2, room=6, device="cpu")
    for count in (1, 33, 50):
        rules.set(1, SamplingParams(logit_bias={i: 1.0 for i in range(count)}), [1])
        assert rules.bias_tokens[1, :count].tolist() == list(range(count))


@pytest.mark.parametrize("biases", [-1, kernels.LOGIT_RULES_MAX_BIASES + 1])
def test_room_for_biases_has_the_kernels_limit(biases):
    with pytest.raises(ValueError, match="biases"):
        LogitRules(vocab=50, slots=2, room=6, device="cpu", biases=biases)


@pytest.mark.gpu
def test_a_recorded_step_sees_what_later_requests_bring():
    from rules_helpers import check_rules

    device = "cuda"
    rules = LogitRules(vocab=700, slots=2, room=8, device=device, biases=4, masks=True)
    logits = torch.randn(2, 700, generator=torch.Generator().manual_seed(3)).to(device)
    slots = torch.tensor([1, 0], dtype=torch.int32, device=device)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        rules.apply(logits, slots)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = rules.apply(logits, slots)
    torch.cuda.synchronize()
    rules.set(1, SamplingParams(logit_bias={3: 2.0, 699: -1.0}, repetition_penalty=1.5), [4, 5], [6])
    rules.set(0, SamplingParams(allowed_token_ids=[7, 8, 699]), [9])
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    check_rules(out, logits, slots=slots, **{name: getattr(rules, name) for name in KEPT})
    assert torch.isfinite(out[1]).nonzero()[:, 0].tolist() == [7, 8, 699] and out[0, 3] == logits[0, 3] + 2.0
    with pytest.raises(ValueError, match="recorded"):
        rules.set(0, SamplingParams(logit_bias={i: 1.0 for i in range(5)}), [1])
