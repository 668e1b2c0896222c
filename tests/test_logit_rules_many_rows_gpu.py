"""Rules on logits of so many rows, or so large a vocabulary, that a CTA takes the larger slice."""

import pytest
import torch

from rules_helpers import check_rules
from test_logit_rules_gpu import DEV, k, made

pytestmark = pytest.mark.gpu
MANY = 160                                             # more rows than the GPU has SMs: one slice each is enough


def some_masked(rules, rows=6):
    """Masks for a few slots alone (the 64-bit form walks over every token of theirs)."""
    rules["mask_rows"][:] = -1
    rules["mask_rows"][:rows] = torch.arange(rows, dtype=torch.int32, device=DEV) % rules["masks"].shape[0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 3, 8])
@pytest.mark.parametrize("vocab", [1, 4095, 4096, 4097, 4104, 8203])
def test_rules(vocab, offset, dtype):
    logits, rules = made(MANY, vocab, 21, biases=12, masks=3, dtype=dtype, offset=offset, seed=21)
    some_masked(rules)
    # tokens and biases at the ends of the slices
    edges = torch.tensor([e for e in (0, 2047, 2048, 4095, 4096, 8191, 8192, vocab - 1) if e < vocab], dtype=torch.int32, device=DEV)
    rules["history"][:, :len(edges)] = edges
    rules["bias_tokens"][::2, :len(edges)] = edges
    before = logits.clone()
    got = k().logit_rules(logits, **rules)
    assert torch.equal(logits, before)
    check_rules(got, logits, **rules)
    memory = torch.full((MANY, vocab + 16), 7.0, dtype=dtype, device=DEV)
    for at in (8, 5):
        assert torch.equal(k().logit_rules(logits, out=memory[:, at:at + vocab], **rules), got)
        assert (memory[:, :at] == 7).all() and (memory[:, at + vocab:] == 7).all()
        memory.fill_(7.0)
    assert torch.equal(k().logit_rules(logits, out=logits, **rules), got)                        # in place


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_whole_vocabulary(dtype):
    logits, rules = made(5, 151936, 700, biases=300, masks=2, dtype=dtype, seed=22)
    some_masked(rules, rows=1)
    rules["history"][:, ::2] = torch.randint(151936 - 384, 151936, (5, 350), generator=torch.Generator().manual_seed(1)).to(torch.int32)
    rules["bias_tokens"][:, ::3] = torch.randint(151936 - 384, 151936, (5, 100), generator=torch.Generator().manual_seed(2)).to(torch.int32)
    check_rules(k().logit_rules(logits, **rules), logits, **rules)


def test_a_token_named_many_times_and_one_token_again_and_again():
    logits, rules = made(MANY, 4097, 3000, biases=1024, seed=23)
    rules["bias_tokens"][:, ::3] = 17
    rules["bias_tokens"][:, 1::3] = 4096
    rules["history"][::2] = 4096
    got = k().logit_rules(logits, **rules)
    rows = slice(0, 12)
    check_rules(got[rows], logits[rows], **dict(rules, slots=rules["slots"][rows]))
    assert torch.equal(k().logit_rules(logits, **rules), got)


def test_rows_without_a_slot_infinities_and_nan():
    logits, rules = made(MANY, 4100, 16, biases=6, masks=3, seed=24)
    some_masked(rules)
    rules["slots"][::3] = -1
    logits[:, 0:4] = torch.tensor([float("inf"), float("-inf"), float("nan"), torch.finfo(torch.float32).min], device=DEV)
    logits[:, 4096:] = logits[:, 0:4]
    rules["history"][:, :4] = torch.arange(4, dtype=torch.int32)
    rules["history"][:, 4:8] = torch.arange(4096, 4100, dtype=torch.int32)
    got = k().logit_rules(logits, **rules)
    check_rules(got, logits, **rules)
    assert torch.equal(got[::3].nan_to_num(), logits[::3].nan_to_num())
