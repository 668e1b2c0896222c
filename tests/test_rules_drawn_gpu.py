"""Tokens drawn by temperature, top-k and top-p from logits under rules: masked tokens never come, the others as often as the
definition says."""

import pytest
import torch

from rules_helpers import plain_rules
from test_logit_rules_gpu import engine_of

pytestmark = pytest.mark.gpu
DEV = "cuda"
ROWS, VOCAB = 4096, 700
ALLOWED = (3, 64, 65, 200, 333, 512, 698, 699)


def shares(logits, params):
    """What the tokens' shares are in 64 bits, from logits under the rules: top-k, then top-p of what it leaves."""
    weights = torch.softmax(logits / params.temperature, dim=0)
    order = logits.argsort(descending=True, stable=True)
    if params.top_k:
        weights[order[params.top_k:]] = 0.0
        weights /= weights.sum()
    if params.top_p < 1.0:
        before = weights[order].cumsum(0) - weights[order]
        weights[order[before > params.top_p]] = 0.0
        weights /= weights.sum()
    return weights


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("draw", [dict(), dict(top_k=3), dict(top_p=0.7), dict(top_k=5, top_p=0.8), dict(top_k=20), dict(top_p=0.999)])
@pytest.mark.parametrize("rule", [dict(allowed_token_ids=ALLOWED), dict(allowed_token_ids=ALLOWED, logit_bias={3: 2.0, 200: -1.0, 5: 50.0}),
                                  dict(allowed_token_ids=ALLOWED, repetition_penalty=1.5, presence_penalty=0.5, frequency_penalty=0.3),
                                  dict(allowed_token_ids=(699,))])
def test_shares(rule, draw, dtype):
    from tinyvllm_b200.sampling import LogitRules, Sampler, SamplingParams
    from tinyvllm_b200.sampling.rules import pack_mask

    params = SamplingParams(temperature=0.9, **rule, **draw)
    book = LogitRules(vocab=VOCAB, slots=1, room=ROWS + 16, device=DEV)
    prompt, answer = [3, 64, 700 - 2, 9], [64, 64, 333]
    book.set(0, params, prompt, answer)
    row = torch.randn(VOCAB, generator=torch.Generator().manual_seed(6)).to(dtype)
    logits = row.to(DEV).expand(ROWS, VOCAB).contiguous()
    rules = dict(slots=torch.zeros(1, dtype=torch.int32), penalties=book.penalties.cpu(), lengths=book.lengths.cpu(), history=book.history.cpu(),
                 masks=pack_mask(params.allowed_token_ids, VOCAB)[None], mask_rows=torch.zeros(1, dtype=torch.int32))
    if params.logit_bias:
        rules.update(bias_tokens=book.bias_tokens.cpu(), bias_values=book.bias_values.cpu())
    want = plain_rules(row[None], **rules)[0][0]
    if dtype == torch.bfloat16:
        want = want.to(torch.bfloat16).double()            # the logits come back in their type
    each = [SamplingParams(temperature=0.9, seed=seed, **rule, **draw) for seed in range(ROWS)]
    tokens = Sampler().sample(logits, each, [0] * ROWS, rules=book, slots=[0] * ROWS).tolist()
    assert set(tokens) <= set(params.allowed_token_ids)
    expected = shares(want, params)
    for token in params.allowed_token_ids:
        p = expected[token].item()
        # a share of ROWS draws is off by more than 5 standard deviations once in 1.7 million times
        assert abs(tokens.count(token) / ROWS - p) <= 5 * (p * (1 - p) / ROWS) ** 0.5 + 1e-12, (token, p)
    total = len(prompt) + len(answer) + ROWS                # and every draw has joined the history, in the rows' order
    assert book.lengths[0].tolist() == [total, len(prompt)] and book.history[0, total - ROWS:total].tolist() == tokens


@pytest.mark.parametrize("draw", [dict(temperature=1.0), dict(temperature=0.8, top_k=4), dict(temperature=1.3, top_p=0.9)])
def test_the_engine_draws_allowed_tokens(model_folders, draw):
    """With and without graphs the same tokens, beside requests without rules, whose tokens do not change."""
    from tiny_configs import TINY_CONFIGS, random_tokens
    from tinyvllm_b200 import GenerateRequest, SamplingParams

    folder, vocab = model_folders["b"], TINY_CONFIGS["b"].vocab_size
    allowed = tuple(range(2, vocab, 11))
    params = [SamplingParams(max_new_tokens=10, ignore_eos=True, seed=5, **draw),
              SamplingParams(max_new_tokens=10, ignore_eos=True, seed=6, allowed_token_ids=allowed, frequency_penalty=1.0, **draw),
              SamplingParams(max_new_tokens=10, ignore_eos=True, seed=7, presence_penalty=1e6, **draw)]
    prompts = [random_tokens(vocab, 5 + 7 * i, 40 + i) for i in range(3)]
    seen = []
    for eager in (False, True):
        with engine_of(folder, enforce_eager=eager) as llm:
            seen.append([list(o.output_token_ids) for o in llm.engine.generate([GenerateRequest(p, s) for p, s in zip(prompts, params)])])
            alone = llm.engine.generate([GenerateRequest(prompts[0], params[0])])
        assert list(alone[0].output_token_ids) == seen[-1][0]
    assert seen[0] == seen[1]
    assert set(seen[0][1]) <= set(allowed) and len(set(seen[0][2])) == 10          # the last one's penalty lets no token come twice
