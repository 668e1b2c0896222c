"""Rules on logits against their definition in 64 bits, in steps that are captured and replayed, and in the engine."""

import pytest
import torch

from rules_helpers import check_rules

pytestmark = pytest.mark.gpu
DEV = "cuda"


def k():
    from tinyvllm_b200.ops import kernels

    return kernels


def made(rows, vocab, room, *, slots=None, biases=0, masks=0, dtype=torch.float32, seed=0, offset=0):
    gen = torch.Generator().manual_seed(seed * 1000 + vocab + rows)
    slots = slots or rows
    logits = (torch.randn(rows, vocab + offset, generator=gen) * 3).to(dtype).to(DEV)[:, offset:]
    penalties = torch.tensor([[1.0, 0.0, 0.0], [1.3, 0.0, 0.0], [1.0, 0.5, 0.25], [0.8, -0.5, 1.5], [2.0, 0.0, -0.3]])
    rules = dict(slots=torch.randperm(slots, generator=gen)[:rows].to(torch.int32),
                 penalties=penalties[torch.randint(0, 5, (slots,), generator=gen)],
                 lengths=torch.stack([torch.randint(0, room + 1, (slots,), generator=gen)] * 2, 1).to(torch.int32),
                 history=torch.randint(0, min(vocab, 2 * room + 1), (slots, room), generator=gen).to(torch.int32))
    rules["lengths"][:, 1] //= 2
    if biases:
        rules["bias_tokens"] = torch.randint(-1, vocab, (slots, biases), generator=gen).to(torch.int32)
        rules["bias_values"] = torch.randn(slots, biases, generator=gen) * 5
    if masks:
        rules["masks"] = torch.randint(-2**31, 2**31, (masks, -(-vocab // 32)), generator=gen).to(torch.int32)
        rules["mask_rows"] = torch.randint(-1, masks, (slots,), generator=gen).to(torch.int32)
    return logits, {name: t.to(DEV) for name, t in rules.items()}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 7, 33, 4095, 4096, 4097, 8203])
def test_rules(vocab, dtype):
    logits, rules = made(5, vocab, 37, slots=9, biases=12, masks=3, dtype=dtype)
    before = logits.clone()
    got = k().logit_rules(logits, **rules)
    assert got.dtype == dtype and torch.equal(logits, before)
    check_rules(got, logits, **rules)
    again = k().logit_rules(logits, **rules)
    assert torch.equal(got, again)                                   # bit for bit
    in_place = logits.clone()
    assert k().logit_rules(in_place, out=in_place, **rules) is in_place and torch.equal(in_place, got)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [1, 3, 8])
def test_strided_rows_off_the_boundary(offset, dtype):
    logits, rules = made(4, 5003, 50, biases=5, masks=2, dtype=dtype, offset=offset)
    room = torch.full((4, 5003 + 9), 7.0, dtype=dtype, device=DEV)
    got = k().logit_rules(logits, out=room[:, 4:5007], **rules)
    check_rules(got, logits, **rules)
    assert (room[:, :4] == 7).all() and (room[:, 5007:] == 7).all()          # nothing beside the rows


def test_each_rule_alone_and_none():
    logits, rules = made(6, 611, 40, biases=9, masks=2, seed=3)
    plain = dict(slots=rules["slots"], penalties=torch.tensor([[1.0, 0.0, 0.0]] * 6, device=DEV),
                 lengths=rules["lengths"], history=rules["history"])
    assert torch.equal(k().logit_rules(logits, **plain), logits)
    for column, value in ((0, 1.7), (1, 0.9), (2, 0.4)):
        one = dict(plain, penalties=plain["penalties"].clone())
        one["penalties"][:, column] = value
        check_rules(k().logit_rules(logits, **one), logits, **one)
    for names in (("bias_tokens", "bias_values"), ("masks", "mask_rows")):
        one = dict(plain, **{name: rules[name] for name in names})
        check_rules(k().logit_rules(logits, **one), logits, **one)


def test_rows_without_a_slot_histories_of_length_0_and_1_and_numbers_out_of_range():
    logits, rules = made(7, 901, 16, slots=7, biases=6, masks=3, seed=5)
    rules["slots"] = torch.tensor([-1, 0, 7, 1, 2, -2**31, 2**31 - 1], dtype=torch.int32, device=DEV)
    rules["lengths"][:4] = torch.tensor([[0, 0], [1, 0], [99, 120], [-3, 5]], dtype=torch.int32)    # cut at the room
    rules["history"][2, :4] = torch.tensor([-1, 901, 2**31 - 1, -2**31], dtype=torch.int32)         # passed over
    rules["bias_tokens"][2, :3] = torch.tensor([901, -7, 2**31 - 1], dtype=torch.int32)
    rules["mask_rows"][:3] = torch.tensor([3, -5, 2**31 - 1], dtype=torch.int32)                    # all allowed
    got = k().logit_rules(logits, **rules)
    check_rules(got, logits, **rules)
    for row in (0, 2, 5, 6):
        assert torch.equal(got[row], logits[row])


def test_infinities_and_nan_in_masked_and_seen_places():
    logits, rules = made(3, 128, 8, masks=1, seed=2)
    logits[:, 0:4] = torch.tensor([float("inf"), float("-inf"), float("nan"), torch.finfo(torch.float32).min], device=DEV)
    rules["history"][:, :4] = torch.arange(4, dtype=torch.int32)
    rules["lengths"][:] = torch.tensor([4, 2], dtype=torch.int32)
    rules["penalties"][:] = torch.tensor([1.5, 0.5, 0.25])
    rules["mask_rows"][:] = torch.tensor([0, -1, 0], dtype=torch.int32)
    rules["masks"][0] = torch.tensor([0, -1, 1, 2**31 - 1], dtype=torch.int32)
    check_rules(k().logit_rules(logits, **rules), logits, **rules)
    rules["masks"][0] = 0                                               # nothing is allowed
    got = k().logit_rules(logits, **rules)
    for row in range(3):
        if int(rules["mask_rows"][int(rules["slots"][row])]) == 0:
            assert (got[row] == float("-inf")).all()


def test_a_token_named_many_times_gets_all_its_biases_in_their_order():
    logits, rules = made(2, 300, 4, biases=64, seed=8)
    rules["bias_tokens"][:, ::3] = 17
    rules["bias_tokens"][:, 1::3] = 299
    got = k().logit_rules(logits, **rules)
    check_rules(got, logits, **rules)
    for _ in range(5):
        assert torch.equal(k().logit_rules(logits, **rules), got)
    tokens, values = rules["bias_tokens"].cpu(), rules["bias_values"].cpu()
    for row in range(2):                                                # float32 sums, first entry first
        slot, total = int(rules["slots"][row]), torch.zeros(())
        for i in range(64):
            if tokens[slot, i] == 17:
                total = total + values[slot, i]
        seen = 17 in rules["history"][slot, :int(rules["lengths"][slot, 0])].tolist()
        if not seen:
            assert got[row, 17].item() == (logits[row, 17].cpu() + total).item()


def test_long_histories_and_most_biases():
    logits, rules = made(3, 151936, 20001, biases=1024, masks=2, seed=4)
    rules["history"][1] = 5                                             # one token again and again
    want_rows = k().logit_rules(logits, **rules)
    part = 9001                                                         # (the oracle walks token by token)
    cut = {name: t for name, t in rules.items()}
    cut["masks"] = rules["masks"][:, :-(-part // 32)].contiguous()
    check_rules(want_rows[:, :part], logits[:, :part], **cut)


def test_two_rows_of_one_slot():
    logits, rules = made(2, 999, 30, slots=2, biases=3, masks=1)
    rules["slots"] = torch.tensor([1, 1], dtype=torch.int32, device=DEV)
    check_rules(k().logit_rules(logits, **rules), logits, **rules)


def test_no_rows():
    logits, rules = made(1, 40, 4)
    rules["slots"] = rules["slots"][:0]
    assert k().logit_rules(logits[:0], **rules).shape == (0, 40)


def test_appended_tokens():
    slots = torch.tensor([2, -1, 0, 2, 5, 2, 0, 9], dtype=torch.int32, device=DEV)
    tokens = torch.arange(10, 18, dtype=torch.int32, device=DEV)
    lengths = torch.tensor([[3, 1], [2, 2], [0, 0], [1, 1], [1, 1], [4, 2]], dtype=torch.int32, device=DEV)
    history = torch.zeros(6, 4, dtype=torch.int32, device=DEV)
    k().append_tokens(tokens, slots=slots, lengths=lengths, history=history)
    assert lengths.tolist() == [[4, 1], [2, 2], [3, 0], [1, 1], [1, 1], [4, 2]]     # slots 0 and 5 are full
    assert history.tolist() == [[0, 0, 0, 12], [0] * 4, [10, 13, 15, 0], [0] * 4, [0] * 4, [0] * 4]
    many = torch.randint(-1, 40, (1500,), dtype=torch.int32, device=DEV)
    lengths, history = torch.zeros(40, 2, dtype=torch.int32, device=DEV), torch.zeros(40, 1500, dtype=torch.int32, device=DEV)
    k().append_tokens(torch.arange(1500, dtype=torch.int32, device=DEV), slots=many, lengths=lengths, history=history)
    for slot in range(40):
        mine = (many == slot).nonzero()[:, 0].tolist()
        assert lengths[slot, 0].item() == len(mine) and history[slot, :len(mine)].tolist() == mine


def test_a_captured_step_counts_the_tokens_of_the_steps_before():
    """Rules, greedy sampling and the tokens' return into the history, captured once and replayed: with a penalty larger
    than any logit no token comes twice."""
    from tinyvllm_b200.sampling import LogitRules, SamplingParams
    from tinyvllm_b200.sampling.sampler import pack_rows, sample_packed

    rules = LogitRules(vocab=1000, slots=3, room=64, device=DEV)
    for slot in range(2):
        rules.set(slot, SamplingParams(presence_penalty=100.0), [5, 6])
    logits = torch.randn(3, 1000, generator=torch.Generator().manual_seed(1)).to(DEV)
    slots = torch.tensor([1, -1, 0], dtype=torch.int32, device=DEV)
    packed = torch.from_numpy(pack_rows([SamplingParams()] * 3, [0] * 3)).to(DEV)
    tokens = torch.zeros(3, dtype=torch.int32, device=DEV)

    def step():
        sample_packed(rules.apply(logits, slots), packed, out=tokens)
        rules.append(tokens, slots)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
        stream.synchronize()
        first = tokens.tolist()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
    drawn = [first]
    for _ in range(20):
        graph.replay()
        drawn.append(tokens.tolist())
    order = [logits[row].argsort(descending=True)[:21].tolist() for row in range(3)]
    assert [t[0] for t in drawn] == order[0] and [t[2] for t in drawn] == order[2]
    assert {t[1] for t in drawn} == {order[1][0]}


def test_on_another_stream():
    logits, rules = made(4, 9001, 30, biases=4, masks=1, seed=11)
    want = k().logit_rules(logits, **rules)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = k().logit_rules(logits, **rules)
    stream.synchronize()
    assert torch.equal(got, want)


# ----------------------------------------------------------------- the engine
def engine_of(folder, **more):
    from tinyvllm_b200 import EngineConfig, LLM

    return LLM(EngineConfig(model=folder, dtype="float32", max_model_len=128, max_num_seqs=4, max_num_batched_tokens=64,
                            prefill_chunk_size=16, kv_block_size=8, kv_cache_memory_bytes=8 * 1024 * 1024,
                            prefill_reserve_tokens=0, prefill_reserve_requests=0, **more))


def plain_generate(cfg, weights, prompt, count, params):
    """Greedy tokens of the plain implementation under the rules."""
    import plain_qwen3 as plain
    from rules_helpers import plain_rules

    tokens = list(prompt)
    for _ in range(count):
        logits = plain.forward(cfg, weights, tokens)[-1:].float()
        history = torch.tensor([tokens], dtype=torch.int32)
        vocab = logits.shape[1]
        rules = dict(slots=torch.zeros(1, dtype=torch.int32), history=history,
                     lengths=torch.tensor([[len(tokens), len(prompt)]]),
                     penalties=torch.tensor([[params.repetition_penalty, params.presence_penalty, params.frequency_penalty]]))
        if params.logit_bias:
            rules.update(bias_tokens=torch.tensor([[t for t, _ in params.logit_bias]]),
                         bias_values=torch.tensor([[b for _, b in params.logit_bias]]))
        if params.allowed_token_ids is not None:
            from tinyvllm_b200.sampling.rules import pack_mask

            rules.update(masks=pack_mask(params.allowed_token_ids, vocab)[None], mask_rows=torch.zeros(1, dtype=torch.int32))
        tokens.append(int(plain_rules(logits, **rules)[0][0].argmax()))
    return tokens[len(prompt):]


@pytest.mark.parametrize("eager", [False, True])
def test_the_engine_generates_under_the_rules(model_folders, eager):
    """Requests with and without rules in one batch, more of them than there are slots: every one gets the tokens the plain
    implementation draws for it alone."""
    import plain_qwen3 as plain
    from tiny_configs import TINY_CONFIGS, random_tokens
    from tinyvllm_b200 import GenerateRequest, SamplingParams

    folder = model_folders["b"]
    vocab = TINY_CONFIGS["b"].vocab_size
    rules = [dict(), dict(repetition_penalty=1.8), dict(presence_penalty=3.0, frequency_penalty=0.7), dict(),
             dict(allowed_token_ids=tuple(range(3, vocab, 7))), dict(logit_bias={11: 50.0}, frequency_penalty=30.0),
             dict(logit_bias=[(5, -2.0)], allowed_token_ids=(5, 6, 8), presence_penalty=1.0)]
    params = [SamplingParams(max_new_tokens=8, ignore_eos=True, **rule) for rule in rules]
    prompts = [random_tokens(vocab, 3 + 5 * i, 70 + i) for i in range(len(rules))]
    with engine_of(folder, enforce_eager=eager) as llm:
        outputs = llm.engine.generate([GenerateRequest(p, s) for p, s in zip(prompts, params)])
        bare = llm.engine.generate([GenerateRequest(p, params[0]) for p in prompts[:2]])      # and runs again behind them
        with pytest.raises(ValueError, match="vocabulary"):
            llm.engine.submit([1], SamplingParams(logit_bias={vocab: 1.0}))
    cfg, weights = plain.read_config(folder), plain.read_weights(folder)
    for prompt, output, param in zip(prompts, outputs, params):
        assert list(output.output_token_ids) == plain_generate(cfg, weights, prompt, 8, param)
    for prompt, output in zip(prompts, bare):
        assert list(output.output_token_ids) == plain.greedy_generate(cfg, weights, prompt, 8)
