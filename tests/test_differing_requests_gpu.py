"""A batch whose requests share their prompt's first pages, have an adapter each and rules of their own: projections with adapters,
attention over the keys in common, rules and sampling in one decode step that is captured and replayed, against the same model run
request by request in 64 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
VOCAB, WIDTH, HEADS, KV, DIM, PAGE, RANK, ROOM = 193, 128, 4, 2, 64, 16, 8, 128


def weights(dtype):
    gen = torch.Generator().manual_seed(5)

    def draw(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen) * scale).to(dtype).to(DEV)

    columns = (HEADS + 2 * KV) * DIM
    return dict(table=draw(VOCAB, WIDTH), qkv=draw(columns, WIDTH, scale=WIDTH**-0.5), out=draw(WIDTH, HEADS * DIM, scale=(HEADS * DIM)**-0.5),
                head=draw(VOCAB, WIDTH, scale=2 * WIDTH**-0.5), qkv_down=draw(2, RANK, WIDTH, scale=WIDTH**-0.5),
                qkv_up=draw(2, columns, RANK, scale=RANK**-0.5), out_down=draw(5, RANK, HEADS * DIM, scale=(HEADS * DIM)**-0.5),
                out_up=draw(5, WIDTH, RANK, scale=2 * RANK**-0.5), out_scales=(torch.rand(5, generator=gen) + 0.5).to(DEV))


# (tokens that the group's requests share, what each has behind them); a group has one adapter where its keys are made
GROUPS = [(list(range(3, 37)), [[40], [41, 5], [42, 9, 11]]), (list(range(60, 108)), [[7, 8], [120]])]
OUT_ADAPTERS = [0, 3, -1, 1, 4]


def rules():
    from tinyvllm_b200 import SamplingParams

    return [SamplingParams(repetition_penalty=1.4), SamplingParams(presence_penalty=2.0, frequency_penalty=0.5), SamplingParams(),
            SamplingParams(allowed_token_ids=tuple(range(0, VOCAB, 3)), frequency_penalty=1.0), SamplingParams(logit_bias={17: 2.5, 90: -3.0})]


def plain_logits(w, tokens, group, adapter):
    """The last token's logits in 64 bits."""
    wide = {name: t.double() for name, t in w.items()}
    x = wide["table"][torch.tensor(tokens, device=DEV)]
    qkv = x @ wide["qkv"].t() + (x @ wide["qkv_down"][group].t()) @ wide["qkv_up"][group].t()
    q, k, v = (part.view(len(tokens), -1, DIM).transpose(0, 1) for part in qkv.split([HEADS * DIM, KV * DIM, KV * DIM], dim=1))
    k, v = (t.repeat_interleave(HEADS // KV, dim=0) for t in (k, v))
    heads = (torch.softmax(q[:, -1:] @ k.transpose(1, 2) * DIM**-0.5, dim=-1) @ v).reshape(1, -1)
    out = heads @ wide["out"].t()
    if adapter >= 0:
        out = out + wide["out_scales"][adapter] * (heads @ wide["out_down"][adapter].t()) @ wide["out_up"][adapter].t()
    return (x[-1:] + out) @ wide["head"].t()


@pytest.mark.parametrize("hints", [{}, dict(max_shared=1 << 30)], ids=["alone", "together"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decode_steps(dtype, hints):
    from rules_helpers import plain_rules
    from tinyvllm_b200.ops import kernels, linear, linear_adapted
    from tinyvllm_b200.sampling import LogitRules
    from tinyvllm_b200.sampling.rules import pack_mask
    from tinyvllm_b200.sampling.sampler import pack_rows, sample_packed

    w, params = weights(dtype), rules()
    requests = [(g, common + own) for g, (common, owns) in enumerate(GROUPS) for own in owns]
    count, steps = len(requests), 6
    int_of = lambda values: torch.tensor(values, dtype=torch.int32, device=DEV)                     # noqa: E731
    # pages: a group's whole shared pages once, everything behind them a request's own
    tables, pages, shared_lens = [], 0, []
    for common, owns in GROUPS:
        whole = len(common) // PAGE
        shared_lens.append(whole * PAGE)
        first = list(range(pages, pages + whole))
        pages += whole
        for own in owns:
            more = -(-(len(common) + len(own) + steps) // PAGE) - whole
            tables.append(first + list(range(pages, pages + more)))
            pages += more
    table = torch.full((count, max(map(len, tables))), -1, dtype=torch.int32, device=DEV)
    for r, t in enumerate(tables):
        table[r, :len(t)] = int_of(t)
    caches = [torch.zeros(pages, KV, PAGE, DIM, dtype=dtype, device=DEV) for _ in range(2)]
    groups = int_of([g for g, _ in requests])
    starts, shared = int_of([0, 3, 5]), int_of(shared_lens)
    book = LogitRules(vocab=VOCAB, slots=count, room=ROOM, device=DEV)
    for r, (_, tokens) in enumerate(requests):
        book.set(r, params[r], tokens)

    def project(ids, adapter, positions, slots):
        x = kernels.embed_rows(w["table"], ids)
        qkv = linear_adapted(x, w["qkv"], w["qkv_down"], w["qkv_up"], adapter)
        kernels.qk_norm_rope_store(qkv, num_q=HEADS, num_kv=KV, head_dim=DIM, positions=positions, q_weight=None, k_weight=None, eps=0.0,
                                   cos=None, sin=None, slots=slots, key_cache=caches[0], value_cache=caches[1])
        return x, qkv

    def slots_of(row, positions):
        return [int(table[row, p // PAGE]) * PAGE + p % PAGE for p in positions]

    for r, (g, tokens) in enumerate(requests):                       # the prompts, but for their last tokens
        places = list(range(len(tokens) - 1))
        project(int_of(tokens[:-1]), int_of([g] * len(places)), int_of(places), int_of(slots_of(r, places)))
    ids = int_of([tokens[-1] for _, tokens in requests])
    positions = int_of([len(tokens) - 1 for _, tokens in requests])
    slots, rows = torch.zeros_like(ids), torch.arange(count, dtype=torch.int32, device=DEV)
    packed = torch.from_numpy(pack_rows([p for p in params], [0] * count)).to(DEV)
    out_adapters, logits_seen = int_of(OUT_ADAPTERS), torch.zeros(count, VOCAB, device=DEV)

    def step():
        x, qkv = project(ids, groups, positions, slots)
        heads = kernels.attention_shared(qkv, qkv.shape[1], *caches, table, rows, positions, group_starts=starts, shared_lens=shared,
                                         num_q=HEADS, num_kv=KV, head_dim=DIM, scale=DIM**-0.5, **hints)
        out = linear_adapted(heads, w["out"], w["out_down"], w["out_up"], out_adapters, w["out_scales"])
        logits = linear(x + out, w["head"], out_dtype=torch.float32)
        logits_seen.copy_(logits)
        sample_packed(book.apply(logits, rows, out=logits), packed, out=ids)
        book.append(ids, rows)

    lengths = book.lengths.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.inference_mode(), torch.cuda.stream(stream):
        kept = ids.clone()
        slots.copy_(int_of([slots_of(r, [int(p)])[0] for r, p in enumerate(positions.tolist())]))
        step()                                                       # settles what libraries set up; then all is as it was
        ids.copy_(kept)
        book.lengths.copy_(lengths)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
        texts = [list(tokens) for _, tokens in requests]
        for _ in range(steps):
            places = positions.tolist()
            slots.copy_(int_of([slots_of(r, [p])[0] for r, p in enumerate(places)]))
            graph.replay()
            stream.synchronize()
            for r, (g, tokens) in enumerate(requests):
                logits = plain_logits(w, texts[r], g, OUT_ADAPTERS[r])
                off = (logits_seen[r].double() - logits[0]).abs().max().item() / logits.abs().max().item()
                # float32: five products in line of up to 256 terms, whose sums are off by some 2^-23 sqrt(256) of what is added up, so
                # 1e-5 in all, and twice that is allowed.  bfloat16: eight roundings on the way (each projection's two, the softmax's
                # weights, the heads, x + out and the rest of its own), 2^-8 each at the most, all of them at once.
                assert off < (2e-5 if dtype == torch.float32 else 8 * 2.0**-8)
                p = params[r]
                held = dict(slots=torch.zeros(1, dtype=torch.int32), history=torch.tensor([texts[r]], dtype=torch.int32),
                            lengths=torch.tensor([[len(texts[r]), len(tokens)]]),
                            penalties=torch.tensor([[p.repetition_penalty, p.presence_penalty, p.frequency_penalty]]))
                if p.logit_bias:
                    held.update(bias_tokens=torch.tensor([[t for t, _ in p.logit_bias]]), bias_values=torch.tensor([[b for _, b in p.logit_bias]]))
                if p.allowed_token_ids is not None:
                    held.update(masks=pack_mask(p.allowed_token_ids, VOCAB)[None], mask_rows=torch.zeros(1, dtype=torch.int32))
                # the rules and the choice from the logits that the step had
                want = int(plain_rules(logits_seen[r:r + 1].cpu(), **held)[0][0].argmax())
                assert int(ids[r]) == want
                texts[r].append(want)
            positions += 1
    kernels.check_finished_launches()
