"""Operators of a batch whose requests differ, or share something: what is measured of them, in plain form and as kernels.

* rules: the logits of every row under its request's own penalties for tokens it has seen, biases and allowed tokens,
  as they stand before sampling (``ops.kernels.logit_rules``).
* adapted: one projection of all rows, to which every row's own low-rank adapter is added (``ops.linear_adapted``).
* shared: attention of decoded tokens over the paged cache, where groups of requests have their first pages in common
  and read them once (``ops.kernels.attention_shared``).

A case holds the sizes of one call.  ``run`` makes the call of a user's program where ``own`` is true, else the same
result from elementary torch operations in 32 bits; ``exact`` has it from the definitions in 64 bits.
"""

import math
import random

import torch

own = False

DEVICE = "cuda"
PAGE = 16
# query heads, key/value heads, head size: the benchmark's layers, and generic ones
HEADS = {"16x8x128": (16, 8, 128), "32x8x128": (32, 8, 128), "64x8x128": (64, 8, 128), "8x8x64": (8, 8, 64),
         "14x2x64": (14, 2, 64), "8x4x256": (8, 4, 256)}
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def _rules(name, rows, vocab, history, biases=0, masked="none", dtype="float32"):
    made = dict(kind="rules", rows=rows, vocab=vocab, history=history, biases=biases, masked=masked, dtype=dtype)
    return made if name is None else dict(name=name, **made)


def _adapted(name, rows, k, n, rank, adapters, spans, bare=False, dtype="bfloat16"):
    made = dict(kind="adapted", rows=rows, k=k, n=n, rank=rank, adapters=adapters, spans=spans, bare=bare, dtype=dtype)
    return made if name is None else dict(name=name, **made)


def _shared(name, groups, members, shared, own_keys, heads="16x8x128", dtype="bfloat16"):
    made = dict(kind="shared", groups=groups, members=members, shared=shared, own_keys=own_keys, heads=heads, dtype=dtype)
    return made if name is None else dict(name=name, **made)


def listed():
    return [
        # one user chatting with a penalty for repetition: the latency before a single token's sampling
        _rules("rules-1", rows=1, vocab=151936, history=607),
        # a busy server: long answers, some requests with biases, a few of them held to a grammar
        _rules("rules-64-long", rows=64, vocab=151936, history=4001, biases=300, masked="some"),
        # structured output: every request may go on with few tokens only
        _rules("rules-24-grammar", rows=24, vocab=151936, history=900, biases=20, masked="few"),
        # bfloat16 logits of an odd vocabulary
        _rules("rules-7-odd", rows=7, vocab=32003, history=333, biases=11, masked="some", dtype="bfloat16"),
        # one request of a tuned model: the latency of its projection
        _adapted("adapted-1", rows=1, k=1024, n=4096, rank=16, adapters=4, spans=1),
        # a decode step of many tenants: 48 requests, 13 adapters, some requests without one
        _adapted("adapted-48", rows=48, k=4096, n=6144, rank=16, adapters=13, spans=48, bare=True),
        # portions of six prompts in one batch, adapters of a higher rank
        _adapted("adapted-prompts", rows=4099, k=4096, n=4096, rank=64, adapters=5, spans=6, bare=True),
        # the 32-bit path, used to check a model's numbers
        _adapted("adapted-float32", rows=301, k=1024, n=2048, rank=8, adapters=3, spans=4, dtype="float32"),
        # two answers to one short question: the latency of a single layer
        _shared("shared-2", groups=1, members=2, shared=208, own_keys=23),
        # sixty answers sampled from one prompt of a document's length
        _shared("shared-60", groups=1, members=60, shared=6144, own_keys=431, heads="32x8x128"),
        # three system prompts, each with its users' questions behind it, at the widest layers
        _shared("shared-3-prompts", groups=3, members=13, shared=2896, own_keys=777, heads="64x8x128"),
        # the 32-bit path
        _shared("shared-float32", groups=2, members=5, shared=608, own_keys=120, dtype="float32"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng):
    kind = rng.choice(["rules", "adapted", "shared"])
    if kind == "rules":
        rows, vocab = _log_int(rng, 1, 64), _log_int(rng, 1009, 151936)
        return _rules(None, rows, vocab, rng.choice([0, _log_int(rng, 1, 4000), _log_int(rng, 64, 4000)]),
                      rng.choice([0, _log_int(rng, 1, 300)]), rng.choice(["none", "some", "few"]),
                      rng.choice(["float32", "float32", "bfloat16"]))
    if kind == "adapted":
        dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
        few = rng.random() < 0.5
        rows = _log_int(rng, 1, 64) if few else _log_int(rng, 65, 4000 if dtype == "bfloat16" else 600)
        k, n = 8 * _log_int(rng, 32, 512), _log_int(rng, 250, 4096)
        return _adapted(None, rows, k, n, rng.choice([4, 8, 16, 32, 64]), _log_int(rng, 1, 32),
                        rng.randint(1, rows) if few else rng.randint(1, min(rows, 12)), rng.random() < 0.5, dtype)
    groups, dtype = rng.randint(1, 4), rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    members = _log_int(rng, 1, 60 // groups if dtype == "bfloat16" else 12 // groups)
    return _shared(None, groups, members, PAGE * _log_int(rng, 1, 380 if dtype == "bfloat16" else 60),
                   _log_int(rng, 1, 430 if dtype == "bfloat16" else 200), rng.choice(sorted(HEADS)), dtype)


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _normal(gen, *shape, dtype=torch.float32, scale=1.0):
    return torch.randn(*shape, generator=gen, device=DEVICE, dtype=torch.float32).mul_(scale).to(dtype)


# -------------------------------------------------------------------------------------------------- rules
def _prepare_rules(case, seed):
    gen, rng = _generator(seed), random.Random(seed)
    rows, vocab, room = case["rows"], case["vocab"], max(1, case["history"])
    # half of each prompt and answer comes from few tokens, as text does
    common = torch.randint(0, vocab, (rows, max(1, room // 8)), generator=gen, device=DEVICE)
    repeated = common.gather(1, torch.randint(0, common.shape[1], (rows, room), generator=gen, device=DEVICE))
    fresh = torch.randint(0, vocab, (rows, room), generator=gen, device=DEVICE)
    history = torch.where(torch.rand(rows, room, generator=gen, device=DEVICE) < 0.5, repeated, fresh).to(torch.int32)
    lengths = [[case["history"] - (case["history"] * i) // (2 * rows), 0] for i in range(rows)]
    for pair in lengths:
        pair[1] = rng.randint(0, pair[0])                                          # of them the prompt
    penalties = [[rng.choice([1.0, 1.1, 1.3]), rng.choice([0.0, 0.5, 1.5]), rng.choice([0.0, 0.25, 0.7])] for _ in range(rows)]
    order = list(range(rows))
    rng.shuffle(order)                                                             # which slot a row's request holds
    state = dict(case=case, logits=_normal(gen, rows, vocab, dtype=TYPES[case["dtype"]], scale=3.0),
                 slots=torch.tensor(order, dtype=torch.int32, device=DEVICE),
                 penalties=torch.tensor(penalties, dtype=torch.float32, device=DEVICE),
                 lengths=torch.tensor(lengths, dtype=torch.int32, device=DEVICE), history=history,
                 bias_tokens=None, bias_values=None, masks=None, mask_rows=None)
    if case["biases"]:
        most = min(case["biases"], vocab)
        tokens = torch.rand(rows, vocab, generator=gen, device=DEVICE).topk(most, dim=1).indices.to(torch.int32)
        counts = torch.tensor([rng.choice([0, most, most // 2]) for _ in range(rows)], device=DEVICE)
        tokens[torch.arange(most, device=DEVICE)[None] >= counts[:, None]] = -1    # places without a bias
        state.update(bias_tokens=tokens, bias_values=_normal(gen, rows, most, scale=4.0))
    if case["masked"] != "none":
        share = 0.9 if case["masked"] == "some" else 0.004
        kinds = 4                                                                  # grammars' states among the requests
        allowed = torch.rand(kinds, -(-vocab // 32) * 32, generator=gen, device=DEVICE) < share
        words = (allowed.view(kinds, -1, 32).to(torch.int64) << torch.arange(32, device=DEVICE)).sum(-1)
        state["masks"] = torch.where(words >= 2**31, words - 2**32, words).to(torch.int32)
        held = [rng.randrange(kinds) if case["masked"] == "few" or rng.random() < 0.25 else -1 for _ in range(rows)]
        state["mask_rows"] = torch.tensor(held, dtype=torch.int32, device=DEVICE)
    return state


def _run_rules(s):
    if own:
        from tinyvllm_b200.ops import kernels

        return kernels.logit_rules(s["logits"], slots=s["slots"], penalties=s["penalties"], lengths=s["lengths"],
                                   history=s["history"], bias_tokens=s["bias_tokens"], bias_values=s["bias_values"],
                                   masks=s["masks"], mask_rows=s["mask_rows"])
    slot, vocab = s["slots"].long(), s["logits"].shape[1]
    x = s["logits"].float()
    at = torch.arange(s["history"].shape[1], device=x.device)[None]
    lengths, penalties, tokens = s["lengths"][slot], s["penalties"][slot], s["history"][slot].long()
    answered = ((at >= lengths[:, 1:]) & (at < lengths[:, :1])).float()
    count = torch.zeros_like(x).scatter_add_(1, tokens, answered)
    seen = torch.zeros_like(x).scatter_add_(1, tokens, (at < lengths[:, :1]).float()) > 0
    repetition, presence, frequency = penalties[:, 0:1], penalties[:, 1:2], penalties[:, 2:3]
    x = torch.where(seen, torch.where(x > 0, x / repetition, x * repetition), x)
    x = x - frequency * count - presence * (count > 0).float()
    if s["bias_tokens"] is not None:
        token, value = s["bias_tokens"][slot].long(), s["bias_values"][slot]
        x = x.scatter_add(1, token.clamp(min=0), torch.where(token >= 0, value, torch.zeros_like(value)))
    if s["masks"] is not None:
        row, v = s["mask_rows"][slot].long(), torch.arange(vocab, device=x.device)
        bit = (s["masks"][row.clamp(min=0)][:, v // 32] >> (v % 32)) & 1
        x = torch.where((bit == 1) | (row < 0)[:, None], x, float("-inf"))
    return x.to(s["logits"].dtype)


def _exact_rules(case, seed):
    s = _prepare_rules(case, seed)
    out = s["logits"].double()
    for r, slot in enumerate(s["slots"].tolist()):
        total, prompt = s["lengths"][slot].tolist()
        repetition, presence, frequency = s["penalties"][slot].double().tolist()
        tokens, counts = s["history"][slot, prompt:total].long().unique(return_counts=True)
        seen = s["history"][slot, :total].long().unique()
        values = out[r, seen]
        out[r, seen] = torch.where(values > 0, values / repetition, values * repetition)
        out[r, tokens] -= frequency * counts.double() + presence
        if s["bias_tokens"] is not None:
            named = s["bias_tokens"][slot] >= 0
            out[r, s["bias_tokens"][slot][named].long()] += s["bias_values"][slot][named].double()
        if s["masks"] is not None and s["mask_rows"][slot] >= 0:
            words = s["masks"][s["mask_rows"][slot]].long() & 0xFFFFFFFF
            bits = torch.stack([(words >> b) & 1 for b in range(32)], dim=1).reshape(-1)[:case["vocab"]]
            out[r, bits == 0] = float("-inf")
    return out


def _work_rules(case):
    rows, vocab, size = case["rows"], case["vocab"], 4 if case["dtype"] == "float32" else 2
    moved = 2 * rows * vocab * size + rows * (3 * case["history"] + 24)            # ragged: three quarters of the longest
    moved += rows * case["biases"] * 4 + (4 * -(-vocab // 32) * 4 if case["masked"] != "none" else 0)
    return {"bytes": moved, "flops": 4 * rows * vocab}


# ------------------------------------------------------------------------------------------------- adapted
def _prepare_adapted(case, seed):
    gen, rng = _generator(seed), random.Random(seed)
    rows, k, n, rank, count, dtype = (case[name] for name in ("rows", "k", "n", "rank", "adapters", "dtype"))
    dtype = TYPES[dtype]
    cuts = sorted(rng.sample(range(1, rows), min(case["spans"], rows) - 1)) if rows > 1 else []
    ids, start = [], 0
    for end in cuts + [rows]:                                                      # a request's rows stand together
        ids += [-1 if case["bare"] and rng.random() < 0.2 else rng.randrange(count)] * (end - start)
        start = end
    return dict(case=case, x=_normal(gen, rows, k, dtype=dtype), weight=_normal(gen, n, k, dtype=dtype, scale=k ** -0.5),
                down=_normal(gen, count, rank, k, dtype=dtype, scale=k ** -0.5),
                up=_normal(gen, count, n, rank, dtype=dtype, scale=0.5 * rank ** -0.5),
                scales=torch.tensor([rng.choice([0.5, 1.0, 2.0]) for _ in range(count)], dtype=torch.float32, device=DEVICE),
                ids=torch.tensor(ids, dtype=torch.int32, device=DEVICE))


def _run_adapted(s):
    if own:
        from tinyvllm_b200.ops import linear_adapted

        return linear_adapted(s["x"], s["weight"], s["down"], s["up"], s["ids"], s["scales"], weight_constant=True)
    x, (count, rank, k), n = s["x"].float(), s["down"].shape, s["weight"].shape[0]
    # all adapters side by side; a row keeps its own one's share
    narrow = (x @ s["down"].float().view(count * rank, k).t()).view(-1, count, rank)
    chosen = s["ids"][:, None] == torch.arange(count, device=x.device)[None]
    narrow = narrow * torch.where(chosen, s["scales"][None], 0.0)[:, :, None]
    wide = s["up"].float().permute(0, 2, 1).reshape(count * rank, n)
    return (x @ s["weight"].float().t() + narrow.view(-1, count * rank) @ wide).to(s["x"].dtype)


def _exact_adapted(case, seed):
    s = _prepare_adapted(case, seed)
    x = s["x"].double()
    out = x @ s["weight"].double().t()
    for a in range(case["adapters"]):
        mine = (s["ids"] == a).nonzero()[:, 0]
        out[mine] += s["scales"][a].double() * ((x[mine] @ s["down"][a].double().t()) @ s["up"][a].double().t())
    return out


def _work_adapted(case):
    rows, k, n, rank = (case[name] for name in ("rows", "k", "n", "rank"))
    size, used = 4 if case["dtype"] == "float32" else 2, min(case["adapters"], case["spans"], rows)
    return {"bytes": size * (rows * (k + n) + n * k + used * rank * (k + n)) + 4 * rows,
            "flops": 2 * rows * (n * k + rank * (k + n))}


# -------------------------------------------------------------------------------------------------- shared
def _own_keys(case, i):
    """Keys that member i of a group has behind the shared ones: from the longest down to a quarter of it."""
    return max(1, case["own_keys"] - (3 * case["own_keys"] * i) // (4 * case["members"]))


def _shared_keys(case, g):
    return PAGE * max(1, (case["shared"] - (case["shared"] * g) // (2 * case["groups"])) // PAGE)


def _prepare_shared(case, seed):
    gen, rng = _generator(seed), random.Random(seed)
    (num_q, num_kv, dim), dtype = HEADS[case["heads"]], TYPES[case["dtype"]]
    rows = case["groups"] * case["members"]
    tables, positions, pages = [], [], 0
    for g in range(case["groups"]):
        common = _shared_keys(case, g)
        first = list(range(pages, pages + common // PAGE))
        pages += len(first)
        for i in range(case["members"]):
            more = -(-_own_keys(case, i) // PAGE)
            tables.append(first + list(range(pages, pages + more)))
            positions.append(common + _own_keys(case, i) - 1)
            pages += more
    place = list(range(pages))
    rng.shuffle(place)                                                             # pages lie anywhere in the pool
    width = max(len(t) for t in tables)
    table = torch.tensor([[place[p] for p in t] + [0] * (width - len(t)) for t in tables], dtype=torch.int32, device=DEVICE)
    return dict(case=case, q=_normal(gen, rows, num_q * dim, dtype=dtype),
                keys=_normal(gen, pages, num_kv, PAGE, dim, dtype=dtype), values=_normal(gen, pages, num_kv, PAGE, dim, dtype=dtype),
                tables=table, token_row=torch.arange(rows, dtype=torch.int32, device=DEVICE),
                positions=torch.tensor(positions, dtype=torch.int32, device=DEVICE),
                group_starts=torch.arange(0, rows + 1, case["members"], dtype=torch.int32, device=DEVICE),
                shared_lens=torch.tensor([_shared_keys(case, g) for g in range(case["groups"])], dtype=torch.int32, device=DEVICE),
                max_shared=_shared_keys(case, 0), max_own=case["own_keys"])


def _run_shared(s):
    num_q, num_kv, dim = HEADS[s["case"]["heads"]]
    if own:
        from tinyvllm_b200.ops import kernels

        return kernels.attention_shared(s["q"], s["q"].shape[1], s["keys"], s["values"], s["tables"], s["token_row"],
                                        s["positions"], group_starts=s["group_starts"], shared_lens=s["shared_lens"],
                                        num_q=num_q, num_kv=num_kv, head_dim=dim, scale=dim ** -0.5,
                                        max_shared=s["max_shared"], max_own=s["max_own"])
    rows = s["tables"][s["token_row"].long()].long()
    tokens = rows.shape[0]

    def gathered(cache):                                                           # [tokens, kv heads, keys, size]
        return cache[rows].permute(0, 2, 1, 3, 4).reshape(tokens, num_kv, -1, dim).float()

    q = s["q"].float().view(tokens, num_kv, num_q // num_kv, dim)
    scores = (q @ gathered(s["keys"]).transpose(2, 3)) * dim ** -0.5
    behind = torch.arange(scores.shape[3], device=q.device)[None] > s["positions"][:, None]
    scores = scores.masked_fill(behind[:, None, None], float("-inf"))
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = (weights @ gathered(s["values"])) / weights.sum(-1, keepdim=True)
    return out.reshape(tokens, num_q * dim).to(s["q"].dtype)


def _exact_shared(case, seed):
    s = _prepare_shared(case, seed)
    num_q, num_kv, dim = HEADS[case["heads"]]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    for t, last in enumerate(s["positions"].tolist()):
        where = torch.arange(last + 1, device=DEVICE)
        page, slot = s["tables"][t].long()[where // PAGE], where % PAGE
        k, v = s["keys"][page, :, slot].double(), s["values"][page, :, slot].double()             # [keys, kv heads, size]
        q = s["q"][t].double().view(num_kv, num_q // num_kv, dim)
        weights = torch.softmax(torch.einsum("hgd,khd->hgk", q, k) / math.sqrt(dim), dim=-1)
        out[t] = torch.einsum("hgk,khd->hgd", weights, v).reshape(-1)
    return out


def _work_shared(case):
    (num_q, num_kv, dim), size = HEADS[case["heads"]], 4 if case["dtype"] == "float32" else 2
    commons = [_shared_keys(case, g) for g in range(case["groups"])]
    owns = [_own_keys(case, i) for i in range(case["members"])]
    rows = case["groups"] * case["members"]
    read = sum(commons) + case["groups"] * sum(owns)
    attended = case["members"] * sum(commons) + case["groups"] * sum(owns)
    return {"bytes": size * (2 * read * num_kv * dim + 2 * rows * num_q * dim), "flops": 4 * attended * num_q * dim}


# ------------------------------------------------------------------------------------------------ the cases
_PARTS = {"rules": (_prepare_rules, _run_rules, _exact_rules, _work_rules),
          "adapted": (_prepare_adapted, _run_adapted, _exact_adapted, _work_adapted),
          "shared": (_prepare_shared, _run_shared, _exact_shared, _work_shared)}


@torch.no_grad()
def prepare(case, seed):
    return _PARTS[case["kind"]][0](case, seed)


@torch.no_grad()
def run(state):
    return _PARTS[state["case"]["kind"]][1](state)


@torch.no_grad()
def exact(case, seed):
    return _PARTS[case["kind"]][2](case, seed)


def work(case):
    return _PARTS[case["kind"]][3](case)
