"""Operands of more than 2^31 elements: what lies at their end is read and written as it is in small ones."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("page, dim, dtype", [(16, 128, torch.bfloat16), (16, 256, torch.bfloat16), (48, 64, torch.bfloat16), (16, 128, torch.float32)])
def test_attention_at_the_end_of_a_long_cache(page, dim, dtype):
    """The same keys in a cache of their own, bit for bit."""
    from shared_helpers import check_attention, made
    from tinyvllm_b200.ops import kernels

    s, sizes = made([(5 * page + 7, [5, 40, 1]), (200, [9, 3])], num_q=4, num_kv=4, dim=dim, page=page, dtype=dtype, seed=41)
    small = s["key_cache"].shape[0]
    more = (2**31 + 2**20) // (4 * page * dim) + 1
    long = {name: torch.empty(more + small, 4, page, dim, dtype=dtype, device=DEV) for name in ("key_cache", "value_cache")}
    for name, cache in long.items():
        assert cache[:more].numel() > 2**31
        cache[more:].copy_(s[name])
    q = s.pop("q")
    tables = torch.where(s["block_tables"] >= 0, s["block_tables"] + more, s["block_tables"])
    for hints in ({}, dict(max_shared=1 << 30)):
        want = kernels.attention_shared(q, q.stride(0), **s, **sizes, **hints)
        check_attention(want, dict(s, q=q), **sizes)
        got = kernels.attention_shared(q, q.stride(0), **(s | long | dict(block_tables=tables)), **sizes, **hints)
        assert torch.equal(got, want)


def test_rules_on_the_last_rows_of_many():
    from rules_helpers import check_rules
    from test_logit_rules_gpu import made
    from tinyvllm_b200.ops import kernels

    vocab, rows = 150000, 2**31 // 150000 + 40
    few, rules = made(30, vocab, 40, biases=8, seed=42)
    logits = torch.empty(rows, vocab, device=DEV)
    logits[-30:] = few
    slots = torch.full((rows,), -1, dtype=torch.int32, device=DEV)
    slots[-30:] = rules["slots"]
    assert (rows - 30) * vocab > 2**31
    kernels.logit_rules(logits, out=logits, **dict(rules, slots=slots))
    check_rules(logits[-30:], few, **rules)


@pytest.mark.parametrize("n", [32768, 32761])
def test_adapters_on_the_last_rows_of_many(n):
    """A product of more than 2^31 results (the last rows' in 64 bits)."""
    from test_adapters_gpu import adapted, check, made

    m = 2**31 // n + 100
    s = made(m, 8, n, 8, 3)
    got = adapted(**s)
    last = slice(m - 90, m)
    assert (m - 90) * n > 2**31
    check(got[last], s | dict(x=s["x"][last], ids=s["ids"][last]))
    check(got[:90], s | dict(x=s["x"][:90], ids=s["ids"][:90]))


@pytest.mark.parametrize("rank", [64, 256])
def test_adapters_of_many(rank):
    """More than 2^31 elements of A and of B: the last adapters."""
    from test_adapters_gpu import BF16, adapted, check, made

    count = 2**31 // (4096 * rank) + 8
    down, up = torch.empty(count, rank, 4096, dtype=BF16, device=DEV), torch.empty(count, 4096, rank, dtype=BF16, device=DEV)
    assert down[:-4].numel() > 2**31 and up[:-4].numel() > 2**31
    for m in (5, 100, 600):
        s = made(m, 4096, 4096, rank, 4, seed=m)
        down[-4:], up[-4:] = s["down"], s["up"]
        scales = torch.zeros(count, device=DEV)
        scales[-4:] = s["scales"]
        ids = torch.where(s["ids"] >= 0, s["ids"] + count - 4, s["ids"])
        check(adapted(**(s | dict(down=down, up=up, scales=scales, ids=ids))), s)
