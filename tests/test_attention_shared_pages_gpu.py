"""Attention over keys in common for every page size that tensor-map copies take (8 to 128) and others, at every head size."""

import pytest
import torch

from shared_helpers import check_attention, made

pytestmark = pytest.mark.gpu
DEV = "cuda"
HINTS = ({}, dict(max_shared=1 << 30))                 # by themselves, and read together
PAGES = [8, 16, 32, 64, 128]
HEADS = [dict(num_q=4, num_kv=2, dim=64), dict(num_q=6, num_kv=2, dim=128), dict(num_q=4, num_kv=2, dim=256)]


def shared(s, sizes, **more):
    from tinyvllm_b200.ops import kernels

    s = dict(s)
    q = s.pop("q")
    return kernels.attention_shared(q, q.stride(0), **s, **sizes, **more)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("page", PAGES + [1, 24, 48, 256])
def test_lengths_inside_pages(page, heads):
    """Shared lengths that end inside a page, at its ends, and behind one key."""
    for length in (1, page - 1, page, page + 1, 3 * page + page // 2, 400, 513):
        s, sizes = made([(length, [1, 3, 30, 2 * page + 5]), (2 * length, [7, 130])], page=page, seed=length + page, **heads)
        for hints in HINTS:
            got = shared(s, sizes, **hints)
            check_attention(got, s, **sizes)
            assert torch.equal(shared(s, sizes, **hints), got)


@pytest.mark.parametrize("heads", [dict(num_q=8, num_kv=1, dim=64), dict(num_q=8, num_kv=1, dim=128), dict(num_q=8, num_kv=2, dim=256)])
@pytest.mark.parametrize("page", PAGES)
def test_many_query_rows_and_members_that_end_early(page, heads):
    own = [[7, 40, -3, 100, 1, 2, -90, 33][i % 8] for i in range(20)]
    s, sizes = made([(300, own), (1030, own[:3])], page=page, padding=(4, 9), seed=page, **heads)
    for hints in HINTS:
        check_attention(shared(s, sizes, **hints), s, **sizes)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("page", PAGES)
def test_what_pages_hold_behind_the_last_key_is_of_no_account(page, heads, dtype):
    s, sizes = made([(page + 5, [3, 20]), (170, [1, 9]), (64, [1])], page=page, dtype=dtype, seed=7, **heads)
    wants = [shared(s, sizes, **hints) for hints in HINTS]
    used = torch.zeros(s["key_cache"].shape[0], page, dtype=torch.bool)
    for t in range(s["positions"].shape[0]):
        for position in range(int(s["positions"][t]) + 1):
            used[int(s["block_tables"][int(s["token_row"][t]), position // page]), position % page] = True
    for cache in ("key_cache", "value_cache"):
        s[cache].masked_fill_(~used[:, None, :, None].to(DEV), float("nan"))
    for hints, want in zip(HINTS, wants):
        check_attention(want, {name: t.nan_to_num() if name.endswith("cache") else t for name, t in s.items()}, **sizes)
        assert torch.equal(shared(s, sizes, **hints), want)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("page", PAGES)
def test_pages_that_are_none_are_not_seen(page, heads):
    s, sizes = made([(5 * page, [page + 3, 30]), (4 * page, [20])], page=page, seed=8, **heads)
    s["block_tables"][0, 2] = s["block_tables"][1, 2] = -1              # of the shared keys, for both
    s["block_tables"][1, 5] = s["key_cache"].shape[0]                   # of its own
    s["block_tables"][2] = -7                                           # all of them: zeros
    two = {name: s[name][:2] for name in ("q", "token_row", "positions")}
    for hints in HINTS:
        got = shared(s, sizes, **hints)
        assert (got[2] == 0).all()
        check_attention(got[:2], dict(s, **two), **sizes)
