"""Groups whose starts fall back, overlap or lie outside the tokens: every token stands in one group at most, and gets what plain
attention gives it."""

import pytest
import torch

from shared_helpers import check_attention, made

pytestmark = pytest.mark.gpu


def settled(starts):
    """The groups as they count: no start below an earlier one."""
    out = []
    for start in starts:
        out.append(max([start] + out[-1:]))
    return out


def calls(s, sizes, starts, lens):
    from tinyvllm_b200.ops import kernels

    s = dict(s)
    q = s.pop("q")
    s["group_starts"] = torch.tensor(starts, dtype=torch.int32, device=q.device)
    s["shared_lens"] = torch.tensor(lens, dtype=torch.int32, device=q.device)
    for hints in ({}, dict(max_shared=1 << 30)):
        yield kernels.attention_shared(q, q.stride(0), **s, **sizes, **hints)


# (heads; head size 256 with many members has the tiles of 64 rows)
HEADS = [dict(num_q=4, num_kv=2, dim=64), dict(num_q=4, num_kv=2, dim=128), dict(num_q=2, num_kv=2, dim=256)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("starts, lens", [
    ([0, 5, 2, 4, 9], [80, 48, 32, 64]),               # falls back in the middle
    ([0, 5, 0, 5, 0, 9], [80, 16, 64, 16, 64]),        # the same tokens named again and again
    ([5, 0, 9, 2], [7, 64, 500]),                      # the first start is the largest of the first three
    ([-7, 5, -100, 2**31 - 1], [80, 500, 64]),         # outside the tokens
    ([9, 0, 0], [80, 80]),                             # none
])
def test_starts_that_fall(starts, lens, heads, dtype):
    s, sizes = made([(80, [5, 17, 1, 40, 9]), (64, [3, 2, 70, 8])], dtype=dtype, seed=31, **heads)
    ends = settled(starts)
    for got in calls(s, sizes, starts, lens):
        check_attention(got, s, **sizes)
    # the same bits as with the groups written down as they count
    for got, want in zip(calls(s, sizes, starts, lens), calls(s, sizes, ends, lens)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_fall_in_one_batch_of_groups_counts_in_the_next(dtype):
    """More than 32 groups; a warp looks at 32 at a time."""
    s, sizes = made([(48, [1 + i % 20 for i in range(60)])], dtype=dtype, seed=32)
    for starts in (list(range(0, 30)) + [50, 3] + list(range(4, 50)) + [60], list(range(31)) + [60] + list(range(31, 61))):
        for got in calls(s, sizes, starts, [48] * (len(starts) - 1)):
            check_attention(got, s, **sizes)
