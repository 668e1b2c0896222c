"""Attention over keys in common against plain attention in 64 bits."""

import pytest
import torch

from shared_helpers import check_attention, made

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


def shared(s, sizes, **more):
    from tinyvllm_b200.ops import kernels

    s = dict(s)
    q = s.pop("q")
    return kernels.attention_shared(q, q.stride(0), **s, **sizes, **more)


# a hint by which even small groups are read together (by what the tables hold here each token would read by itself)
TOGETHER = dict(max_shared=1 << 30)


def check_both(s, sizes, **more):
    """Read together and by themselves, each twice; the former's result."""
    for hints in ({}, TOGETHER):
        got = shared(s, sizes, **hints, **more)
        assert got.dtype == s["q"].dtype
        check_attention(got, s, **sizes)
        assert torch.equal(shared(s, sizes, **hints, **more), got)       # bit for bit
    return got


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads", [(4, 2, 64), (2, 2, 128), (16, 2, 64), (3, 1, 256), (33, 1, 64), (8, 1, 128)])
def test_heads(heads, dtype):
    num_q, num_kv, dim = heads
    s, sizes = made([(96, [5, 17, 1]), (32, [40])], num_q=num_q, num_kv=num_kv, dim=dim, dtype=dtype, seed=num_q)
    check_both(s, sizes)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("length", [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 500, 1300])
def test_shared_lengths(length, dtype):
    """Also in the middle of a page, where every member has a page of its own from there on."""
    s, sizes = made([(length, [1, 3, 30, 70, 200])], dtype=dtype, seed=length)
    check_both(s, sizes)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("own", [1, 2, 64, 65, 300, 1000])
def test_own_lengths(own, dtype):
    s, sizes = made([(64, [own, 1, own]), (16, [own])], dtype=dtype, seed=own)
    check_both(s, sizes)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("page", [1, 4, 16, 48, 256])
def test_page_sizes(page, dtype):
    s, sizes = made([(100, [9, 33]), (256, [1, 2, 3])], page=page, dtype=dtype, seed=page)
    check_both(s, sizes)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_many_groups_some_empty_and_tokens_in_none(dtype):
    groups = [(16 * (1 + g % 5), [1 + (g * 7 + i) % 40 for i in range(g % 4)]) for g in range(70)]
    s, sizes = made(groups, dtype=dtype, seed=3)
    check_both(s, sizes)
    none = torch.zeros(1, dtype=torch.int32, device=DEV)
    check_both(dict(s, group_starts=none, shared_lens=none[:0]), sizes)
    # the first and the last groups' tokens stand in none
    check_both(dict(s, group_starts=s["group_starts"][20:41].contiguous(), shared_lens=s["shared_lens"][20:40].contiguous()), sizes)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_padding_and_a_group_whose_first_token_is_none(dtype):
    s, sizes = made([(80, [5, 6, 7, 8]), (48, [1, 2]), (32, [9])], dtype=dtype, padding=(0, 1, 3, 6), seed=9)
    out = torch.full_like(s["q"], 5.0)
    for hints in ({}, TOGETHER):
        got = shared(s, sizes, out=out, **hints)
        assert got is out
        check_attention(got, s, **sizes)
        assert (got[[0, 1, 3, 6]] == 0).all()
        out.fill_(5.0)
    s["token_row"][:] = -1
    for hints in ({}, TOGETHER, dict(max_own=128, max_shared=0)):
        assert (shared(s, sizes, **hints) == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_members_that_end_before_the_shared_keys_do(dtype):
    """A group's length that not every member reaches: those read what they have by themselves, as plain attention does."""
    s, sizes = made([(256, [0, 4, -100, -255, 30]), (64, [-3, -60])], dtype=dtype, seed=12)
    check_both(s, sizes)


@pytest.mark.parametrize("heads", [(8, 4), (16, 1), (2, 2)])
@pytest.mark.parametrize("members", [1, 4, 8, 9, 20])
def test_head_size_256_with_few_and_more_query_rows(members, heads):
    """Up to 16 rows a group and more; a length in the middle of a page, members that end before it, padding, a page that is none."""
    own = [[7, 40, -3, 100, 1, 2, -90, 33][i % 8] for i in range(members)]
    s, sizes = made([(312, own), (1056, own[::-1]), (64, own[:1])], num_q=heads[0], num_kv=heads[1], dim=256, padding=(members // 2,), seed=members)
    check_both(s, sizes)
    s["block_tables"][:members, 5] = -1
    s["block_tables"][-1, 1] = s["key_cache"].shape[0]
    for hints in ({}, TOGETHER):
        check_attention(shared(s, sizes, **hints), s, **sizes)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_several_tokens_of_a_request(dtype):
    s, sizes = made([(128, [5, 9, 40]), (16, [7])], tokens_of=5, dtype=dtype, seed=21)
    check_both(s, sizes)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_hints_that_are_wrong_change_rounding_only(dtype):
    s, sizes = made([(640, [5, 170, 300]), (320, [40])], dtype=dtype, seed=5)
    for hints in (dict(max_shared=0, max_own=0), dict(max_shared=1, max_own=1), dict(max_shared=10**9, max_own=10**9),
                  dict(max_shared=640, max_own=300), dict(max_shared=10**9, max_own=0), dict(max_shared=0, max_own=10**9)):
        check_attention(shared(s, sizes, **hints), s, **sizes)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_what_pages_hold_behind_the_last_key_is_of_no_account(dtype):
    s, sizes = made([(40, [3, 20]), (16, [1])], dtype=dtype, seed=7)
    wants = [shared(s, sizes, **hints) for hints in ({}, TOGETHER)]
    page = 16
    used = torch.zeros(s["key_cache"].shape[0], page, dtype=torch.bool)
    for t in range(s["positions"].shape[0]):
        for position in range(int(s["positions"][t]) + 1):
            used[int(s["block_tables"][int(s["token_row"][t]), position // page]), position % page] = True
    for cache in ("key_cache", "value_cache"):
        s[cache].masked_fill_(~used[:, None, :, None].to(DEV), float("nan"))
    for hints, want in zip(({}, TOGETHER), wants):
        assert torch.equal(shared(s, sizes, **hints), want)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_pages_that_are_none_are_not_seen(dtype):
    s, sizes = made([(160, [50, 30]), (64, [20])], dtype=dtype, seed=8)
    s["block_tables"][0, 2] = s["block_tables"][1, 2] = -1              # of the shared keys, for both
    s["block_tables"][1, 10] = s["key_cache"].shape[0]                  # of its own
    s["block_tables"][2] = -7                                           # all of them: zeros
    two = {name: s[name][:2] for name in ("q", "token_row", "positions")}
    for hints in ({}, TOGETHER):
        got = shared(s, sizes, **hints)
        assert (got[2] == 0).all()
        check_attention(got[:2], dict(s, **two), **sizes)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_large_scores_and_a_row_of_nan(dtype):
    s, sizes = made([(192, [5, 40, 3])], dtype=dtype, seed=4)
    s["q"] *= 60.0                                                       # weights of one key nearly
    check_both(s, sizes)
    wants = [shared(s, sizes, **hints) for hints in ({}, TOGETHER)]
    s["q"][1] = float("nan")
    for hints, want in zip(({}, TOGETHER), wants):
        got = shared(s, sizes, **hints)
        assert torch.isnan(got[1]).all() and torch.equal(got[[0, 2]], want[[0, 2]])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strided_q_and_results(dtype):
    """q inside a packed projection, the result inside a larger tensor."""
    s, sizes = made([(48, [5, 40, 3])], dtype=dtype, seed=2)
    packed = torch.randn(3, 256 + 2 * 128, device=DEV).to(dtype)
    packed[:, :256] = s["q"]
    memory = torch.full((3, 300), 7.0, dtype=dtype, device=DEV)
    from tinyvllm_b200.ops import kernels

    rest = {name: t for name, t in s.items() if name != "q"}
    for hints in ({}, TOGETHER):
        got = kernels.attention_shared(packed, packed.stride(0), **rest, **sizes, out=memory[:, 20:276], **hints)
        check_attention(got, s, **sizes)
        assert (memory[:, :20] == 7).all() and (memory[:, 276:] == 7).all()
        memory[:, 20:276] = 0


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_cache_without_pages(dtype):
    s, sizes = made([(48, [5, 2])], dtype=dtype)
    for cache in ("key_cache", "value_cache"):
        s[cache] = s[cache][:0]
    for hints in ({}, TOGETHER):
        assert (shared(s, sizes, **hints) == 0).all()


def test_no_tokens():
    s, sizes = made([(48, [5])])
    empty = {name: s[name][:0] for name in ("q", "token_row", "positions")}
    assert shared(dict(s, **empty), sizes).shape == (0, 256)


@pytest.mark.parametrize("heads", [(16, 8, 128), (32, 4, 128), (14, 2, 64), (12, 12, 64), (8, 4, 256)])
def test_a_decode_step_at_a_layers_size(heads):
    num_q, num_kv, dim = heads
    s, sizes = made([(1600, [5 + 9 * i for i in range(30)]), (333, [100, 7])], num_q=num_q, num_kv=num_kv, dim=dim, seed=1)
    check_attention(shared(s, sizes, max_shared=1600, max_own=300), s, **sizes)


def test_as_the_attention_without_groups_has_it():
    """The package's own attention over the same tables: float32, the bounds of both."""
    from shared_helpers import plain_attention
    from tinyvllm_b200.ops import kernels

    s, sizes = made([(208, [5, 50, 23])], dtype=F32, seed=6)
    rows = kernels.attention_rows(s["q"], s["q"].shape[1], s["key_cache"], s["value_cache"], s["block_tables"].clamp(min=0),
                                  s["token_row"], s["positions"], **{n: sizes[n] for n in ("num_q", "num_kv", "head_dim", "scale")},
                                  window=None)
    _, bound = plain_attention(s, **sizes)
    for hints in ({}, TOGETHER):
        assert ((shared(s, sizes, **hints) - rows).abs() <= 2 * bound).all()


@pytest.mark.parametrize("hints", [{}, TOGETHER], ids=["alone", "together"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_captured_twice_while_requests_grow(dtype, hints):
    """Two graphs of one step, replayed in turn with positions that move on, and an eager call on another stream beside them."""
    s, sizes = made([(96, [40, 41, 42]), (16, [40])], dtype=dtype, seed=14)
    last = s["positions"].clone()
    s["positions"] -= 39
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(stream):
        shared(s, sizes, **hints)
        stream.synchronize()
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                outs.append(shared(s, sizes, **hints))
            graphs.append(graph)
    torch.cuda.synchronize()
    for step in (0, 1, 17, 39):
        s["positions"].copy_(last - 39 + step)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            eager = shared(s, sizes, **hints)
        stream.synchronize()
        assert torch.equal(outs[0], eager) and torch.equal(outs[1], eager)
        check_attention(eager, s, **sizes)
