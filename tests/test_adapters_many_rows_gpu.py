"""Adapters beside so many rows that they go 64 at a time: with tensor maps, and every way without them.  Sizes follow the package's
own thresholds, so that moving one takes no way out of the tests."""

import pytest
import torch

from test_adapters_gpu import BF16, DEV, adapted, check, made

pytestmark = pytest.mark.gpu


def rows_of(which):
    from tinyvllm_b200.ops import kernels

    few = kernels.ADAPTERS_FEW_ROWS
    return {"just": few + 1, "some": few + 108, "more": 4 * few + 3}[which]


ROWS = ["just", "some", "more"]


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("rows", ROWS[:2])
@pytest.mark.parametrize("rank", [1, 3, 4, 8, 15, 16, 17, 24, 40, 63, 64, 65, 72, 100, 128, 200, 256])
def test_ranks(rank, rows, dtype):
    for n in (264, 263):
        s = made(rows_of(rows), 320, n, rank, 5, dtype=dtype)
        got = adapted(**s)
        check(got, s)
        assert torch.equal(adapted(**s), got)


@pytest.mark.parametrize("rank", [8, 12, 40, 100])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("k, n", [(8, 8), (16, 16), (64, 136), (72, 1032), (2056, 250), (4096, 40), (1000, 1)])
def test_sizes(k, n, rows, rank):
    s = made(rows_of(rows), k, n, rank, 4)
    check(adapted(**s), s)


@pytest.mark.parametrize("rank", [4, 8, 16, 40, 100])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("k", [1, 7, 33, 130, 1031, 2052])
def test_a_k_that_is_no_multiple_of_8(k, rows, rank):
    """x and A value by value.  The projection is as the package's ``linear`` gives it (n is a multiple of 8): the adapter's part is held
    to 64 bits, and the sum is rounded once."""
    from tinyvllm_b200.ops import linear

    s = made(rows_of(rows), k, 136, rank, 4)
    got = adapted(**s)
    base = linear(s["x"], s["weight"])
    x, want, sizes = s["x"].double(), base.double(), torch.zeros(got.shape, dtype=torch.float64, device=DEV)
    for a in range(4):
        mine = (s["ids"] == a).nonzero()[:, 0]
        down, up, scale = s["down"][a].double(), s["up"][a].double(), s["scales"][a].double()
        want[mine] += scale * (x[mine] @ down.t()) @ up.t()
        sizes[mine] += scale.abs() * (x[mine].abs() @ down.abs().t()) @ up.abs().t()
    # float32 sums of k and rank products (2^-23 of their sizes a step), u in two parts, the last addition's rounding to float32
    bound = ((k + rank + 16) * 2.0**-23 + 2.0**-16) * sizes + 2.0**-23 * want.abs()
    assert ((got.double() - want).abs() <= bound + 2.0**-8 * (want.abs() + bound)).all()
    assert torch.equal(got[s["ids"] < 0], base[s["ids"] < 0])


@pytest.mark.parametrize("rank", [8, 20])
@pytest.mark.parametrize("rows", ROWS[1:])
def test_numbers_outside_and_no_scales(rows, rank):
    s = made(rows_of(rows), 128, 72, rank, 3)
    s["ids"][:4] = torch.tensor([3, -2**31, 2**31 - 1, -1], dtype=torch.int32)
    s["ids"][64:130] = -1                                               # a whole tile without
    s["scales"] = None
    check(adapted(**s), s)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("rank, n, k", [(16, 136, 128), (64, 136, 128), (100, 136, 128), (4, 136, 128), (16, 91, 128), (16, 136, 132)])
@pytest.mark.parametrize("rows", ROWS[1:])
def test_another_adapters_infinities_reach_nobody(rows, rank, n, k, dtype):
    m = rows_of(rows)
    s = made(m, k, n, rank, 4, dtype=dtype)
    want = adapted(**s)
    s["down"][2], s["up"][2] = float("inf"), float("nan")
    s["scales"][2] = float("nan")
    got = adapted(**s)
    mine = s["ids"] == 2
    assert torch.equal(got[~mine], want[~mine]) and not torch.isfinite(got[mine]).any()
    s = made(m, k, n, rank, 4, dtype=dtype)
    s["x"][m // 2] = float("nan")                                      # and a row's stay in the row
    s["x"][70] = float("inf")
    got = adapted(**s)
    others = (torch.arange(m, device=DEV) != m // 2) & (torch.arange(m, device=DEV) != 70)
    assert torch.isnan(got[m // 2]).all() and not torch.isfinite(got[70]).any() and torch.equal(got[others], want[others])


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("rank", [8, 12])
@pytest.mark.parametrize("pad, at", [(8, 8), (8, 3), (3, 0), (3, 1)])
def test_strided_operands_and_results(pad, at, rank, dtype):
    """Rows with a stride, on 16 bytes and off them."""
    m = rows_of("some")
    s = made(m, 192, 88, rank, 3, dtype=dtype)
    wide = torch.zeros(m, 192 + pad, dtype=dtype, device=DEV)
    wide[:, at % pad:at % pad + 192] = s["x"]
    memory = torch.full((m, 88 + 2 * pad), 3.0, dtype=dtype, device=DEV)
    got = adapted(**(s | dict(x=wide[:, at % pad:at % pad + 192])), out=memory[:, pad:pad + 88])
    check(got, s)
    assert got.data_ptr() == memory[:, pad:].data_ptr()
    assert (memory[:, :pad] == 3).all() and (memory[:, pad + 88:] == 3).all()


@pytest.mark.parametrize("rank", [4, 16, 100])
@pytest.mark.parametrize("rows", ROWS)
def test_float32_results_of_bfloat16_operands(rows, rank):
    s = made(rows_of(rows), 256, 120, rank, 3)
    got = adapted(**s, out_dtype=torch.float32)
    assert got.dtype == torch.float32
    check(got, s)


@pytest.mark.parametrize("rank", [8, 16, 72])
@pytest.mark.parametrize("adapters", [9, 33])
def test_more_rows_than_are_sorted(adapters, rank):
    """Many adapters in any order, in tiles of 64."""
    for m in (513, 1100):
        for n in (168, 91):
            s = made(m, 136, n, rank, adapters)
            check(adapted(**s), s)
