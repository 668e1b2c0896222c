"""Adapters with infinite weights, or whose x A^T is infinite or nearly so: the results are those of the definition, infinities with
their signs and NaN where it has NaN, in the rows of that adapter alone."""

import pytest
import torch

from test_adapters_gpu import BF16, DEV, adapted, made

pytestmark = pytest.mark.gpu
F32 = torch.float32
# rows, adapters, rank, n, types of the operands and the result: rows as they lie, sorted, 64 at a time (with tensor maps and without)
WAYS = [(5, 4, 16, 136, BF16, BF16), (60, 4, 9, 136, BF16, F32), (60, 4, 4, 91, BF16, BF16), (100, 12, 16, 136, BF16, BF16),
        (100, 12, 16, 91, BF16, BF16), (300, 4, 16, 136, BF16, BF16), (300, 4, 64, 200, BF16, BF16), (300, 4, 100, 136, BF16, BF16),
        (300, 4, 4, 136, BF16, BF16), (300, 4, 16, 91, BF16, BF16), (300, 4, 24, 136, BF16, F32), (300, 4, 8, 136, F32, F32),
        (40, 4, 8, 91, F32, F32)]


def plain(s):
    """(result, size of the products) in 64 bits."""
    wide = {name: t.double() for name, t in s.items() if name != "ids"}
    want, sizes = wide["x"] @ wide["weight"].t(), wide["x"].abs() @ wide["weight"].abs().t()
    for a in range(wide["down"].shape[0]):
        rows = (s["ids"] == a).nonzero()[:, 0]
        u = wide["scales"][a] * (wide["x"][rows] @ wide["down"][a].t())
        # (written out: what a library does with infinities is its own affair)
        want[rows] += (u[:, None, :] * wide["up"][a][None]).sum(-1)
        sizes[rows] += wide["scales"][a].abs() * (wide["x"][rows].abs() @ wide["down"][a].abs().t()) @ wide["up"][a].abs().t()
    return want, sizes


def check(got, s):
    want, sizes = plain(s)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    infinite = torch.isinf(want)
    assert torch.equal(torch.isinf(got), infinite) and torch.equal(got[infinite].double(), want[infinite])
    finite = torch.isfinite(want)
    # sums in float32, u in two parts, two roundings of a bfloat16 result at most: the bounds of the finite cases
    k, rank, half = s["x"].shape[1], s["down"].shape[1], 2.0**-8 if got.dtype == BF16 else 2.0**-24
    bound = ((k + rank + 24) * 2.0**-23 + 2.0**-16) * sizes
    base = (s["x"].double() @ s["weight"].double().t()).abs()
    bound = (bound + half * (base + bound) + half * (want.abs() + bound))[finite]
    assert ((got.double() - want).abs()[finite] <= bound).all()
    return want


@pytest.mark.parametrize("m, adapters, rank, n, dtype, out_dtype", WAYS)
def test_an_infinite_weight(m, adapters, rank, n, dtype, out_dtype):
    s = made(m, 128, n, rank, adapters, dtype=dtype, seed=3)
    s["ids"][:2] = torch.tensor([1, 2], dtype=torch.int32)
    s["up"][1, 5, rank // 2] = float("inf")              # of B: one column
    s["up"][1, n - 1, 0] = float("-inf")
    s["down"][2, rank - 1, 7] = float("inf")             # of A: u of one rank
    want = check(adapted(**s, out_dtype=out_dtype), s)
    one, two = s["ids"] == 1, s["ids"] == 2
    assert torch.isinf(want[one][:, [5, n - 1]]).all() and torch.isinf(want[two]).all()
    assert torch.isfinite(want[~(one | two)]).all() and torch.isinf(want[one]).sum() == 2 * one.sum()


@pytest.mark.parametrize("m, adapters, rank, n, dtype, out_dtype", WAYS)
def test_zeros_beside_infinities_are_nan_as_in_the_definition(m, adapters, rank, n, dtype, out_dtype):
    s = made(m, 128, n, rank, adapters, dtype=dtype, seed=4)
    s["ids"][:] = torch.arange(m) % 2
    s["x"][:, 3] = s["x"][:, 3].abs() + 1
    s["down"][1, 0, 3] = float("inf")                    # u of rank 0 is +-infinity by the scale's sign
    s["up"][1, 4, 0] = 0.0                               # times 0
    s["up"][1, 6:8, 0] = torch.tensor([1.0, -1.0], dtype=dtype)
    want = check(adapted(**s, out_dtype=out_dtype), s)
    mine = want[s["ids"] == 1]
    assert torch.isnan(mine[:, 4]).all() and torch.isinf(mine[:, 6:8]).all() and torch.isfinite(want[s["ids"] == 0]).all()


@pytest.mark.parametrize("m, adapters, rank, n, dtype, out_dtype", WAYS)
def test_a_u_that_bfloat16_would_round_to_infinity(m, adapters, rank, n, dtype, out_dtype):
    """3.4e38 is finite in float32, and not in bfloat16; with a B of about 2^-120 the result is an ordinary number."""
    s = made(m, 128, n, rank, adapters, dtype=dtype, seed=5)
    s["x"].zero_()
    s["x"][:, 0] = 1.0
    s["down"].zero_()
    s["down"][:, 0, 0] = 2.0**127
    s["scales"][:] = 1.998                               # above 2 - 2^-8 = 1.99609, from where 2^127 of it rounds to infinity
    s["up"] *= 2.0**-120
    s["weight"].zero_()
    want = check(adapted(**s, out_dtype=out_dtype), s)
    assert torch.isfinite(want).all() and want.abs().max() > 1
