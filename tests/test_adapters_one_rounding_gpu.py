"""The projection beside adapters stays float32 where the result is float32, and where n is no multiple of 8: whatever k is."""

import pytest
import torch

from test_adapters_gpu import BF16, DEV, adapted, check, made

pytestmark = pytest.mark.gpu


def check_once(got, s):
    """One rounding of the sum.  Sums of k and of rank products in float32, 2^-23 of their sizes a step at most (twice what one
    rounding to nearest takes); u in two parts of 8 bits, 2^-16 of it; the result off by 2^-8 (float32: 2^-24) of itself."""
    wide = {name: t.double() for name, t in s.items() if name not in ("ids", "scales")}
    k, rank = wide["x"].shape[1], wide["down"].shape[1]
    want, sizes = wide["x"] @ wide["weight"].t(), wide["x"].abs() @ wide["weight"].abs().t()
    for a in range(wide["down"].shape[0]):
        rows = (s["ids"] == a).nonzero()[:, 0]
        scale = s["scales"][a].double()
        want[rows] += scale * (wide["x"][rows] @ wide["down"][a].t()) @ wide["up"][a].t()
        sizes[rows] += scale.abs() * (wide["x"][rows].abs() @ wide["down"][a].abs().t()) @ wide["up"][a].abs().t()
    bound = ((k + rank + 24) * 2.0**-23 + 2.0**-16) * sizes
    half = 2.0**-8 if got.dtype == BF16 else 2.0**-24
    off = (got.double() - want).abs() - bound - half * (want.abs() + bound)
    assert off.max().item() <= 0.0, f"{off.max().item():.3g} beyond the bound"


@pytest.mark.parametrize("adapters", [3, 20])
@pytest.mark.parametrize("m", [200, 256, 257, 600])
@pytest.mark.parametrize("k", [1, 7, 33, 1031, 2052])
def test_any_k(k, m, adapters):
    s = made(m, k, 91, 8, adapters)
    got = adapted(**s)
    assert got.dtype == BF16
    check_once(got, s)
    s = made(m, k, 96, 8, adapters)
    got = adapted(**s, out_dtype=torch.float32)
    assert got.dtype == torch.float32
    check_once(got, s)
    memory = torch.full((m, 100), 3.0, device=DEV)
    assert torch.equal(adapted(**s, out=memory[:, 2:98]), got)
    assert (memory[:, :2] == 3).all() and (memory[:, 98:] == 3).all()


@pytest.mark.parametrize("m", [5, 200, 300])
@pytest.mark.parametrize("k", [1, 40, 43])
def test_a_weight_that_lies_the_other_way(k, m):
    for n, more in ((91, {}), (96, dict(out_dtype=torch.float32))):
        s = made(m, k, n, 8, 3)
        s["weight"] = s["weight"].t().contiguous().t()
        assert k == 1 or s["weight"].stride(0) == 1
        check_once(adapted(**s, **more), s)


@pytest.mark.parametrize("m", [5, 300])
def test_one_column_of_x(m):
    """k = 1: the rows are single values, however far apart their (only) columns stand."""
    for n, more in ((91, {}), (96, dict(out_dtype=torch.float32)), (96, {})):
        s = made(m, 1, n, 8, 3)
        s["x"] = torch.zeros(4, m, dtype=BF16, device=DEV).t()[:, :1].copy_(s["x"])
        assert s["x"].stride() == (1, m)
        check(adapted(**s, **more), s)


def test_captured():
    s = made(300, 1031, 91, 8, 3)
    want = adapted(**s)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        adapted(**s)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = adapted(**s)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    check(got, s)
