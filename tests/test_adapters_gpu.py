"""The projection with adapters against its definition in 64 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def adapted(*args, **kwargs):
    from tinyvllm_b200.ops import linear_adapted

    return linear_adapted(*args, **kwargs)


def made(m, k, n, rank, adapters, *, dtype=BF16, seed=0, kind="mixed"):
    gen = torch.Generator().manual_seed(seed + 7 * m + k + n)
    ids = {"mixed": torch.randint(-1, adapters, (m,), generator=gen), "one": torch.full((m,), adapters - 1),
           "none": torch.full((m,), -1), "spans": torch.arange(m) * adapters // max(m, 1)}[kind]
    state = dict(x=torch.randn(m, k, generator=gen).to(dtype), weight=(torch.randn(n, k, generator=gen) * k**-0.5).to(dtype),
                 down=(torch.randn(adapters, rank, k, generator=gen) * k**-0.5).to(dtype),
                 up=(torch.randn(adapters, n, rank, generator=gen) * rank**-0.5).to(dtype), ids=ids.to(torch.int32),
                 scales=torch.rand(adapters, generator=gen) * 4 - 2)
    return {name: t.to(DEV) for name, t in state.items()}


def check(got, s):
    """Sums of k products in float32, however ordered, are off by at most about k 2^-23 of the products' sizes (each
    addition by 2^-24 of the sum, twice that where the tensor cores cut instead of rounding; three bfloat16 parts of a
    float32 operand leave less than 8 such steps); u passes in two parts on (2^-16 of it); a bfloat16 result is rounded
    once as the projection and once at the end, by 2^-8 of itself each."""
    x, w, down, up = (s[name].double() for name in ("x", "weight", "down", "up"))
    ids, scales = s["ids"].long(), s["scales"].double() if s["scales"] is not None else torch.ones(down.shape[0], device=DEV).double()
    k, rank, step = x.shape[1], down.shape[1], 2.0**-23
    base = x @ w.t()
    bound = (k + 8) * step * (x.abs() @ w.abs().t())
    want = base.clone()
    for a in range(down.shape[0]):
        rows = (ids == a).nonzero()[:, 0]
        want[rows] += scales[a] * (x[rows] @ down[a].t()) @ up[a].t()
        sizes = scales[a].abs() * (x[rows].abs() @ down[a].abs().t()) @ up[a].abs().t()
        bound[rows] += ((k + rank + 16) * step + 2.0**-16) * sizes
    half = 2.0**-8 if got.dtype == BF16 else 2.0**-24
    bound += half * (base.abs() + bound)
    bound += half * (want.abs() + bound)
    assert got.shape == want.shape
    off = (got.double() - want).abs() - bound
    assert off.numel() == 0 or off.max().item() <= 0.0, f"{off.max().item():.3g} beyond the bound"


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 48, 128, 129, 200])
def test_rows(m, dtype):
    s = made(m, 256, 136, 16, 5, dtype=dtype)
    got = adapted(**s)
    assert got.dtype == dtype
    check(got, s)
    assert torch.equal(adapted(**s), got)                              # bit for bit
    if m > 1:
        from tinyvllm_b200.ops import linear

        bare = (s["ids"] < 0).nonzero()[:, 0]
        assert torch.equal(got[bare], linear(s["x"], s["weight"])[bare])


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("m", [9, 150])
@pytest.mark.parametrize("rank", [1, 3, 4, 8, 17, 24, 64, 100, 256])
def test_ranks(rank, m, dtype):
    s = made(m, 320, 264, rank, 3, dtype=dtype)
    check(adapted(**s), s)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("m", [5, 140])
@pytest.mark.parametrize("k, n", [(8, 8), (1, 1), (7, 5), (33, 31), (1000, 1), (64, 129), (2056, 250), (4096, 40)])
def test_sizes(k, n, m, dtype):
    s = made(m, k, n, 8, 4, dtype=dtype)
    check(adapted(**s), s)


@pytest.mark.parametrize("rank", [8, 16, 24, 64])
@pytest.mark.parametrize("m, k, n", [(129, 72, 8), (191, 8, 72), (300, 2056, 200), (1025, 520, 1032)])
def test_more_rows_with_tails_of_every_size(m, k, n, rank):
    s = made(m, k, n, rank, 6)
    check(adapted(**s), s)
    s["x"] = s["x"][:1].expand(m, k)                                   # one row for all
    check(adapted(**s), s)


@pytest.mark.parametrize("rank", [8, 40])
@pytest.mark.parametrize("adapters", [2, 8, 9, 60])
@pytest.mark.parametrize("m", [33, 128, 192, 193, 511, 512, 513])
def test_rows_in_any_order(m, adapters, rank):
    s = made(m, 200, 168, rank, adapters)
    got = adapted(**s)
    check(got, s)
    order = torch.randperm(m, generator=torch.Generator().manual_seed(m)).to(DEV)
    other = s | dict(x=s["x"][order], ids=s["ids"][order])
    check(adapted(**other), other)
    check(adapted(**other, out_dtype=torch.float32), other)


@pytest.mark.parametrize("rank", [4, 5, 16])
@pytest.mark.parametrize("adapters", [3, 40])
@pytest.mark.parametrize("m", [5, 100, 192, 193, 512, 600])
def test_widths_that_are_no_multiple_of_8_are_rounded_once(m, adapters, rank):
    """Every way the rows go, and rows without an adapter among them; the bound has one rounding to bfloat16."""
    s = made(m, 136, 171, rank, adapters)
    memory = torch.full((m, 180), 3.0, dtype=BF16, device=DEV)
    got = adapted(**s, out=memory[:, 5:176])
    check(got, s)
    wide = {name: t.double() for name, t in s.items() if name not in ("ids", "scales")}
    has = (s["ids"] >= 0)[:, None]
    rows = s["ids"].long().clamp(min=0)
    narrow = torch.einsum("tk,trk->tr", wide["x"], wide["down"][rows]) * s["scales"].double()[rows][:, None]
    want = wide["x"] @ wide["weight"].t() + torch.where(has, torch.einsum("tr,tnr->tn", narrow, wide["up"][rows]), 0.0)
    # sums of 136 products, then of up to 16: 2^-23 of some 12 + 4 times their size each, u in two parts; one rounding, 2^-8 of the result
    sizes = wide["x"].abs() @ wide["weight"].abs().t() + torch.where(has, torch.einsum(
        "tr,tnr->tn", torch.einsum("tk,trk->tr", wide["x"].abs(), wide["down"][rows].abs()) * s["scales"].double().abs()[rows][:, None],
        wide["up"][rows].abs()), 0.0)
    bound = ((136 + rank + 24) * 2.0**-23 + 2.0**-16) * sizes
    assert ((got.double() - want).abs() <= bound + 2.0**-8 * (want.abs() + bound)).all()
    assert (memory[:, :5] == 3).all() and (memory[:, 176:] == 3).all()


@pytest.mark.parametrize("kind", ["one", "none", "spans"])
@pytest.mark.parametrize("m", [20, 333])
def test_which_rows_have_which(kind, m):
    s = made(m, 128, 128, 8, 40, kind=kind)
    check(adapted(**s), s)


@pytest.mark.parametrize("rank", [4, 32])
@pytest.mark.parametrize("m", [64, 260])
def test_every_row_another_adapter(m, rank):
    s = made(m, 128, 96, rank, m)
    s["ids"] = torch.randperm(m, generator=torch.Generator().manual_seed(m)).to(torch.int32).to(DEV)
    check(adapted(**s), s)


@pytest.mark.parametrize("m", [6, 180])
def test_numbers_outside_and_no_scales(m):
    s = made(m, 128, 72, 8, 3)
    s["ids"][:4] = torch.tensor([3, -2**31, 2**31 - 1, -1], dtype=torch.int32)
    s["scales"] = None
    check(adapted(**s), s)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("m", [40, 170])
def test_another_adapters_infinities_reach_nobody(m, dtype):
    s = made(m, 128, 136, 16, 4, dtype=dtype)
    want = adapted(**s)
    s["down"][2], s["up"][2] = float("inf"), float("nan")
    s["scales"][2] = float("nan")
    got = adapted(**s)
    mine = s["ids"] == 2
    assert torch.equal(got[~mine], want[~mine]) and not torch.isfinite(got[mine]).any()
    s = made(m, 128, 136, 16, 4, dtype=dtype)
    s["x"][m // 2] = float("nan")                                      # and a row's stay in the row
    got = adapted(**s)
    others = torch.arange(m, device=DEV) != m // 2
    assert torch.isnan(got[m // 2]).all() and torch.equal(got[others], want[others])


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("m", [7, 150])
def test_strided_operands_and_results(m, dtype):
    for pad in (8, 3):
        s = made(m, 192, 88, 8, 3, dtype=dtype)
        wide = torch.zeros(m, 192 + pad, dtype=dtype, device=DEV)
        wide[:, :192] = s["x"]
        memory = torch.full((m, 88 + 2 * pad), 3.0, dtype=dtype, device=DEV)
        got = adapted(**(s | dict(x=wide[:, :192])), out=memory[:, pad:pad + 88])
        check(got, s)
        assert got.data_ptr() == memory[:, pad:].data_ptr()
        assert (memory[:, :pad] == 3).all() and (memory[:, pad + 88:] == 3).all()


@pytest.mark.parametrize("m", [1, 30, 150])
def test_float32_result_of_bfloat16_operands(m):
    s = made(m, 256, 120, 16, 3)
    got = adapted(**s, out_dtype=torch.float32)
    assert got.dtype == torch.float32
    check(got, s)


def test_no_rows():
    s = made(0, 64, 48, 8, 2)
    assert adapted(**s).shape == (0, 48)


def test_prompts_and_a_decode_step_at_a_layers_size():
    for m, rank in ((48, 16), (700, 64)):
        s = made(m, 1024, 4096, rank, 13)
        check(adapted(**s, weight_constant=True), s)


@pytest.mark.parametrize("m", [24, 300])
def test_captured_twice_and_on_another_stream(m):
    """Two graphs of the same call, replayed one after the other with inputs that change, and an eager call beside them."""
    s = made(m, 256, 200, 16, 4)
    wants = []
    for seed in range(3):
        wants.append(adapted(**(s | dict(x=made(m, 256, 200, 16, 4, seed=seed)["x"]))))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    x = s["x"].clone()
    with torch.cuda.stream(stream):
        adapted(**(s | dict(x=x)))
        stream.synchronize()
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                out = adapted(**(s | dict(x=x)))
            graphs.append(graph)
            outs.append(out)
    torch.cuda.synchronize()
    for seed in range(3):
        x.copy_(made(m, 256, 200, 16, 4, seed=seed)["x"])
        for graph, out in zip(graphs, outs):
            out.zero_()
            graph.replay()
        eager = adapted(**(s | dict(x=x)))
        assert torch.equal(outs[0], wants[seed]) and torch.equal(outs[1], wants[seed]) and torch.equal(eager, wants[seed])


def test_waits_of_many_rows_are_recorded():
    from tinyvllm_b200.ops import kernels

    s = made(700, 512, 264, 16, 3)
    adapted(**s)
    assert kernels._adapters_unchecked
    kernels.check_finished_launches()                                  # none ran out
    assert not kernels._adapters_unchecked and kernels.adapters_status() == 0
