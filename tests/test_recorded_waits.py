"""Bounded waits of the adapters' and the shared keys' kernels inside recorded steps: the replays pass through no Python, yet a wait
that ran out in any of them is reported.  The status functions are replaced here (no GPU)."""

import pytest
import torch

from tinyvllm_b200.ops import kernels

PARTS = ["adapters", "attention_shared"]


@pytest.fixture
def fake(monkeypatch):
    state = dict(capturing=False, reads=[], codes={part: 0 for part in PARTS})

    def status_of(part):
        def status():
            setattr(kernels, f"_{part}_unchecked", False)
            state["reads"].append(part)
            code, state["codes"][part] = state["codes"][part], 0
            return code
        return status

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capturing"])
    for name in ("_gemm_tc_unchecked", "_attention_tc_unchecked", *(f"_{part}_{what}" for part in PARTS for what in ("unchecked", "captured"))):
        monkeypatch.setattr(kernels, name, False)
    for part in PARTS:
        monkeypatch.setattr(kernels, f"{part}_status", status_of(part))
    return state


@pytest.mark.parametrize("part", PARTS)
def test_an_eager_launch_is_checked_once(fake, part):
    kernels.check_finished_launches()
    assert fake["reads"] == []
    getattr(kernels, f"_note_{part}_launch")(1)
    kernels.check_finished_launches()
    kernels.check_finished_launches()
    assert fake["reads"] == [part]


@pytest.mark.parametrize("part", PARTS)
def test_every_replay_of_a_recorded_launch_is_checked(fake, part):
    fake["capturing"] = True
    getattr(kernels, f"_note_{part}_launch")(1)
    fake["capturing"] = False
    for _ in range(3):                                     # replays
        kernels.check_finished_launches()
    assert fake["reads"] == [part] * 3
    fake["codes"][part] = 5                                # a wait of the next one gives up
    with pytest.raises(kernels.KernelError, match=f"{'add_' if part == 'adapters' else ''}{part}.*code 5"):
        kernels.check_finished_launches()
    getattr(kernels, f"_note_{part}_launch")(1)             # an eager launch in between changes nothing
    kernels.check_finished_launches()
    kernels.check_finished_launches()
    assert fake["reads"] == [part] * 6


@pytest.mark.gpu
@pytest.mark.parametrize("part", PARTS)
def test_a_recorded_call_is_still_checked_at_its_second_replay(part, monkeypatch):
    """The calls themselves; the code is put into the reader, no wait runs out."""
    from shared_helpers import made
    from tinyvllm_b200.ops import linear_adapted

    device, bf16 = "cuda", torch.bfloat16
    if part == "adapters":
        def call():
            return linear_adapted(torch.ones(300, 64, dtype=bf16, device=device), torch.ones(64, 64, dtype=bf16, device=device),
                                  torch.ones(2, 8, 64, dtype=bf16, device=device), torch.ones(2, 64, 8, dtype=bf16, device=device),
                                  torch.zeros(300, dtype=torch.int32, device=device))
    else:
        s, sizes = made([(48, [5, 40])])
        q = s.pop("q")

        def call():
            return kernels.attention_shared(q, q.stride(0), **s, **sizes)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call()
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        kernels.check_finished_launches()
    read = getattr(kernels, f"{part}_status")
    assert read() == 0
    graph.replay()
    torch.cuda.synchronize()
    monkeypatch.setattr(kernels, f"{part}_status", lambda: read() or 5)
    with pytest.raises(kernels.KernelError, match="code 5"):
        kernels.check_finished_launches()
