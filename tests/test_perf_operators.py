"""The measured calls of perf/operators.py: ordered with the caller's stream."""

from __future__ import annotations

import pytest

from perf import operators


@pytest.fixture()
def own(monkeypatch):
    monkeypatch.setattr(operators, "own", True)
    operators._stream.cache_clear()
    operators._engine.cache_clear()
    yield
    operators._stream.cache_clear()
    operators._engine.cache_clear()


@pytest.mark.parametrize("idle", [False, True])
def test_a_run_waits_for_the_caller_and_the_caller_for_it(own, monkeypatch, idle):
    """On recorded calls: the run's stream waits for the current one before the
    run (unless that has nothing left to do), the current one for the run's
    after it, and the context's last run is taken in first."""
    import torch

    log = []

    class Event:
        def record(self, stream):
            self.of = stream.name

    class Stream:
        def __init__(self, name="side"):
            self.name, self.cuda_stream = name, name

        def query(self):
            return idle

        def wait_event(self, event):
            log.append((self.name, "waits for", event.of))

        def wait_stream(self, other):
            log.append((self.name, "waits for", other.name))

    class Context:
        def synchronize(self):
            log.append("synchronize")

        def run_async(self, stream):
            log.append(("run", stream))

    monkeypatch.setattr(torch.cuda, "Stream", Stream)
    monkeypatch.setattr(torch.cuda, "Event", Event)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: Stream("caller"))
    outputs = [object()]
    assert operators.run({"context": Context(), "outputs": outputs}) is outputs
    assert log[0] == "synchronize"
    assert log[1:] == [("side", "waits for", "caller")][idle:] + [("run", "side"), ("caller", "waits for", "side")]


@pytest.mark.gpu
@pytest.mark.parametrize("default_stream", [True, False])
@pytest.mark.parametrize("name", ["quantize-8x4096", "qgemm-8x12288x4096"])
def test_runs_read_and_are_read_in_stream_order(cuda, own, name, default_stream):
    """Inputs written late on the current stream, outputs copied right after
    the call and overwritten by the next one, with no synchronisation between."""
    import torch

    (case,) = [c for c in operators.listed() if c["name"] == name]
    state = operators.prepare(case, 1)
    others = [operators.prepare(case, seed) for seed in (2, 3)]
    torch.cuda.synchronize()
    wants = []
    for other in others:
        wants.append([t.clone() for t in operators.run(other)])
        torch.cuda.synchronize()
    operators.run(state)  # captured here, so that the runs below are launches only
    torch.cuda.synchronize()
    busy = torch.randn(8192, 8192, device="cuda", dtype=torch.float16)
    torch.cuda.synchronize()
    stream = torch.cuda.default_stream() if default_stream else torch.cuda.Stream()
    got = []
    with torch.cuda.stream(stream):
        for other in others:
            for _ in range(10):  # about 7 ms in front of the inputs
                busy @ busy
            for key, tensor in state["tensors"].items():
                tensor.copy_(other["tensors"][key])
            outputs = operators.run(state)
            got.append([t.clone() for t in outputs])
    torch.cuda.synchronize()
    for have, want in zip(got, wants):
        assert all(torch.equal(a, b) for a, b in zip(have, want))
