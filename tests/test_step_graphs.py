"""Steps that replay captured graphs, without a GPU: what is replayed is not run again."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from pylon_b200.engine import graphs as graphs_module
from pylon_b200.engine.graphs import StepGraphs
from pylon_b200.engine.step import StepEntry, StepFunction


class Request:
    request_id, length, slot = "a", 0, 0


class Cache:
    def __init__(self):
        self.log = []

    def prepare(self, batch):
        self.log.append("prepare")

    def commit(self, request):
        self.log.append("commit")

    def save_state(self, requests):
        self.log.append("save")


@pytest.mark.parametrize("want", [(), (31,)])
def test_a_portion_that_is_replayed_does_not_run_again(want, monkeypatch):
    """A middle portion of a prompt wants no logits: that it returns none does not say that it had no graph."""
    eager, replayed = [], []
    function = StepFunction.__new__(StepFunction)
    function.cache, function.evicts = Cache(), False
    function.validate = lambda entries: None
    function.fill_padded = lambda *arguments: None
    function.sampled_source = lambda entries: None
    function._run_eager = lambda entries: eager.append(entries)
    graphs = StepGraphs.__new__(StepGraphs)
    graphs.step_function, graphs.cache, graphs.pad_steps, graphs.failed = function, function.cache, True, set()
    logits = torch.zeros(1, 5)
    graphs.captured_padded = {(0, 1, 32): SimpleNamespace(layout=SimpleNamespace(total=4))}
    graphs._replay = lambda captured, host, kind, sampled: replayed.append(kind) or logits
    monkeypatch.setattr(graphs_module, "torch", SimpleNamespace(empty=lambda total, **options: torch.empty(total, dtype=torch.int32), int32=torch.int32))
    function.graphs = graphs
    got = function([StepEntry(Request(), list(range(32)), want)])
    assert replayed == ["padded"] and eager == [] and function.cache.log == ["prepare", "commit"]
    assert (got is None) == (want == ())
    # a step without a graph runs eagerly, once
    graphs.captured_padded, graphs.seen_padded, graphs.capture_at_once = {}, {}, False
    function([StepEntry(Request(), list(range(32)), want)])
    assert len(eager) == 1 and replayed == ["padded"]


def test_a_capture_that_fails_half_way_puts_states_back(monkeypatch):
    """The step runs eagerly after that: what the failed run had advanced already must not be advanced again."""
    cache = Cache()
    cache.save_state = lambda requests: cache.log.append("save") or ["saved"]
    cache.restore_state = lambda saved: cache.log.append(("restore", saved))

    def forward(step, caches):
        cache.log.append("forward")
        raise RuntimeError("no memory")

    graphs = StepGraphs.__new__(StepGraphs)
    graphs.cache, graphs.failed, graphs.device, graphs.pool = cache, set(), None, None
    graphs.step_function = SimpleNamespace(model=SimpleNamespace(forward=forward))
    monkeypatch.setattr(graphs_module, "torch", SimpleNamespace(cuda=SimpleNamespace(synchronize=lambda device: None)))
    assert graphs._capture("key", None, [], None, None, []) is None
    assert cache.log == ["save", "forward", ("restore", ["saved"])] and graphs.failed == {"key"}
