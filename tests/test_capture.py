"""Captures of the engine: no collection of cyclic garbage happens within one."""
import contextlib
import gc

import pytest
import torch

from orinfer_b200.utils.capture import recording


@pytest.mark.parametrize("collects", [True, False])
@pytest.mark.parametrize("raises", [True, False])
def test_the_collector_rests_and_goes_on(monkeypatch, collects, raises):
    seen = []

    @contextlib.contextmanager
    def graph(g):
        seen.append((g, gc.isenabled()))
        yield
    monkeypatch.setattr(torch.cuda, "graph", graph)
    before = gc.isenabled()
    try:
        (gc.enable if collects else gc.disable)()
        with pytest.raises(KeyError) if raises else contextlib.nullcontext():
            with recording("g"):
                assert not gc.isenabled()
                if raises:
                    raise KeyError
        assert gc.isenabled() == collects and seen == [("g", False)]
    finally:
        (gc.enable if before else gc.disable)()


@pytest.mark.gpu
def test_an_engine_captures_while_a_dead_one_awaits_its_collection(cuda, monkeypatch):
    """Each captured forward collects, as the collector may at any allocation, where it is at work."""
    from orinfer_b200.config import PRESETS, GraphMode, LoadOptions, SchedulerOptions
    from orinfer_b200.engine.engine import Engine
    from orinfer_b200.models.runner import ModelRunner
    from orinfer_b200.models.weights import random_model
    w = random_model(PRESETS["tiny"], seed=0).to(cuda)
    make = lambda: Engine(w, load=LoadOptions(cuda_graph=GraphMode.DECODE_ONLY), kv_pages=40, max_context=1024,
                          sched=SchedulerOptions(max_active=4, prefill_chunk=64))
    prompt = list(range(1, 100))
    dead = make()
    dead.itself = dead                               # only a collection finds it
    want = dead.generate([prompt], max_new=8)[0]
    assert dead.stats.graph_captures >= 1
    ours, captured = ModelRunner.greedy, []

    def greedy(self, *args, **kw):
        if torch.cuda.is_current_stream_capturing():
            captured.append(gc.isenabled())
            if gc.isenabled():
                gc.collect()
        return ours(self, *args, **kw)
    monkeypatch.setattr(ModelRunner, "greedy", greedy)
    eng = make()
    assert gc.isenabled()
    del dead
    assert eng.generate([prompt], max_new=8)[0] == want
    assert captured and not any(captured) and eng.stats.graph_captures >= 1 and gc.isenabled()
