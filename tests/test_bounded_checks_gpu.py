"""Requests with a bounded cache when something goes wrong: what is held afterwards is what was held."""
import pytest
import torch

from test_bounded_requests_gpu import make, text  # noqa: F401

pytestmark = pytest.mark.gpu


def state(pool):
    kv = pool.runner.kv
    return [t.clone() for t in (pool.table, pool.lens, pool.refs, pool.weights)], dict(pool._len), \
        {s: list(t) for s, t in pool.text.items()}, [t.clone() for t in (*kv.k, *kv.v, *kv.ks, *kv.vs)]


def same(a, b, cache=True):
    return all(torch.equal(x, y) for x, y in zip(a[0], b[0])) and a[1:3] == b[1:3] and (
        not cache or all(torch.equal(x, y) for x, y in zip(a[3], b[3])))


def failing(monkeypatch, runner, method, at):
    """Call number ``at`` of a method raises, behind what it has done, once."""
    ours, calls = getattr(runner, method), []

    def call(*args, **kw):
        got = ours(*args, **kw)
        calls.append(1)
        if len(calls) == at:
            raise MemoryError("no memory")
        return got
    monkeypatch.setattr(runner, method, call)


@pytest.mark.parametrize("preset", ["tiny", "tiny-moe"])
@pytest.mark.parametrize("method,at", [("logits", 1), ("_attention_core", 1), ("_attention_core", 2)])
def test_a_step_that_raises_leaves_every_request_as_it_was(make, monkeypatch, preset, method, at):  # noqa: F811
    """At the end of a page, within one and at the bound; the step that follows is that of a pool in which
    nothing happened, bit for bit."""
    pools = [make(preset), make(preset)]
    cfg = pools[0].runner.cfg
    prompts = [text(n, cfg.vocab, n) for n in (128, 77, 300)]
    slots = [[pool.add(p) for p in prompts] for pool in pools]
    assert slots[0] == slots[1]
    tokens = dict(zip(slots[0], (5, 6, 7)))
    for pool in pools:
        pool.cut([slots[0][2]])
    before = state(pools[0])
    failing(monkeypatch, pools[0].runner, method, at)
    with pytest.raises(MemoryError):
        pools[0].step(tokens)
    assert same(state(pools[0]), before, cache=False)
    monkeypatch.undo()
    assert torch.equal(*(pool.step(tokens) for pool in pools))
    assert same(state(pools[0]), state(pools[1]), cache=False)
    for s in slots[0]:
        pools[0].drop(s)
    assert pools[0].held == 0 and bool((pools[0].weights == 0).all())


def test_a_step_of_recurrent_layers_that_raises_gives_its_requests_up(make, monkeypatch):  # noqa: F811
    """Their states have moved on; another request stays, and the slots serve new ones."""
    pool, fresh = make("tiny-hybrid"), make("tiny-hybrid")
    cfg = pool.runner.cfg
    other, *slots = [pool.add(text(n, cfg.vocab, n)) for n in (50, 128, 77)]
    assert fresh.add(text(50, cfg.vocab, 50)) == other
    failing(monkeypatch, pool.runner, "_gdn_block", 1)
    with pytest.raises(MemoryError):
        pool.step(dict.fromkeys(slots, 3))
    monkeypatch.undo()
    assert list(pool.text) == [other] and pool.held == 1 and len(pool._free) == 3
    assert same(state(pool), state(fresh), cache=False)
    again = [p.add(text(128, cfg.vocab, 128)) for p in (pool, fresh)]
    assert torch.equal(*(p.logits[s] for p, s in zip((pool, fresh), again)))
    tokens = [{other: 9, s: 4} for s in again]
    assert torch.equal(*(p.step(t) for p, t in zip((pool, fresh), tokens)))


def test_a_prompt_that_raises_takes_nothing(make, monkeypatch):  # noqa: F811
    pool = make("tiny")
    cfg = pool.runner.cfg
    pool.add(text(300, cfg.vocab))
    before = state(pool)
    for method, at in (("logits", 1), ("logits", 2), ("_attention_core", 3)):
        failing(monkeypatch, pool.runner, method, at)
        with pytest.raises(MemoryError):
            pool.add(text(500, cfg.vocab, 1))
        monkeypatch.undo()
        after = state(pool)
        assert same(after, before, cache=False) and len(pool._free) == 3
