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


def recurrent(runner):
    pools = getattr(runner, "_gdn", None)
    return [] if pools is None else [pools["state"].clone(), pools["hist"].clone()]


@pytest.mark.parametrize("preset", ["tiny", "tiny-hybrid"])
def test_a_packet_that_is_refused_changes_nothing(make, preset):  # noqa: F811
    """Whatever layer would refuse it: keys, values, recurrent states and weights stay as they were."""
    from orinfer_b200.models.runner import Packet
    from orinfer_b200.ops import native
    pool = make(preset)
    runner, i32, w = pool.runner, pool._i32, pool.weights
    slot = pool.add(text(100, runner.cfg.vocab))
    layers = list(w)
    last = lambda t: layers[:-1] + [t]
    single = lambda **kw: Packet(i32([1]), i32([slot]), i32([100]), pool.table, 1, 101,
                                 **{"weights": w, **kw})
    chunk = lambda **kw: Packet(i32([1] * 5), i32([slot] * 5), i32(list(range(100, 105))), pool.table, 5, 105,
                                chunks=i32([[0, 5, 100, slot]]), max_q_len=5, max_chunk_kv=105,
                                **{"weights": w, **kw})
    bad = [single(weights=layers[:-1]), chunk(weights=layers[:-1]), single(weights=[]),
           single(attend_pos=i32([100])), single(weigh_chunks=i32([[0, 1, 100, slot]])),
           chunk(weigh_chunks=i32([[0, 1, 100, slot]] * 513)),
           chunk(weigh_chunks=i32([[0, 1, 100, slot]]).long()),
           single(rope_pos=i32([100]).long()), single(rope_pos=i32([[100]])), single(rope_pos=i32([])),
           chunk(rope_pos=i32([100] * 4)), single(rope_pos=i32([100]).cpu()),
           single(rope_pos=i32([100]), mrope=i32([[100]] * 3))]
    for make_packet in (single, chunk):
        bad += [make_packet(weights=last(t)) for t in (
            layers[-1].double(), layers[-1][:-1], layers[-1][:, :-1], layers[-1].transpose(1, 2),
            layers[-1][..., ::2], layers[-1].cpu())]
    before = state(pool), recurrent(runner)
    for packet in bad:
        with pytest.raises((ValueError, native.KernelError)):
            runner.logits(packet)
        assert same(state(pool), before[0])
        assert all(torch.equal(a, b) for a, b in zip(recurrent(runner), before[1]))
    runner.logits(single())
    assert not same(state(pool), before[0])


def test_a_cut_of_slots_without_a_request_is_refused(make):  # noqa: F811
    pool = make("tiny")
    slot = pool.add(text(300, pool.runner.cfg.vocab))
    before = state(pool)
    for slots in ([slot, pool._free[0]], [9], [-1]):
        with pytest.raises(ValueError, match="holds no request"):
            pool.cut(slots)
        assert same(state(pool), before)
    pool.cut([slot, slot])
    assert pool._len == {slot: 150} and pool.lens[slot] == 150 and pool.held == 2
