"""Requests with a bounded cache through the model: weights counted by prefill and decode, keys evicted,
positions kept, pages given back."""
import pytest
import torch

from orinfer_b200.config import PRESETS
from orinfer_b200.core import sampling as S
from orinfer_b200.models.weights import random_model
from orinfer_b200.ops import functional as F
from orinfer_b200.ref import eviction_ref as E

pytestmark = pytest.mark.gpu


@pytest.fixture
def make(cuda):
    from orinfer_b200.models.bounded import BoundedRequests
    from orinfer_b200.models.runner import KVPool, ModelRunner

    def make(preset, pages=24, slots=4, bound=300, keep=150, rows=256, **options):
        cfg = PRESETS[preset]
        runner = ModelRunner(random_model(cfg, seed=3).to(cuda), KVPool.allocate(cfg, pages, cuda),
                             max_rows=rows)
        return BoundedRequests(runner, slots, bound, keep, **options)
    return make


def text(n, vocab, seed=0):
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.parametrize("preset", ["tiny", "tiny-moe", "tiny-hybrid"])
def test_below_the_bound_nothing_differs_and_weights_add_up(make, preset):
    """Logits are those of packets that count nothing, bit for bit.  Every row gives each query head
    a weight of one: |score| <= sqrt(D) (max |norm weight|)^2 <= 32 here, in base-2 exponents 47,
    formed by D + 8 roundings in each of two passes: 2 (64 + 8) 2^-24 47 = 4e-4, and 2^-16 for the
    exponentials, reciprocals and sums of 600 terms."""
    from orinfer_b200.models.runner import KVPool, ModelRunner, Packet
    pool = make(preset, bound=700, keep=600)
    runner, cfg, i32 = pool.runner, pool.runner.cfg, pool._i32
    assert cfg.head_dim == 64
    plain = ModelRunner(runner.w, KVPool.allocate(cfg, 24, pool.device), max_rows=256)
    prompts = [text(n, cfg.vocab, n) for n in (300, 61, 128)]
    slots, table = [], pool.table.clone()
    for i, prompt in enumerate(prompts):
        slots.append(pool.add(prompt))
        table[slots[-1]] = torch.arange(1 + 6 * i, 7 + 6 * i)
        for at in range(0, len(prompt), 256):
            n = min(256, len(prompt) - at)
            p = Packet(i32(prompt[at:at + n]), i32([slots[-1]] * n), i32(list(range(at, at + n))),
                       table, n, at + n, torch.tensor([n - 1], device=pool.device),
                       chunks=i32([[0, n, at, slots[-1]]]), max_q_len=n, max_chunk_kv=at + n)
            want = plain.logits(p)[0]
        assert torch.equal(pool.logits[slots[-1]], want)
    for step in range(3):
        tokens = text(3, cfg.vocab, step)
        at = [len(p) + step for p in prompts]
        want = plain.logits(Packet(i32(tokens), i32(slots), i32(at), table, 3, max(at) + 1))
        assert torch.equal(pool.step(dict(zip(slots, tokens))), want)
    for lw in runner.w.layers:
        if lw.kind == "attn" and cfg.qk_norm:
            plus = 1.0 if cfg.zero_centered_norm else 0.0
            assert max(float((lw.q_norm.float() + plus).abs().max()),
                       float((lw.k_norm.float() + plus).abs().max())) <= 2
    assert cfg.qk_norm
    heads = cfg.q_heads // cfg.kv_heads
    for slot, prompt in zip(slots, prompts):
        n = len(prompt) + 3
        sums = pool.weights[:, slot].double()
        assert bool((sums[..., n:] == 0).all()) and bool((sums[..., :n] >= 0).all())
        assert float((sums.sum(2) / (n * heads) - 1).abs().max()) <= 5e-4
    assert bool((pool.weights[:, pool._free] == 0).all())


@pytest.mark.parametrize("preset,last_rows,first,recent", [("tiny", None, 4, 64), ("tiny-moe", 32, 0, 0),
                                                           ("tiny-hybrid", None, 1, 149)])
def test_requests_are_cut_as_the_host_law_says(make, monkeypatch, preset, last_rows, first, recent):
    """Every cut is that of the host statement, bit for bit; afterwards keys are written at the angle
    of their place in the text and nobody holds more than the bound."""
    pool = make(preset, first=first, recent=recent, last_rows=last_rows)
    cfg, cuts = pool.runner.cfg, []
    ours = F.evict_keys

    def checked(cache, table, lens, refs, weights, slots, keep, **options):
        n = cache.layers
        host = [t.cpu() for t in cache.tensors]
        parts = [host[i * n:(i + 1) * n] for i in range(4)]
        want = E.evict_keys(*parts, table.cpu(), lens.cpu(), refs.cpu(), weights.cpu(), slots.cpu(),
                            keep, first, recent)
        got = ours(cache, table, lens, refs, weights, slots, keep, **options)
        assert int(got[3]) == want[4] == 0
        for mine, law in zip((table, lens, refs, weights, *cache.tensors),
                             (*want[:4], *(t for part in parts for t in part))):
            assert torch.equal(mine.cpu(), law)
        cuts.append(slots.tolist())
        return got

    monkeypatch.setattr(F, "evict_keys", checked)
    prompts = [text(n, cfg.vocab, n) for n in (700, 90, 290)]
    slots = [pool.add(p) for p in prompts]
    assert len(cuts) == 3                                # 256 + 44, then 150 more each time
    options = [S.SamplingOptions(temperature=0.9, top_k=20, seed=i) for i in range(3)]
    drawn = pool.generate(slots, options, 30)
    assert [len(d) for d in drawn] == [30] * 3
    assert [pool.text[s] for s in slots] == [p + d for p, d in zip(prompts, drawn)]
    assert len(cuts) > 3 and slots[2] in cuts[-1]
    assert pool.lens.tolist() == [pool._len.get(s, 0) for s in range(4)]
    assert all(pool._len[s] <= 300 for s in slots)
    # the same text in a cache without a bound: the first layer's keys do not depend on what is seen
    if cfg.is_full_attention(0):
        from orinfer_b200.models.runner import KVPool, ModelRunner, Packet
        i32, whole = pool._i32, pool.text[slots[0]]
        plain = ModelRunner(pool.runner.w, KVPool.allocate(cfg, 8, pool.device), max_rows=1)
        at, place = len(whole) - 1, pool._len[slots[0]] - 1
        plain.logits(Packet(i32(whole[-1:]), i32([0]), i32([at]),
                            torch.arange(1, 8, device=pool.device, dtype=torch.int32)[None], 1, at + 1))
        mine = int(pool.table[slots[0], place // 128])
        assert torch.equal(pool.runner.kv.k[0][mine, place % 128], plain.kv.k[0][1 + at // 128, at % 128])
    for s in slots:
        pool.drop(s)
    assert pool.held == 0 and sorted(pool._free) == list(range(4))


@pytest.mark.parametrize("preset,cosine", [("tiny", 0.999), ("tiny-moe", 0.998)])
def test_a_step_behind_a_cut_is_that_of_the_plain_runner_on_the_same_cache(make, preset, cosine):
    """The cosines are those to which whole passes of the two runners are held elsewhere."""
    from orinfer_b200.models.runner import KVPool, Packet
    from orinfer_b200.models.torch_runner import TorchRunner
    pool = make(preset)
    cfg = pool.runner.cfg
    slots = [pool.add(text(n, cfg.vocab, n)) for n in (520, 300, 77)]
    cpu = TorchRunner(random_model(cfg, seed=3), KVPool.allocate(cfg, 24, "cpu"), 8)
    pool.step({s: 5 for s in slots})                     # cuts the second
    for mine, theirs in zip(pool.cache.tensors, [*cpu.kv.k, *cpu.kv.v, *cpu.kv.ks, *cpu.kv.vs]):
        theirs.copy_(mine.cpu())
    place, where, table = [pool._len[s] for s in slots], [len(pool.text[s]) for s in slots], pool.table
    assert place[0] < where[0] and place[1] == 151 and place[2] == where[2] == 78
    tokens = text(3, cfg.vocab, 1)
    got = pool.step(dict(zip(slots, tokens))).cpu()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)
    want = cpu.logits(Packet(i32(tokens), i32(slots), i32(place), table.cpu(), 3, max(place) + 1,
                             rope_pos=i32(where)))
    assert float(torch.nn.functional.cosine_similarity(got, want, dim=1).min()) > cosine


def test_what_cannot_be_is_refused_and_changes_nothing(make):
    from orinfer_b200.models.runner import Packet
    for bad in (dict(bound=150, keep=150), dict(keep=0), dict(first=100, recent=51), dict(recent=-1),
                dict(last_rows=0)):
        with pytest.raises(ValueError):
            make("tiny", **bad)
    pool = make("tiny", pages=4, slots=3, first=4, recent=64)
    cfg, i32 = pool.runner.cfg, pool._i32
    slot = pool.add(text(128, cfg.vocab))
    state = [t.clone() for t in (pool.table, pool.lens, pool.refs, pool.weights)]
    for call, error in [(lambda: pool.add([]), ValueError), (lambda: pool.step({}), ValueError),
                        (lambda: pool.step({slot + 9: 1}), ValueError),
                        (lambda: pool.generate([slot], [], 3), ValueError),
                        (lambda: pool.add(text(290, cfg.vocab)), MemoryError)]:   # two pages are left
        with pytest.raises(error):
            call()
        for t, before in zip((pool.table, pool.lens, pool.refs, pool.weights), state):
            assert torch.equal(t[slot] if t.shape[:1] == (3,) else t[:4], before[slot] if t.shape[:1] == (3,) else before[:4])
    assert len(pool._free) == 2 and pool.held == 1
    one = lambda **kw: Packet(i32([1]), i32([slot]), i32([128]), pool.table, 1, 129, weights=pool.weights, **kw)
    for packet in (one(attend_pos=i32([128])), one(weigh_chunks=i32([[0, 1, 128, slot]]))):
        with pytest.raises(ValueError):
            pool.runner.logits(packet)
    with pytest.raises(ValueError):
        p = one()
        p.weights = pool.weights[:1]                     # a layer has none
        pool.runner.logits(p)


def test_requests_are_cut_one_after_the_other_where_pages_are_few(make):
    """Two requests hold three pages each of eight, two are free; each cut wants two."""
    pool = make("tiny", pages=9, slots=2)
    cfg = pool.runner.cfg
    slots = [pool.add(text(300, cfg.vocab, n)) for n in (1, 2)]
    assert pool.held == 6
    pool.step({s: 3 for s in slots})
    assert pool.held == 4 and [pool._len[s] for s in slots] == [151] * 2


def test_the_example_runs(cuda):
    import importlib.util
    from pathlib import Path
    path = Path(__file__).resolve().parents[1] / "examples" / "bounded-cache.py"
    spec = importlib.util.spec_from_file_location("bounded_cache", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    assert [len(d) for d in module.main("tiny", 3, 20)] == [20] * 3


def test_a_packet_of_decode_rows_and_chunks_counts_both(make):
    """Two requests take a step while two prompts are prefilled, one of which lets its last ten rows count.
    Every row that counts gives each head a weight of one (5e-4: see above), to its own request."""
    from orinfer_b200.models.runner import Packet
    pool = make("tiny", slots=4, bound=300, keep=200)
    cfg, i32, heads = pool.runner.cfg, pool._i32, pool.runner.cfg.q_heads // pool.runner.cfg.kv_heads
    a, b = pool.add(text(200, cfg.vocab, 1)), pool.add(text(33, cfg.vocab, 2))
    free = [s for s in range(4) if s not in (a, b)]
    pool._take([free[0], free[1]], [0, 0])
    pool._grow([a, b], 1)
    before = pool.weights.double().sum(3)
    n = (100, 41)
    ids = [7, 8, *text(n[0], cfg.vocab, 3), *text(n[1], cfg.vocab, 4)]
    slots = [a, b, *[free[0]] * n[0], *[free[1]] * n[1]]
    chunks = [[2, n[0], 0, free[0]], [2 + n[0], n[1], 0, free[1]]]
    count = [chunks[0], [2 + n[0] + n[1] - 10, 10, n[1] - 10, free[1]]]
    p = Packet(i32(ids), i32(slots), i32([200, 33, *range(n[0]), *range(n[1])]), pool.table, sum(n) + 2, 201,
               torch.tensor([0, 1, sum(n) + 1], device=pool.device), chunks=i32(chunks), max_q_len=100,
               decode_rows=2, max_chunk_kv=100, weights=list(pool.weights), weigh_chunks=i32(count))
    logits = pool.runner.logits(p)
    got = pool.weights.double().sum(3) - before
    for slot, rows in ((a, 1), (b, 1), (free[0], n[0]), (free[1], 10)):
        assert float((got[:, slot] / (rows * heads) - 1).abs().max()) <= 5e-4
    assert bool((pool.weights[:, free[0], :, 100:] == 0).all())
    assert bool((pool.weights[:, free[1], :, :n[1]] > 0).all()) and bool((pool.weights[:, b, :, 34:] == 0).all())
    plain = pool.runner.logits(Packet(p.ids, p.row_req, p.row_pos, pool.table, p.rows, 201, p.logit_rows,
                                      chunks=p.chunks, max_q_len=100, decode_rows=2, max_chunk_kv=100))
    assert torch.equal(logits, plain)


def test_a_slot_without_a_request_is_refused(make):
    pool = make("tiny")
    slot = pool.add([1, 2, 3])
    option = S.SamplingOptions(temperature=0.9, top_k=5)
    other = slot - 1 if slot else slot + 1
    for call in (lambda: pool.generate([slot, other], [option] * 2, 2), lambda: pool.step({other: 1}),
                 lambda: pool.drop(other), lambda: pool.generate([slot, slot], [option] * 2, 2)):
        with pytest.raises(ValueError):
            call()
    assert pool.text[slot] == [1, 2, 3] and pool.held == 1
    assert pool.generate([slot], [option], 0) == [[]] and pool.generate([], [], 3) == []
