"""The 64-bit statements of the sample operators, against the host's law, pool and small cases."""
import math

import numpy as np
import pytest
import torch

from orinfer_b200.core import sampling as S
from orinfer_b200.engine.pages import PagePool
from orinfer_b200.ref import ops_ref, samples_ref as R


@pytest.mark.parametrize("seed", range(4))
def test_scores_are_those_of_the_host_law(seed):
    """log-softmax of the statement's scores against the log-probabilities that the host reports."""
    g = np.random.default_rng(seed)
    vocab = 97
    logits = (g.normal(size=vocab) * 3).astype(np.float32)
    history = g.integers(0, vocab + 5, size=60).tolist()
    bias = {int(t): float(g.normal() * 4) for t in g.integers(0, vocab, size=9)}
    allowed = g.random(vocab) < 0.5
    allowed[3] = True
    mask = np.zeros((vocab + 31) // 32, np.uint32)
    for t in np.flatnonzero(allowed):
        mask[t // 32] |= np.uint32(1) << np.uint32(t % 32)
    o = S.SamplingOptions(repetition_penalty=1.2, presence_penalty=0.4, frequency_penalty=-0.3,
                          logit_bias=bias)
    got, flag = R.process_logits(torch.from_numpy(logits), history, 1.2, 0.4, -0.3,
                                 sorted(bias.items()), torch.from_numpy(allowed))
    want = torch.log_softmax(got[torch.from_numpy(allowed)], 0)
    assert flag == 0
    for i, t in enumerate(np.flatnonzero(allowed)):
        lp, _ = S.logprobs(logits, history, o, int(t), 0, mask)
        assert abs(lp - float(want[i])) < 1e-12


def test_flags_say_what_the_host_law_refuses():
    x = torch.tensor([1.0, -2.0, 0.5])
    none = torch.zeros(3, dtype=torch.bool)
    assert R.process_logits(x, permitted=none)[1] == 1
    assert R.process_logits(torch.tensor([1.0, math.nan, 0.0]), permitted=none)[1] == 2
    assert R.process_logits(x, [0], repetition=1e-300)[1] == 2
    only = torch.tensor([False, True, True])
    assert R.process_logits(x, [0], repetition=1e-300, permitted=only)[1] == 0


def test_rows_are_causal_attention():
    g = torch.Generator().manual_seed(3)
    kvh, d, n = 2, 64, 150
    cells = lambda: torch.randint(-127, 128, (3, 128, kvh, d), generator=g, dtype=torch.int8)
    scales = lambda: (torch.rand(3, 128, kvh, 1, generator=g) * 0.02 + 0.01).half()
    k, v, ks, vs = cells(), cells(), scales(), scales()
    q = torch.randn(3, 4, d, generator=g).half()
    table = torch.tensor([[2, 1]], dtype=torch.int32)
    out, size, reach = R.attention_rows(q, None, torch.zeros(3, dtype=torch.int32),
                                        torch.tensor([n - 1, 0, -1], dtype=torch.int32), table, k,
                                        v, ks, vs)
    read = lambda c, s: ops_ref.kv_dequant(c, s)[[2, 1]].reshape(-1, kvh, d)
    for row, keys in ((0, n), (1, 1)):
        want = ops_ref.causal_gqa(q[row:row + 1], read(k, ks)[:keys], read(v, vs)[:keys], keys - 1)
        assert (out[row] - want[0].double()).abs().max() < 2e-3
    assert bool((out[2] == 0).all()) and bool((size >= out.abs() - 1e-9).all())
    assert bool((reach[:2] > 0).all())


def _pool(seed, slots=12, pages=40, width=6):
    """A host pool with requests on it: (table, lens, refs, tensors, pool)."""
    g = torch.Generator().manual_seed(seed)
    pool = PagePool(pages)
    table = torch.zeros(slots, width, dtype=torch.int32)
    lens = torch.zeros(slots, dtype=torch.int32)
    for s, n in ((1, 300), (4, 256), (5, 1), (8, 128), (9, 700)):
        pages_of = pool.take((n + 127) // 128)
        table[s, :len(pages_of)] = torch.tensor(pages_of)
        lens[s] = n
    tensors = [torch.randint(-100, 100, (pages, 128, 2, 64), generator=g, dtype=torch.int8),
               torch.rand(pages, 128, 2, 1, generator=g).half()]
    return table, lens, torch.tensor(pool.refs, dtype=torch.int32), tensors, pool


def _text(tensors, table, lens, s):
    """What slot s holds, token by token."""
    n = int(lens[s])
    return [t[table[s].long()].reshape(-1, *t.shape[2:])[:n] for t in tensors]


def test_a_fork_holds_what_its_parent_holds_and_is_its_own():
    table, lens, refs, tensors, _ = _pool(1)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)
    before = {s: [x.clone() for x in _text(tensors, table, lens, s)] for s in (1, 4, 5)}
    t, l, r, status = R.fork_pages(tensors, table, lens, refs, i32([1, 4, 1, 5]), i32([0, 2, 3, 6]))
    assert status == 0
    for p, c in ((1, 0), (4, 2), (1, 3), (5, 6)):
        for a, b in zip(before[p], _text(tensors, t, l, c)):
            assert torch.equal(a, b)
    last = t[[1, 0, 3], 2].tolist()
    assert len(set(last)) == 3 and r[t[1, 0]] == 3 and all(r[p] == 1 for p in last)
    # freed again, everything is as before
    t2, l2, r2 = R.free_pages(t, l, r, i32([0, 2, 3, 6, 0]))
    assert torch.equal(t2, table) and torch.equal(l2, lens) and torch.equal(r2, refs)


@pytest.mark.parametrize("parents,children,status", [
    ([1], [1], 2), ([1], [4], 2), ([1, 4], [0, 0], 2), ([99], [0], 2), ([1], [-1], 2),
    ([2, 1], [0, 2], 2), ([1] * 6, [0, 2, 3, 6, 7, 10], 1), ([2], [0], 0)])
def test_forks_that_cannot_be_change_nothing(parents, children, status):
    table, lens, refs, tensors, pool = _pool(2)
    while pool.available > 5:
        refs[pool.take(1)[0]] = 1
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)
    t, l, r, got = R.fork_pages(tensors, table, lens, refs, i32(parents), i32(children))
    assert got == status
    assert torch.equal(t, table) and torch.equal(l, lens) and torch.equal(r, refs)


def test_compaction_keeps_every_slot():
    table, lens, refs, tensors, _ = _pool(3)
    table, lens, refs = R.free_pages(table, lens, refs, torch.tensor([1, 5], dtype=torch.int32))
    before = {s: [x.clone() for x in _text(tensors, table, lens, s)] for s in (4, 8, 9)}
    t, r, moved = R.compact_pages(tensors, table, refs)
    live = int((refs > 0).sum())
    assert bool((r[1:live + 1] > 0).all()) and bool((r[live + 1:] == 0).all())
    for s, text in before.items():
        assert all(torch.equal(a, b) for a, b in zip(text, _text(tensors, t, lens, s)))
    assert sorted(moved[refs > 0].tolist()) == list(range(1, live + 1))
