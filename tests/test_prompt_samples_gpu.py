"""Samples of shared prompts through the model: decoding, penalties, masks, pages given back."""
import importlib.util
from pathlib import Path

import numpy as np
import pytest
import torch

from orinfer_b200.config import PRESETS
from orinfer_b200.core import sampling as S
from orinfer_b200.models.weights import random_model
from orinfer_b200.ops import functional as F

pytestmark = pytest.mark.gpu


@pytest.fixture
def pool_of(cuda):
    from orinfer_b200.models.runner import KVPool, ModelRunner
    from orinfer_b200.models.samples import PromptSamples

    def make(preset, pages=40, slots=12, max_tokens=700):
        cfg = PRESETS[preset]
        runner = ModelRunner(random_model(cfg, seed=3, device=cuda),
                             KVPool.allocate(cfg, pages, cuda), max_rows=256)
        return PromptSamples(runner, slots, max_tokens)
    return make


def text(n, vocab, seed=0):
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.parametrize("preset", ["tiny", "tiny-moe", "tiny-hybrid"])
def test_a_step_with_shared_prefixes_has_the_logits_of_a_step_without(pool_of, preset):
    """Both are held to a cosine of 0.999 against the quantised reference model elsewhere; between
    themselves they differ by the rounding of the attention to FP16 and what the INT8 activations
    make of it."""
    from orinfer_b200.models.runner import Packet
    pool = pool_of(preset)
    cfg, dev, n = pool.runner.cfg, pool.device, 5
    prompt = pool.add(text(300, cfg.vocab))
    slots = [pool._free[-1 - i] for i in range(n)]
    F.fork_pages(pool.cache, pool.table, pool.lens, pool.refs, pool._i32([prompt] * n),
                 pool._i32(slots), out=(pool.table, pool.lens, pool.refs))
    plan = F.SharedPrefix([(0, n, 256)], n, qh=cfg.q_heads, kvh=cfg.kv_heads,
                          head_dim=cfg.head_dim, max_kv_len=301, device=dev, force=True)
    tokens = pool._i32(text(n, cfg.vocab, 1))
    got = []
    for shared in (None, plan):
        for s in slots:
            if pool._prompts[prompt][2] is not None:
                pool.runner.gdn_restore(s, pool._prompts[prompt][2], pool.slots)
        p = Packet(tokens, pool._i32(slots), pool._i32([300] * n), pool.table, n, 301,
                   shared=shared)
        got.append(pool.runner.logits(p).clone())
    cos = torch.nn.functional.cosine_similarity(got[0], got[1], dim=1)
    assert float(cos.min()) > 0.999
    p = Packet(tokens, pool._i32(slots), pool._i32([300] * n), pool.table, n, 301, shared=plan,
               chunks=pool._i32([[0, n, 300, slots[0]]]))
    with pytest.raises(ValueError):
        pool.runner.logits(p)


@pytest.mark.parametrize("preset,force", [("tiny", False), ("tiny", True), ("tiny-hybrid", True)])
def test_samples_follow_the_host_law(pool_of, preset, force):
    """Every token is the one that the host law draws from the step's logits.  (The device rounds
    the scores to FP32 once: a draw moves with a chance of about 1e-7.)  All pages come back."""
    pool = pool_of(preset)
    vocab = pool.runner.cfg.vocab
    lens = (300, 128, 90)
    prompts = [pool.add(text(n, vocab, n)) for n in lens]
    options = [[S.SamplingOptions(temperature=0.9, top_k=20, top_p=0.9, seed=1,
                                  repetition_penalty=1.3),
                S.SamplingOptions(temperature=0.9, top_k=20, seed=2, presence_penalty=0.5,
                                  logit_bias={7: 4.0, 9: -3.0}),
                S.SamplingOptions(temperature=0.0, frequency_penalty=0.4)],
               [S.SamplingOptions(temperature=0.7, top_k=64, seed=i) for i in range(4)],
               [S.SamplingOptions(temperature=1.1, top_k=0, seed=9)]]
    flat = [o for group in options for o in group]
    of = [0] * 3 + [1] * 4 + [2]
    mask = np.random.default_rng(0).integers(0, 2 ** 32, (vocab + 31) // 32, dtype=np.uint32)
    before = pool.refs.clone()
    history = [list(pool._prompts[prompts[p]][0]) for p in of]
    steps = []

    def on_step(rows, logits, tokens):
        for r, i in enumerate(rows):
            u = S.counter_uniform(flat[i].seed, 0, len(history[i]) - lens[of[i]])
            want = S.sample(logits[r].cpu().numpy(), history[i], flat[i], u, mask)
            assert int(tokens[r]) == want
            assert int(mask[want // 32]) >> (want % 32) & 1
            history[i].append(want)
        steps.append(len(rows))

    stop = lambda tokens: len(tokens) > 3 and tokens[-1] % 16 == 0
    out = pool.sample(prompts, options, 60, mask=mask, stop=stop, force=force, on_step=on_step)
    assert [t for group in out for t in group] == [h[lens[p]:] for h, p in zip(history, of)]
    assert steps[0] == 8 and len(set(steps)) > 2          # samples ended one after the other
    assert torch.equal(pool.refs, before)
    assert sorted(pool._free) == [s for s in range(12) if s not in prompts]


def test_a_prompt_that_moved_gives_the_same_samples(pool_of):
    pool = pool_of("tiny")
    vocab = pool.runner.cfg.vocab
    a, b = pool.add(text(500, vocab, 1)), pool.add(text(333, vocab, 2))
    options = [[S.SamplingOptions(temperature=0.9, top_k=30, seed=i) for i in range(6)]]
    first = pool.sample([b], options, 20, force=True)
    where = pool.table[b].clone()
    pool.drop(a)
    assert pool.compact() == 3
    assert not torch.equal(where, pool.table[b]) and int(pool.table[b].max()) == 3
    assert pool.sample([b], options, 20, force=True) == first


def test_what_does_not_fit_is_refused_and_changes_nothing(pool_of):
    pool = pool_of("tiny", pages=6, slots=8, max_tokens=256)
    vocab = pool.runner.cfg.vocab
    one = S.SamplingOptions(temperature=0.9, top_k=5)
    slot = pool.add(text(200, vocab))
    state = [t.clone() for t in (pool.table, pool.lens, pool.refs)]
    free = list(pool._free)
    for call, error in [
            (lambda: pool.add([]), ValueError), (lambda: pool.add([1] * 257), ValueError),
            (lambda: pool.sample([slot + 1], [[one]], 4), ValueError),
            (lambda: pool.sample([slot], [[one]], 58), ValueError),
            (lambda: pool.sample([slot], [[one] * 8], 4), MemoryError),      # slots
            (lambda: pool.sample([slot], [[one] * 4], 4), MemoryError)]:     # pages
        with pytest.raises(error):
            call()
        assert all(torch.equal(x, y) for x, y in zip(state, (pool.table, pool.lens, pool.refs)))
        assert pool._free == free
    assert pool.sample([slot], [[one] * 2], 0) == [[[], []]]
    # Pages end in the middle of a run: what the samples held comes back.
    pool.drop(slot)
    slot = pool.add(text(120, vocab))
    held = pool.held
    with pytest.raises(MemoryError):
        pool.sample([slot], [[one] * 3], 30)
    assert pool.held == held
    assert [len(t) for t in pool.sample([slot], [[one] * 2], 30)[0]] == [30, 30]


def test_the_example(cuda):
    path = Path(__file__).resolve().parents[1] / "examples" / "parallel-samples.py"
    spec = importlib.util.spec_from_file_location("parallel_samples", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    drawn, again = module.main("tiny", 3, 8)
    assert [[len(s) for s in g] for g in drawn] == [[8] * 3] * 2 and len(again) == 3
