"""Scores that cancel: every operation of the host law is rounded by itself."""
import numpy as np
import pytest
import torch

from orinfer_b200.core import sampling as S

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(cuda):
    return cuda


def run(dev, logits, history, rep, pres, freq):
    from orinfer_b200.ops import functional as F
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    f64 = lambda v: torch.tensor(v, dtype=torch.float64, device=dev)
    n = max(len(h) for h in history)
    got, flags = F.process_logits(
        torch.from_numpy(logits).to(dev), history=i32([h + [0] * (n - len(h)) for h in history]),
        history_len=i32([len(h) for h in history]), repetition=f64(rep), presence=f64(pres),
        frequency=f64(freq))
    assert int(flags.sum()) == 0
    return got.cpu().numpy()


@pytest.mark.parametrize("rows", [1, 64])
def test_a_product_is_rounded_before_it_is_taken_away(dev, rows):
    """Row r: token 5 occurs as often, and its logit is what frequency times that rounds to; token 9 has
    a negative logit whose product with the repetition penalty the presence penalty takes away.  Both
    leave nothing, where an unrounded product leaves 1e-17."""
    rng = np.random.default_rng(rows)
    logits = np.full((rows, 100), -30.0, dtype=np.float32)
    history, rep, pres, freq, want = [], [], [], [], []
    for r in range(rows):
        x, times = (np.float32(1.0), 10) if r == 0 else (np.float32(rng.uniform(0.1, 9)),
                                                         int(rng.integers(3, 40)))
        if r % 2 == 0:
            logits[r, 5] = x
            history.append([5] * times)
            rep.append(1.0), pres.append(0.0), freq.append(float(x) / times)
            want.append((5, np.float32(float(x) - freq[-1] * times)))
        else:
            logits[r, 9] = -x
            history.append([9])
            rep.append(float(rng.uniform(1.01, 1.9)))
            pres.append(-float(x) * rep[-1])
            freq.append(0.0)
            want.append((9, np.float32(0.0)))
    got = run(dev, logits, history, rep, pres, freq)
    for r, (token, score) in enumerate(want):
        assert got[r, token] == score, (r, got[r, token])


def test_ties_are_broken_as_the_host_breaks_them(dev):
    """Two tokens of score 0, one of which is a difference: the lower id wins on both sides."""
    logits = np.full((2, 64), -5.0, dtype=np.float32)
    logits[0, 3], logits[0, 40] = 1.0, 0.0
    logits[1, 40], logits[1, 3] = 1.0, 0.0
    history = [[3] * 10, [40] * 10]
    got = run(dev, logits, history, [1.0] * 2, [0.0] * 2, [0.1] * 2)
    for r in range(2):
        o = S.SamplingOptions(temperature=0.0, frequency_penalty=0.1)
        assert int(got[r].argmax()) == S.sample(logits[r], history[r], o, 0.5) == 3
