"""The device sampler on scores at and below the one that masked tokens get."""
import numpy as np
import pytest
import torch

from orinfer_b200.core import sampling as S

pytestmark = pytest.mark.gpu


def test_rows_of_low_scores_only_are_drawn_as_by_the_host_law(cuda):
    """Whatever a row's scores are, the draw is the host law's: all below -1e30, some, or one above."""
    from orinfer_b200.ops import functional as F
    rows, vocab = 24, 900
    g = torch.Generator().manual_seed(5)
    logits = -1e30 * (1.0 + torch.rand(rows, vocab, generator=g))
    logits[8:16] *= 1e7
    logits[16] = -1e30 * (1.0 + torch.arange(vocab) / vocab)      # the largest is -1e30 itself
    logits[17, 100:120] = -1e30
    logits[18:, 3] = torch.tensor([-9.9e29, 0.0, 5.0, -1e20, 1e30, -9.9e29])
    logits[21:, 800] = torch.tensor([-9.8e29, 2.0, -9.9e29])
    ks = [1 + (5 * i) % 40 for i in range(rows)]
    us = [S.counter_uniform(7, 0, i) for i in range(rows)]
    dev = lambda v, dt: torch.tensor(v, dtype=dt, device=cuda)
    tok, flag = F.sample_topk(logits.to(cuda), dev(ks, torch.int32), dev([0.8] * rows, torch.float64),
                              dev([0.95] * rows, torch.float64), dev(us, torch.float64))
    assert flag.tolist() == [0] * rows
    want = [S.sample(logits[i].numpy(), [], S.SamplingOptions(temperature=0.8, top_p=0.95, top_k=ks[i]),
                     us[i]) for i in range(rows)]
    assert tok.tolist() == want


@pytest.mark.parametrize("permitted", [1, 2, 39, 40, 41])
def test_few_permitted_tokens_leave_fewer_candidates(cuda, permitted):
    from orinfer_b200.ops import functional as F
    rows, vocab = 6, 3000
    g = torch.Generator().manual_seed(permitted)
    logits = torch.randn(rows, vocab, generator=g) * 3
    words = np.zeros((vocab + 31) // 32, np.uint32)
    for t in torch.randperm(vocab, generator=g)[:permitted].tolist():
        words[t // 32] |= np.uint32(1) << np.uint32(t % 32)
    mask = torch.from_numpy(words.view(np.int32)).to(cuda).view(1, -1)
    out, flags = F.process_logits(logits.to(cuda), mask=mask,
                                  mask_rows=torch.zeros(rows, dtype=torch.int32, device=cuda))
    us = [S.counter_uniform(3, 0, i) for i in range(rows)]
    f64 = lambda v: torch.tensor(v, dtype=torch.float64, device=cuda)
    tok, flag = F.sample_topk(out, torch.full((rows,), 40, dtype=torch.int32, device=cuda),
                              f64([0.9] * rows), f64([1.0] * rows), f64(us))
    assert int((flag | flags).sum()) == 0
    o = S.SamplingOptions(temperature=0.9, top_k=40)
    assert tok.tolist() == [S.sample(logits[i].numpy(), [], o, us[i], words) for i in range(rows)]
