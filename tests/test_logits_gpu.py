"""Penalties, biases and masks on logits, against the 64-bit statement rounded once."""
import math

import pytest
import torch

from orinfer_b200.ref import samples_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(cuda):
    return cuda


def words(permitted):
    """bool [m, vocab] -> int32 [m, (vocab + 31) / 32]"""
    m, vocab = permitted.shape
    bits = torch.zeros(m, (vocab + 31) // 32 * 32, dtype=torch.int64)
    bits[:, :vocab] = permitted.long()
    v = (bits.view(m, -1, 32) << torch.arange(32)).sum(2)
    return torch.where(v >= 2 ** 31, v - 2 ** 32, v).int()


def case(rows, vocab, hist, biases, seed=0, masks=True):
    g = torch.Generator().manual_seed(seed + vocab + 31 * rows)
    r = lambda *s: torch.rand(*s, generator=g, dtype=torch.float64)
    lens = torch.randint(0, hist + 1, (rows,), generator=g, dtype=torch.int32)
    lens[0] = hist
    ids = (r(rows, hist) ** 4 * vocab).int()
    far = r(rows, hist) < 0.05                       # media rows and other vocabularies
    ids[far] = torch.randint(-5, vocab + 2 ** 30, (int(far.sum()),), generator=g,
                             dtype=torch.int32)
    count = torch.randint(0, biases + 1, (rows,), generator=g)
    start = torch.cat([torch.zeros(1, dtype=torch.int64), count.cumsum(0)]).int()
    total = int(start[-1])
    which = torch.arange(rows, dtype=torch.int32)
    which[1::3] = -1
    permitted = r(rows, vocab) < 0.3
    permitted[:, vocab // 2] = True
    kw = dict(history=ids, history_len=lens, repetition=r(rows) + 0.7, presence=r(rows) * 3 - 1,
              frequency=r(rows) * 2 - 1)
    if biases:
        kw.update(bias_start=start, bias_values=r(total) * 200 - 100,
                  bias_ids=torch.randint(-2, vocab + 2, (total,), generator=g, dtype=torch.int32))
    if masks:
        kw.update(mask=words(permitted), mask_rows=which)
    return torch.randn(rows, vocab, generator=g) * 4, kw, permitted


def expected(logits, kw, permitted, masked):
    scores, flags = [], []
    for i in range(logits.shape[0]):
        n = int(kw["history_len"][i]) if "history" in kw else 0
        bias = []
        if "bias_start" in kw:
            lo, hi = kw["bias_start"][i:i + 2].tolist()
            bias = list(zip(kw["bias_ids"][lo:hi].tolist(), kw["bias_values"][lo:hi].tolist()))
        which = int(kw["mask_rows"][i]) if "mask_rows" in kw else i
        s, f = R.process_logits(
            logits[i], kw["history"][i, :n].tolist() if n else None,
            *(float(kw[k][i]) if k in kw else d
              for k, d in (("repetition", 1.0), ("presence", 0.0), ("frequency", 0.0))), bias,
            permitted[which] if "mask" in kw and which >= 0 else None, masked)
        scores.append(s)
        flags.append(f)
    return torch.stack(scores), torch.tensor(flags, dtype=torch.int32)


def check(dev, logits, kw, permitted, masked=-1e30, out=None, x=None):
    """The host law's 64-bit score, rounded to FP32: the operations are the same, so every bit is."""
    from orinfer_b200.ops import functional as F
    want, flags = expected(logits, kw, permitted, masked)
    x = logits.to(dev) if x is None else x
    got, f = F.process_logits(x, masked=masked, out=out, **{k: v.to(dev) for k, v in kw.items()})
    assert torch.equal(f.cpu(), flags)
    same = (got.cpu() == want.float()) | (got.cpu().isnan() & want.isnan())
    assert bool(same.all()), (~same).nonzero()[:4]
    return got


@pytest.mark.parametrize("rows,vocab,hist,biases", [
    (1, 1, 1, 1), (1, 31, 4, 0), (2, 33, 70, 3), (3, 1024, 200, 10), (5, 4097, 33, 5),
    (4, 8192, 5000, 100), (3, 50001, 1, 300), (2, 151936, 3000, 50), (40, 1000, 64, 8)])
@pytest.mark.parametrize("masked", [-1e30, -math.inf])
def test_against_the_host_law(dev, rows, vocab, hist, biases, masked):
    check(dev, *case(rows, vocab, hist, biases), masked=masked)


@pytest.mark.parametrize("drop", [("history", "history_len", "repetition", "presence", "frequency"),
                                  ("bias_start", "bias_ids", "bias_values"), ("mask", "mask_rows"),
                                  ("mask_rows",), ("repetition",), ("presence", "frequency"),
                                  ("repetition", "presence", "frequency")])
def test_parts_that_are_absent(dev, drop):
    logits, kw, permitted = case(6, 3001, 100, 7)
    check(dev, logits, {k: v for k, v in kw.items() if k not in drop}, permitted)


def test_neutral_rows_are_copied(dev):
    logits, kw, permitted = case(3, 2000, 50, 0, masks=False)
    kw["repetition"][:], kw["presence"][:], kw["frequency"][:] = 1.0, 0.0, 0.0
    logits[1, 5] = -0.0
    got = check(dev, logits, kw, permitted)
    assert torch.equal(got.cpu().view(torch.int32), logits.view(torch.int32))


def test_strides_and_in_place(dev):
    logits, kw, permitted = case(4, 777, 60, 5)
    wide = torch.full((4, 1000), 9.0, device=dev)
    wide[:, 3:780] = logits.to(dev)
    to = torch.full((4, 901), 7.0, device=dev)
    check(dev, logits, kw, permitted, x=wide[:, 3:780], out=to[:, 1:778])
    assert bool((to[:, 0] == 7).all()) and bool((to[:, 778:] == 7).all())
    view = wide[:, 3:780]
    got = check(dev, logits, kw, permitted, x=view, out=view)
    assert got.data_ptr() == view.data_ptr() and bool((wide[:, :3] == 9).all())
    hist = torch.zeros(4, 100, dtype=torch.int32)
    hist[:, :60] = kw["history"]
    cut = hist.to(dev)[:, :60]
    from orinfer_b200.ops import functional as F
    more = {k: v.to(dev) for k, v in kw.items()}
    again, _ = F.process_logits(logits.to(dev), **{**more, "history": cut})
    assert torch.equal(again, got)


def test_one_token_many_times_and_the_last_bias_wins(dev):
    logits, kw, permitted = case(2, 640, 9000, 0, masks=False)
    kw["history"][:] = 17
    kw["history_len"][:] = torch.tensor([9000, 1])
    kw.update(bias_start=torch.tensor([0, 3, 6], dtype=torch.int32),
              bias_ids=torch.tensor([17, 4, 17, 639, 639, 0], dtype=torch.int32),
              bias_values=torch.tensor([5.0, 2.0, -1.5, 1.0, 1e-9, 0.0], dtype=torch.float64))
    check(dev, logits, kw, permitted)


def test_rows_that_the_host_law_refuses(dev):
    logits, kw, permitted = case(7, 500, 20, 2)
    kw["mask_rows"] = torch.arange(7, dtype=torch.int32)
    permitted[1] = False                             # nothing permitted
    permitted[2] = False
    permitted[2, 499] = True                         # one token, the last
    logits[3, 7], logits[4, 499], logits[5, 0] = math.nan, math.inf, -math.inf
    kw["repetition"][6] = 1e-300                     # a score past FP32's range
    kw["history"][6, :3] = 3
    permitted[6, 3] = True
    kw["mask"] = words(permitted)
    from orinfer_b200.ops import functional as F
    _, flags = F.process_logits(logits.to(dev), **{k: v.to(dev) for k, v in kw.items()})
    want, f = expected(logits, kw, permitted, -1e30)
    assert torch.equal(flags.cpu(), f) and f.tolist()[1:] == [1, 0, 2, 2, 2, 2]
    kw["mask_rows"][0] = 7                           # a mask that does not exist
    _, flags = F.process_logits(logits.to(dev), **{k: v.to(dev) for k, v in kw.items()})
    assert int(flags[0]) == 2


@pytest.mark.parametrize("hist,step", [(32767, 8), (60000, 1), (40000, 8)])
def test_long_histories_of_many_tokens(dev, hist, step):
    """Counts of 16 bits and more, and tokens that all fall to one CTA or fill every list."""
    logits, kw, permitted = case(2, 151936, hist, 20, seed=hist)
    g = torch.Generator().manual_seed(step)
    kw["history"] = torch.randint(0, 151936 // step, (2, hist), generator=g, dtype=torch.int32) * step
    check(dev, logits, kw, permitted)


@pytest.mark.parametrize("rows,vocab,hist,biases", [
    (3, 5000, 2048, 9), (3, 5000, 2049, 9), (38, 5000, 1280, 9), (38, 4000, 1283, 9),
    (2, 3000, 16384, 5), (2, 3000, 16385, 5), (39, 2000, 17001, 5), (3, 500001, 20001, 40),
    (38, 200003, 2500, 10), (38, 3001, 33001, 5)])
def test_histories_that_the_ctas_of_a_row_sort(dev, rows, vocab, hist, biases):
    """As long as each CTA looks through, one token more, as long as is sorted at a time and more,
    for few rows and many, on vocabularies of one table and of several; at any alignment."""
    logits, kw, permitted = case(rows, vocab, hist, biases)
    kw["history_len"][-1] = hist - 1
    check(dev, logits, kw, permitted)


def test_many_biases_of_a_row_among_many(dev):
    n, rows, vocab = 32768, 38, 30000
    g = torch.Generator().manual_seed(4)
    logits, kw, permitted = case(rows, vocab, 40, 0, masks=False)
    start = torch.full((rows + 1,), n, dtype=torch.int32)
    start[0] = 0
    kw.update(bias_start=start, bias_values=torch.rand(n, generator=g, dtype=torch.float64),
              bias_ids=torch.randint(0, vocab, (n,), generator=g, dtype=torch.int32))
    check(dev, logits, kw, permitted)


def test_many_biases_on_a_large_vocabulary(dev):
    """As many entries as a row may have, most tokens named more than once, on more tokens than the
    tables of a cluster hold; one entry more is refused."""
    vocab, n = 300001, 32768
    g = torch.Generator().manual_seed(3)
    logits, kw, permitted = case(2, vocab, 500, 0, masks=False)
    kw.update(bias_start=torch.tensor([0, n, n + 9], dtype=torch.int32),
              bias_ids=torch.randint(0, vocab // 20, (n + 9,), generator=g, dtype=torch.int32) * 19,
              bias_values=torch.rand(n + 9, generator=g, dtype=torch.float64))
    check(dev, logits, kw, permitted)
    from orinfer_b200.ops import functional as F
    kw["bias_start"] = torch.tensor([0, n + 1, n + 9], dtype=torch.int32)
    _, flags = F.process_logits(logits.to(dev), **{k: v.to(dev) for k, v in kw.items()})
    assert flags.tolist() == [2, 0]


def test_the_sampler_and_the_argmax_take_masked_scores(dev):
    """One permitted token is drawn by both, whatever the others' logits are."""
    from orinfer_b200.ops import functional as F
    rows, vocab = 5, 4000
    logits = torch.randn(rows, vocab, device=dev) * 5
    permitted = torch.zeros(rows, vocab, dtype=torch.bool)
    only = [0, 31, 32, 3999, 1777]
    permitted[torch.arange(rows), torch.tensor(only)] = True
    out, flags = F.process_logits(logits, mask=words(permitted).to(dev))
    f64 = lambda v: torch.full((rows,), v, dtype=torch.float64, device=dev)
    tok, flag = F.sample_topk(out, torch.full((rows,), 40, dtype=torch.int32, device=dev),
                              f64(0.8), f64(0.95), f64(0.7))
    assert tok.tolist() == only and F.argmax(out).tolist() == only
    assert int((flag | flags).sum()) == 0


def test_a_large_batch_with_offsets_past_32_bits(dev):
    """rows x vocab x 4 bytes past 2^32: the last rows, and a row stride of its own."""
    from orinfer_b200.ops import functional as F
    rows, vocab = 9, 140000000
    x = torch.zeros(rows, vocab, device=dev)
    x[-1, -1] = 2.0
    hist = torch.full((rows, 1), vocab - 1, dtype=torch.int32, device=dev)
    ones = torch.ones(rows, dtype=torch.int32, device=dev)
    out, flags = F.process_logits(x, history=hist, history_len=ones,
                                  repetition=torch.full((rows,), 4.0, dtype=torch.float64,
                                                        device=dev), out=x)
    assert float(out[-1, -1]) == 0.5 and int(flags.sum()) == 0


def test_on_another_stream_and_in_a_graph(dev):
    from orinfer_b200.ops import functional as F
    logits, kw, _ = case(8, 5000, 300, 9)
    x, gpu = logits.to(dev), {k: v.to(dev) for k, v in kw.items()}
    want, flags = (t.clone() for t in F.process_logits(x, **gpu))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got, _ = F.process_logits(x, **gpu)
    side.synchronize()
    assert torch.equal(got, want)
    out, f = torch.empty_like(want), torch.empty_like(flags)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        F.process_logits(x, out=out, flags=f, **gpu)
    for _ in range(3):
        out.zero_()
        f.fill_(9)
        graph.replay()
        assert torch.equal(out, want) and torch.equal(f, flags)


def test_refusals(dev):
    from orinfer_b200.ops import functional as F
    from orinfer_b200.ops.native import KernelError
    logits, kw, _ = case(3, 100, 10, 4)
    x, gpu = logits.to(dev), {k: v.to(dev) for k, v in kw.items()}
    F.process_logits(x, **gpu)
    for bad in (x.half(), x[0], x.t(), logits, x[:2]):
        with pytest.raises(KernelError):
            F.process_logits(bad, **gpu)
    for name, values in {
            "history": [gpu["history"].long(), gpu["history"][:2], gpu["history"].t()],
            "history_len": [None, gpu["history_len"].long(), gpu["history_len"][:2]],
            "repetition": [gpu["repetition"].float(), gpu["repetition"][:2]],
            "presence": [kw["presence"]], "frequency": [gpu["frequency"][None]],
            "bias_start": [gpu["bias_start"][:3], gpu["bias_start"].long()],
            "bias_ids": [None, gpu["bias_ids"][:-1], gpu["bias_ids"].long()],
            "bias_values": [None, gpu["bias_values"].float()],
            "mask": [gpu["mask"][:, :3], gpu["mask"].long(), gpu["mask"][0]],
            "mask_rows": [gpu["mask_rows"].long(), gpu["mask_rows"][:2]]}.items():
        for v in values:
            with pytest.raises(KernelError):
                F.process_logits(x, **{**gpu, name: v})
    with pytest.raises(KernelError):
        F.process_logits(x, mask=gpu["mask"][:2])
    with pytest.raises(KernelError):
        F.process_logits(x, repetition=gpu["repetition"])
    with pytest.raises(KernelError):
        F.process_logits(x, out=x[:2])
    with pytest.raises(KernelError):
        F.process_logits(x, flags=torch.zeros(3, device=dev))


def test_no_rows(dev):
    from orinfer_b200.ops import functional as F
    out, flags = F.process_logits(torch.empty(0, 50, device=dev))
    assert out.shape == (0, 50) and flags.shape == (0,)
