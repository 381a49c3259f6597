"""Decode attention that weighs its keys: outputs bit for bit those of ``attention``, sums of weights
against the 64-bit statement."""
import pytest
import torch

from orinfer_b200.ref import eviction_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(cuda):
    return cuda


def batch(dev, lens, qh, kvh, d, *, per=1, seed=0, score=1.0, gated=False):
    """Requests of these lengths with ``per`` rows each, the last at its end, on pages in any order;
    what no row sees holds numbers that are none."""
    g = torch.Generator().manual_seed(seed * 7919 + qh * 31 + d)
    width = max([-(-n // 128) for n in lens] + [1]) + 1
    counts = [-(-n // 128) for n in lens]
    pages = sum(counts) + 1
    order, at = torch.randperm(pages - 1, generator=g) + 1, 0
    table = torch.zeros(len(lens), width, dtype=torch.int32)
    kc, vc = (torch.randint(-127, 128, (pages, 128, kvh, d), generator=g, dtype=torch.int8)
              for _ in range(2))
    ks, vs = ((torch.rand(pages, 128, kvh, d // 64, generator=g) * 0.019 + 1e-3).half()
              for _ in range(2))
    for s, n in enumerate(counts):
        table[s, :n] = order[at:at + n].int()
        at += n
        if lens[s] % 128:
            ks[table[s, n - 1], lens[s] % 128:] = float("nan")
            vs[table[s, n - 1], lens[s] % 128:] = float("inf")
    ks[0], vs[0] = float("nan"), float("nan")
    req = [s for s in range(len(lens)) for _ in range(per)]
    pos = [max(-1, n - per + i) for n in lens for i in range(per)]
    q = (torch.randn(len(req), qh, d, generator=g) * score).half()
    gate = torch.randn(len(req), qh, d, generator=g).half().to(dev) if gated else None
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    return (q.to(dev), gate, i32(req), i32(pos), table.to(dev), kc.to(dev), vc.to(dev), ks.to(dev),
            vs.to(dev))


def near(got, base, args, per=1):
    """A score's FP32 sums of 64 products at a time are off by 64 steps of 2^-23 of its terms'
    magnitudes and eight roundings, twice (its own and the sum's); a row's sum of weights is a chain
    of a 128th of its keys and 64 more; the exponentials and the division eight roundings; then a
    rounding for each weight that is added."""
    q, _, req, pos, table, kc, _, ks, _ = args
    added, reach = R.key_weights(q, req, pos, table, kc, ks)
    keys = int(pos.max()) + 1
    rel = 2 * (64 * 2 + 8) * 2.0 ** -24 * reach + (keys / 128 + 72) * 2.0 ** -24
    adds = q.shape[1] // kc.shape[2] * per + 1
    want = base.double()
    want[..., :added.shape[-1]] += added
    limit = adds * 2.0 ** -24 * want
    limit[..., :added.shape[-1]] += added * rel
    off = (got.double() - want).abs()
    assert bool((off <= limit).all()), f"{float((off / limit.clamp(min=1e-30)).max())} of the limit"


def sums(dev, args, extra=0, seed=3):
    g = torch.Generator().manual_seed(seed)
    table, kvh = args[4], args[5].shape[2]
    return torch.rand(table.shape[0], kvh, table.shape[1] * 128 + extra, generator=g).to(dev)


GEOMETRIES = [(4, 2, 64), (16, 8, 64), (8, 8, 64), (8, 1, 64), (32, 8, 128), (40, 8, 128), (2, 2, 128),
              (16, 4, 128), (16, 2, 256), (4, 4, 256)]


@pytest.mark.parametrize("qh,kvh,d", GEOMETRIES)
@pytest.mark.parametrize("splits", [1, 2, 5])
def test_lengths(dev, qh, kvh, d, splits):
    from orinfer_b200.ops import functional as F
    args = batch(dev, [1, 2, 31, 32, 33, 127, 128, 129, 0, 500, 1111], qh, kvh, d, gated=d == 256)
    base = sums(dev, args)
    weights = base.clone()
    out = F.attention_weighed(*args, weights, splits=splits)
    assert torch.equal(out, F.attention(*args, splits=splits))
    near(weights, base, args)


@pytest.mark.parametrize("qh,kvh,d", [(4, 2, 64), (32, 8, 128), (40, 8, 128), (16, 2, 256)])
@pytest.mark.parametrize("splits", [1, 3, 32])
def test_long_rows(dev, qh, kvh, d, splits):
    """Both forms of the row kernel, several launch shapes of the sums."""
    from orinfer_b200.ops import functional as F
    args = batch(dev, [5000, 3, 2047], qh, kvh, d, seed=splits)
    base = sums(dev, args)
    weights = base.clone()
    out = F.attention_weighed(*args, weights, splits=splits, max_kv_len=5000)
    assert torch.equal(out, F.attention(*args, splits=splits, max_kv_len=5000))
    near(weights, base, args)


@pytest.mark.parametrize("d,score", [(64, 8.0), (128, 8.0), (256, 8.0), (128, 0.0)])
def test_leaping_and_equal_scores(dev, d, score):
    from orinfer_b200.ops import functional as F
    args = batch(dev, [700, 90, 1500], 8, 2, d, score=score)
    base = sums(dev, args)
    weights = base.clone()
    F.attention_weighed(*args, weights, splits=2)
    near(weights, base, args)


def test_many_short_rows_share_a_cta(dev):
    """The form of four heads to a CTA."""
    from orinfer_b200.ops import functional as F
    args = batch(dev, [1 + i % 60 for i in range(300)], 8, 8, 64, seed=5)
    base = sums(dev, args)
    weights = base.clone()
    out = F.attention_weighed(*args, weights)
    assert torch.equal(out, F.attention(*args))
    near(weights, base, args)


@pytest.mark.parametrize("per", [2, 5])
def test_rows_of_one_request_add_up(dev, per):
    """Neighbouring or not, in the order of the rows, the same bits every time."""
    from orinfer_b200.ops import functional as F
    args = list(batch(dev, [1030, 4, 300, 1], 8, 2, 128, per=per))
    order = torch.randperm(args[0].shape[0], generator=torch.Generator().manual_seed(1)).to(dev)
    base = sums(dev, args)
    got = []
    for _ in range(3):
        got.append(base.clone())
        F.attention_weighed(*args, got[-1], splits=2)
    near(got[0], base, args, per)
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
    for i in (0, 2, 3):
        args[i] = args[i][order].contiguous()
    weights = base.clone()
    F.attention_weighed(*args, weights, splits=2)
    near(weights, base, args, per)


def test_more_rows_than_a_cta_looks_at_once(dev):
    from orinfer_b200.ops import functional as F
    args = list(batch(dev, [40, 41, 42], 2, 2, 64, per=1))
    n = 700
    g = torch.Generator().manual_seed(2)
    req = torch.randint(0, 3, (n,), generator=g, dtype=torch.int32)
    pos = torch.randint(-1, 40, (n,), generator=g, dtype=torch.int32)
    args[0] = torch.randn(n, 2, 64, generator=g).half().to(dev)
    args[2], args[3] = req.to(dev), pos.to(dev)
    base = sums(dev, args)
    weights = base.clone()
    F.attention_weighed(*args, weights)
    near(weights, base, args, n)


def test_rows_that_see_nothing_and_rows_behind(dev):
    from orinfer_b200.ops import functional as F
    args = list(batch(dev, [200, 0, 77, 300], 4, 2, 128))
    args[2] = torch.tensor([0, 99, 2, 3], dtype=torch.int32, device=dev)     # row 1: any request
    base = sums(dev, args)
    weights = base.clone()
    out = F.attention_weighed(*args, weights, rows=3, out=torch.full((4, 512), 7.0, device=dev,
                                                                   dtype=torch.float16))
    assert bool((out[3] == 7.0).all()) and bool((out[1] == 0).all())
    assert torch.equal(weights[3], base[3]) and torch.equal(weights[1], base[1])
    args[3] = torch.tensor([199, -1, 76, -1], dtype=torch.int32, device=dev)
    args[2] = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=dev)
    near(weights, base, args)


def test_strided_sums_and_a_buffer_of_their_own(dev):
    from orinfer_b200.ops import functional as F
    args = batch(dev, [200, 700], 4, 2, 128)
    whole = torch.rand(5, 3, 4, args[4].shape[1] * 128 + 3, device=dev)
    view = whole[1:3, 0, 1:3]                        # slots and heads apart, an odd address
    before, keep = view.clone(), whole.clone()
    other = torch.full_like(before, -1.0)
    F.attention_weighed(*args, view, splits=2, weights_out=other)
    assert torch.equal(whole, keep)
    unseen = torch.arange(other.shape[2], device=dev)[None, :] > args[3][:, None]
    assert bool((other.transpose(1, 2)[unseen] == -1.0).all())
    F.attention_weighed(*args, view, splits=2)
    seen = ~unseen[:, None].expand_as(view)
    assert torch.equal(view[seen], other[seen])
    near(view, before, args)
    keep[1:3, 0, 1:3] = view
    assert torch.equal(whole, keep)


def test_queries_off_16_bytes(dev):
    from orinfer_b200.ops import functional as F
    args = list(batch(dev, [200, 700, 2000], 4, 2, 128))
    flat = torch.empty(args[0].numel() + 8, dtype=torch.float16, device=dev)
    args[0] = flat[1:1 + args[0].numel()].view(args[0].shape).copy_(args[0])
    base = sums(dev, args)
    weights = base.clone()
    assert torch.equal(F.attention_weighed(*args, weights), F.attention(*args))
    near(weights, base, args)


def test_captured_and_on_another_stream(dev):
    from orinfer_b200.ops import functional as F
    args = batch(dev, [200, 900], 8, 2, 128)
    base = sums(dev, args)
    weights = base.clone()
    F.attention_weighed(*args, weights, splits=2)
    want = weights.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        weights.copy_(base)
        F.attention_weighed(*args, weights, splits=2)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(weights, want)
    graphs = []
    for _ in range(2):                               # two graphs, each with a workspace of its own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = F.attention_weighed(*args, weights, splits=2)
        graphs.append((g, out))
    for g, out in graphs:
        weights.copy_(base)
        g.replay()
        assert torch.equal(weights, want)
        assert torch.equal(out, F.attention(*args, splits=2))


def test_keys_beyond_the_place_set_the_status(dev):
    from orinfer_b200.ops import functional as F, native
    args = batch(dev, [300, 40], 4, 2, 64)
    base = sums(dev, args)
    weights = base.clone()
    out = F.attention_weighed(*args, weights, max_kv_len=100)
    assert native.read_status() >> 16 == 6
    native.clear_status()
    assert torch.equal(out, F.attention(*args, max_kv_len=100))
    assert torch.equal(weights[0, :, 100:], base[0, :, 100:])
    short = base[:, :, :256].contiguous()
    F.attention_weighed(*args, short)
    assert native.read_status() >> 16 == 6
    native.clear_status()
