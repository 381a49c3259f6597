"""Attention of rows that share a prefix: what its kernels hand to one another, rows that have ended,
and how near the results come to 64 bits."""
import pytest
import torch

from orinfer_b200.ref import samples_ref as R
from test_attention_shared_gpu import batch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(cuda):
    return cuda


def plan_of(args, spec, dev, **kw):
    from orinfer_b200.ops import functional as F
    q, pos = args[0], args[3]
    return F.SharedPrefix(spec, q.shape[0], **{**dict(
        qh=q.shape[1], kvh=args[5].shape[2], head_dim=q.shape[2], max_kv_len=int(pos.max()) + 1,
        device=dev, force=True), **kw})


@pytest.mark.parametrize("rows,shared,own,qh,kvh,d", [
    (40, 2048, 30, 8, 2, 128), (150, 512, 200, 16, 8, 128), (3, 1024, 2500, 4, 2, 64),
    (9, 640, 90, 16, 2, 256)])
def test_the_row_kernels_see_what_came_before_the_prefix(dev, rows, shared, own, qh, kvh, d):
    """A long kernel writes the queries, the own keys' scales and the positions just ahead of each call,
    and zeros stand there until then.  The word by which the kernel of the prefix hands on what it has
    waited for is clear behind every call, so that no call finds an earlier one's."""
    from orinfer_b200.ops import functional as F
    spec, args = batch(dev, [(shared, [shared + 1 + (7 * r) % own for r in range(rows)])], qh, kvh, d,
                       seed=rows, fill=False)
    q, gate, req, pos, table, kc, vc, ks, vs = args
    plan = plan_of(args, spec, dev)
    assert plan.items is not None
    word = plan.part_buffer[-1:].view(torch.int32)
    want = F.attention_shared(*args, plan).clone()
    torch.cuda.synchronize()
    assert int(word) == 0
    late = [t.clone() for t in (q, pos, ks)]
    big = torch.empty(1 << 26, device=dev)
    got = torch.empty(8, *want.shape, dtype=want.dtype, device=dev)

    def step(out):
        for t in (q, pos, ks):
            t.zero_()
        big.normal_()
        for t, v in zip((q, pos, ks), late):
            t.copy_(v)
        F.attention_shared(*args, plan, out=out)

    for out in got:
        step(out)
    torch.cuda.synchronize()
    assert bool((got == want).all()) and int(word) == 0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for out in got:
            step(out)
    for _ in range(2):
        got.zero_()
        graph.replay()
        assert bool((got == want).all()) and int(word) == 0


def near(ref, size, reach):
    """What arithmetic in FP32 leaves, and the output's rounding, 2^-11 of it at most.  A weight of two
    BF16 numbers is off by 2^-9 of 2^-9 of it; a score, a sum of up to 256 products of the queries with
    integers and FP16 scales, by 2^-19 of its terms' magnitudes (2^-23 for each of its up to sixteen
    additions of sixteen products, which may be cut off); the sums over up to 1200 keys, by 2^-23 for
    each of 75 additions of sixteen.  FP16 ends at 2^-25."""
    return 2.0 ** -11 * ref.abs() + size * (2.0 ** -18 + 2.0 ** -19 * reach + 75 * 2.0 ** -23) + 2.0 ** -24


def assert_near(args, out, reach=None):
    ref, size, all_reach = R.attention_rows(*args)
    reach = all_reach if reach is None else reach
    off = ((out.double().view_as(ref) - ref).abs() / near(ref, size, reach)).max()
    assert float(off) <= 1, float(off)


@pytest.mark.parametrize("qh,kvh,d", [(2, 2, 64), (8, 2, 64), (8, 2, 128), (10, 2, 128), (8, 1, 128),
                                      (8, 1, 256), (4, 2, 256)])
@pytest.mark.parametrize("score", [1.0, 4.0])
def test_weights_have_the_bits_that_decode_attention_has(dev, qh, kvh, d, score):
    """Few heavy keys, whose roundings do not cancel, and many light ones; nothing but the output is
    rounded to FP16."""
    from orinfer_b200.ops import functional as F
    spec, args = batch(dev, [(1024, [1024 + n for n in (0, 1, 40, 130)]), (3, [3, 3, 2, 1]),
                             (64, [64, 70, 65]), (130, [130, 131])], qh, kvh, d, seed=3, score=score,
                       gated=d == 256)
    plan = plan_of(args, spec, dev)
    assert plan.items is not None
    assert_near(args, F.attention_shared(*args, plan))


@pytest.mark.parametrize("qh,kvh,d", [(4, 2, 64), (8, 2, 128), (8, 1, 256)])
@pytest.mark.parametrize("key", [0, 70, 500, 1023])
@pytest.mark.parametrize("binades", [10, 18, 26])
def test_a_large_value_scale_without_weight_costs_nothing(dev, qh, kvh, d, key, binades):
    """One key whose values are 2^binades times the others' and whose weight is e^-50 or less."""
    from orinfer_b200.ops import functional as F
    spec, args = batch(dev, [(1024, [1024 + n for n in (0, 3, 200)])], qh, kvh, d, seed=binades,
                       scales=(2.0 ** -12, 2.0 ** -11), fill=False)
    q, gate, req, pos, table, kc, vc, ks, vs = args
    q.abs_().add_(0.25)
    page, at = int(table[int(req[0]), key // 128]), key % 128
    kc[page, at], ks[page, at], vs[page, at] = 0, 0.06, 2.0 ** (binades - 12)
    _, _, reach = R.attention_rows(*args)            # (of the keys that have a weight)
    kc[page, at] = -127
    assert_near(args, F.attention_shared(*args, plan_of(args, spec, dev)), reach)


@pytest.mark.parametrize("qh,kvh,d", [(4, 2, 64), (8, 2, 128), (8, 1, 256)])
@pytest.mark.parametrize("key", [0, 1000])
@pytest.mark.parametrize("scale", [0.0, 2.0 ** -24])
def test_a_key_that_takes_the_weight_and_has_no_value(dev, qh, kvh, d, key, scale):
    """What the other keys give is small beside it in weight, and all that there is in value."""
    from orinfer_b200.ops import functional as F
    spec, args = batch(dev, [(1024, [1024 + n for n in (0, 3, 200)])], qh, kvh, d, seed=key,
                       scales=(0.01, 0.02), score=0.5, fill=False)
    q, gate, req, pos, table, kc, vc, ks, vs = args
    q.abs_().add_(0.25)
    vs.mul_(1000.0)
    page, at = int(table[int(req[0]), key // 128]), key % 128
    kc[page, at], ks[page, at], vs[page, at] = 127, 0.02, scale
    assert_near(args, F.attention_shared(*args, plan_of(args, spec, dev)))


@pytest.mark.parametrize("qh,kvh,d", [(4, 2, 64), (8, 2, 128), (8, 1, 256)])
@pytest.mark.parametrize("way", ["up", "down", "steps"])
def test_references_that_have_to_move_far(dev, qh, kvh, d, way):
    """Scores over several hundred binades, that climb, fall, or leap every 160 keys."""
    from orinfer_b200.ops import functional as F
    spec, args = batch(dev, [(1024, [1024 + n for n in (0, 3, 200)])], qh, kvh, d, seed=len(way),
                       score=0.5, fill=False)
    q, gate, req, pos, table, kc, vc, ks, vs = args
    q.abs_().add_(0.25)
    kc.copy_(kc.abs().clamp(min=100))
    at = torch.arange(1024)
    ramp = {"up": at, "down": 1023 - at, "steps": at // 160 * 170}[way].to(dev) * 2e-4
    pages = table[req[0].long(), :8].long()
    ks[pages] = ramp.view(8, 128, 1, 1).half().expand_as(ks[pages])
    assert_near(args, F.attention_shared(*args, plan_of(args, spec, dev)))


@pytest.mark.parametrize("qh,kvh,d", [(4, 2, 64), (8, 2, 128), (8, 1, 128), (8, 1, 256)])
@pytest.mark.parametrize("nobody", [0, -1, 1 << 20])
def test_rows_that_have_ended_anywhere_in_a_group(dev, qh, kvh, d, nobody):
    """Rows at position -1, whose table rows have been given back or whose requests do not exist, at the
    start of every tile of 128 / rep rows, between the others, and as whole tiles and groups; the plan
    stays.  The others see their prefix, those give zeros."""
    from orinfer_b200.ops import functional as F
    per = 128 // (qh // kvh)
    rows = 3 * per + 2
    spec, args = batch(dev, [(640, [641 + r % 90 for r in range(rows)]), (256, [300, 280])], qh, kvh, d,
                       seed=d, gated=d == 256)
    q, gate, req, pos, table, *cache = args
    ended = [0, 1, 5, per, 3 * per, 3 * per + 1, rows, rows + 1] + list(range(2 * per, 3 * per))
    for r in ended:
        table[int(req[r])] = 0
    pos[ended] = -1
    if nobody:
        req[ended] = nobody
    plan = plan_of((q, gate, req, pos, table, *cache), spec, dev, max_kv_len=731)
    assert plan.items is not None
    plan.part_buffer[:-1] = float("nan")             # what nobody writes is not read
    out = F.attention_shared(q, gate, req, pos, table, *cache, plan)
    assert bool((out[ended] == 0).all())
    safe = req.clone()
    safe[ended] = 0
    assert_near((q, gate, safe, pos, table, *cache), out)


@pytest.mark.parametrize("qh,kvh,d", [(4, 2, 64), (8, 2, 128), (8, 1, 256)])
@pytest.mark.parametrize("first", [1, 63, 64, 100, 129, 500])
def test_a_first_row_that_ends_inside_the_prefix(dev, qh, kvh, d, first):
    """Its table row has nothing that can be read behind its last page, and the rows behind it see all.
    Where nobody sees the rest of a prefix, nothing of it is read."""
    from orinfer_b200.ops import functional as F
    groups = [(1024, [first, 1024, 1030, 900]), (1024, [first, max(1, first // 2)])]
    spec, args = batch(dev, groups, qh, kvh, d, seed=first)
    req, pos, table = args[2], args[3], args[4]
    for r in (0, 4, 5):
        table[int(req[r]), (int(pos[r]) + 128) // 128:] = -7
    plan = plan_of(args, spec, dev)
    plan.part_buffer[:-1] = float("nan")
    assert_near(args, F.attention_shared(*args, plan))


@pytest.mark.parametrize("qh,kvh,d", [(4, 2, 64), (8, 2, 128), (8, 1, 256)])
@pytest.mark.parametrize("key", [1, 40, 64, 200, 1023])
@pytest.mark.parametrize("what", [float("inf"), float("nan")])
def test_a_key_that_a_row_does_not_see_may_be_no_number(dev, qh, kvh, d, key, what):
    """Shared keys that some rows of the group see and others end ahead of."""
    from orinfer_b200.ops import functional as F
    spec, args = batch(dev, [(1024, [key, 1030, max(1, key - 1), max(1, key // 2), 1024])], qh, kvh, d,
                       seed=key)
    req, table, ks, vs = args[2], args[4], args[7], args[8]
    page = int(table[int(req[1]), key // 128])
    clean = [t.clone() for t in (ks, vs)]
    vs[page, key % 128] = what
    plan = plan_of(args, spec, dev)
    assert not bool(F.attention_shared(*args, plan)[1].isfinite().any())
    ks[page, key % 128] = what
    out = F.attention_shared(*args, plan)
    ref, size, reach = R.attention_rows(*args[:7], *clean)
    for r in (0, 2, 3):
        off = (out[r].double() - ref[r]).abs() / near(ref[r], size[r], reach[r])
        assert float(off.max()) <= 1 and bool(out[r].isfinite().all())


@pytest.mark.parametrize("qh,kvh,d", [(16, 8, 64), (32, 8, 128), (32, 4, 128), (16, 2, 256)])
@pytest.mark.parametrize("listed", [True, False])
def test_a_long_row_beside_short_ones(dev, qh, kvh, d, listed):
    """In no group, and behind a shorter prefix; most parts of the short rows are empty then."""
    from orinfer_b200.ops import functional as F
    lens = [1024 + n for n in (1, 30, 60, 0, 90, 9)]
    spec, args = batch(dev, [(1024, lens), (128, [4000, 140])], qh, kvh, d, seed=d, loners=(4100, 3, 0),
                       gated=d == 256)
    bounds = [n + 64 for n in lens] + [4064, 204, 4164, 64, 0]
    plan = plan_of(args, spec, dev, max_kv_len=bounds if listed else 4164)
    assert plan.splits > 1
    out = F.attention_shared(*args, plan)
    ref, size, reach = R.attention_rows(*args)
    # (the sums of 4100 keys, 2^-23 for each of 257 additions of sixteen)
    off = (out.double().view_as(ref) - ref).abs() / (near(ref, size, reach) + size * 182 * 2.0 ** -23)
    assert float(off.max()) <= 1 and bool((out[-1] == 0).all())
