"""Cutting requests down to the keys with the most weight, against the host statement."""
import math

import pytest
import torch

from orinfer_b200.ref import eviction_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(cuda):
    return cuda


def state(seed, lens, *, slots=None, spare=40, kvh=2, d=64, layers=2, share=0, more=0, ties=False,
          reserve=0):
    """Requests of these lengths in random slots, on random pages; the first ``share`` pages are
    everybody's that has as many; ``reserve`` more pages stand behind a request's tokens."""
    g = torch.Generator().manual_seed(seed)
    slots = slots or len(lens) + 3
    where = torch.randperm(slots, generator=g).tolist()
    counts = [-(-n // 128) for n in lens]
    width = max(counts + [1]) + reserve + 1
    pages = share + sum(counts) + reserve * len(lens) + spare + 1
    order = (torch.randperm(pages - 1, generator=g) + 1).tolist()
    front = [order.pop() for _ in range(share)]
    table = torch.zeros(slots, width, dtype=torch.int32)
    length, refs = torch.zeros(slots, dtype=torch.int32), torch.zeros(pages, dtype=torch.int32)
    used = []
    for n, k in zip(lens, counts):
        s = where.pop()
        common = min(share, n // 128)
        row = front[:common] + [order.pop() for _ in range(k - common + reserve)]
        table[s, :len(row)], length[s] = torch.tensor(row, dtype=torch.int32), n
        refs[row] += 1
        used.append(s)
    byte = lambda: torch.randint(-128, 128, (layers, pages, 128, kvh, d), generator=g).to(torch.int8)
    half = lambda: torch.randn(layers, pages, 128, kvh, d // 64, generator=g).half()
    cap = width * 128 + more
    weights = torch.rand(layers, slots, kvh, cap, generator=g) ** 6
    if ties:
        weights = (weights * 4).floor() * 0.25
    return table, length, refs, weights, (byte(), byte(), half(), half()), used


def i32(v, dev="cpu"):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def check(dev, st, named, keep, first=0, recent=0, inplace=False, status=0):
    from orinfer_b200.ops import functional as F
    table, lens, refs, weights, cache, _ = st
    gpu = [t.to(dev) for t in cache]
    tables = [t.to(dev) for t in (table, lens, refs)]
    w = weights.to(dev)
    other = None if inplace else torch.full_like(w, -3.0)
    handle = F.KeyCache(*(t.unbind(0) for t in gpu))
    got = F.evict_keys(handle, *tables, w, i32(named, dev), keep, first=first, recent=recent,
                       out=tables if inplace else None, weights_out=other)
    *want, code = R.evict_keys(*(list(t.unbind(0)) for t in cache), table, lens, refs, weights,
                               i32(named), keep, first, recent)
    assert code == status and int(got[3]) == status
    for a, b in zip(got[:3], want[:3]):
        assert torch.equal(a.cpu(), b)
    for a, b in zip(gpu, cache):
        assert torch.equal(a.cpu(), b)
    same = lambda a, b: torch.equal(a.cpu().view(torch.int32), b.view(torch.int32))
    if inplace:
        assert same(w, want[3])
    else:
        assert same(w, weights)
        rows = [s for s in range(table.shape[0]) if s in named]
        assert same(other[:, rows], want[3][:, rows])
        rest = [s for s in range(table.shape[0]) if s not in named]
        assert bool((other[:, rest] == -3.0).all())
        assert all(torch.equal(a.cpu(), b) for a, b in zip(tables, (table, lens, refs)))
    return got


@pytest.mark.parametrize("kvh,d", [(2, 64), (1, 64), (3, 128), (8, 128), (2, 256)])
@pytest.mark.parametrize("inplace", [False, True])
def test_batch(dev, kvh, d, inplace):
    st = state(kvh + d, [700, 129, 256, 255, 1500, 130], kvh=kvh, d=d)
    check(dev, st, st[5][:5], 200, 4, 32, inplace)


@pytest.mark.parametrize("keep,first,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (127, 0, 0), (128, 64, 64),
                                               (129, 0, 128), (255, 200, 55), (384, 3, 7), (1024, 0, 0),
                                               (1087, 0, 0)])
@pytest.mark.parametrize("ties", [False, True])
def test_bounds(dev, keep, first, recent, ties):
    st = state(keep, [1088, 1, 0, 1087, 2049], ties=ties, layers=1)
    check(dev, st, st[5], keep, first, recent)


def test_one_key_more_than_stays(dev):
    for n in (2, 128, 129, 257, 1025):
        check(dev, state(n, [n]), [state(n, [n])[5][0]], n - 1)


@pytest.mark.parametrize("inplace", [False, True])
def test_shared_pages_are_left_to_the_others(dev, inplace):
    """Samples of one prompt, of which some are cut."""
    st = state(5, [900, 901, 1023, 700, 300], share=5)
    check(dev, st, st[5][:3], 333, 4, 100, inplace)
    st = state(6, [900, 901, 1023, 700, 300], share=5)
    check(dev, st, st[5], 256, 0, 256, inplace)


def test_pages_that_stand_ready_are_given_back(dev):
    st = state(8, [300, 640, 100], reserve=3)
    check(dev, st, st[5], 150)


def test_a_slot_that_is_named_again(dev):
    st = state(9, [300, 640, 100])
    a, b, c = st[5]
    check(dev, st, [b, a, b, c, a, a], 150, inplace=True)
    check(dev, state(9, [300, 640, 100]), [b, a, b, c, a, a], 150)


def test_nothing_to_do(dev):
    st = state(10, [300, 640])
    check(dev, st, [], 100)
    check(dev, st, [], 100, inplace=True)
    check(dev, st, st[5], 640)


def test_weights_of_every_kind(dev):
    """Negative ones, infinities, zeros of both signs, subnormal numbers and such that are none."""
    for seed in range(4):
        st = state(seed, [1500, 600], layers=3)
        w = st[3]
        g = torch.Generator().manual_seed(seed)
        kind = torch.randint(0, 9, w.shape, generator=g)
        for i, x in enumerate([0.0, -0.0, math.inf, -math.inf, math.nan, 1e-42, -2.5, -1e-42]):
            w[kind == i] = x
        w[0, :, :, ::2] = -math.nan
        check(dev, st, st[5], 400, 5, 20)


def test_equal_weights_keep_the_earlier_keys(dev):
    st = state(12, [3000], layers=1)
    st[3][:] = 0.25
    check(dev, st, st[5], 1500, 10, 100)


@pytest.mark.parametrize("spare,status", [(9, 1), (10, 0)])
def test_too_few_free_pages_change_nothing(dev, spare, status):
    for inplace in (False, True):
        st = state(13, [1000, 700, 100], spare=spare)
        check(dev, st, st[5], 600, inplace=inplace, status=status)


@pytest.mark.parametrize("what", ["slot", "negative", "length", "page", "page0", "held"])
@pytest.mark.parametrize("inplace", [False, True])
def test_wrong_requests_change_nothing(dev, what, inplace):
    st = state(14, [1000, 700, 100])
    table, lens, refs, _, _, used = st
    named = list(used)
    if what == "slot":
        named.append(table.shape[0])
    elif what == "negative":
        named.append(-1)
    elif what == "length":
        lens[used[2]] = table.shape[1] * 128 + 1
    elif what == "page":
        table[used[0], 2] = refs.shape[0]
    elif what == "page0":
        table[used[0], 2] = 0
    else:
        refs[table[used[0], 2]] = 0
    check(dev, st, named, 300, inplace=inplace, status=2)


def test_many_requests_and_pages(dev):
    """More than the planning CTA has threads."""
    lens = [130 + i % 200 for i in range(1100)]
    st = state(15, lens, spare=2300, layers=1, kvh=1, slots=1200)
    check(dev, st, st[5], 128)


def test_capacity_beyond_the_table(dev):
    st = state(16, [700, 300], more=37)
    check(dev, st, st[5], 256)
    check(dev, st, st[5], 256, inplace=True)


def test_captured_and_repeated(dev):
    from orinfer_b200.ops import functional as F
    table, lens, refs, weights, cache, used = state(17, [900, 500, 70])
    gpu = [t.to(dev) for t in cache]
    args = [t.to(dev) for t in (table, lens, refs, weights)]
    handle = F.KeyCache(*(t.unbind(0) for t in gpu))
    named, other = i32(used, dev), torch.zeros_like(args[3])
    F.evict_keys(handle, *args, named, 300, weights_out=other)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = F.evict_keys(handle, *args, named, 300, weights_out=other)
    *want, _ = R.evict_keys(*(list(t.unbind(0)) for t in cache), table, lens, refs, weights, i32(used), 300)
    other.zero_()
    for _ in range(2):
        g.replay()
    assert int(got[3]) == 0
    for a, b in zip(got[:3], want[:3]):
        assert torch.equal(a.cpu(), b)
    assert torch.equal(other[:, used].cpu(), want[3][:, used])
    for a, b in zip(gpu, cache):
        assert torch.equal(a.cpu(), b)


def test_attention_over_what_is_left(dev):
    """A cut request's attention is that over the kept keys alone."""
    from orinfer_b200.ops import functional as F
    table, lens, refs, weights, cache, used = state(18, [900, 500], layers=1, kvh=2, d=64)
    cache = [t if t.dtype == torch.int8 else t.abs() * 0.01 for t in cache]
    gpu = [t.to(dev) for t in cache]
    handle = F.KeyCache(*(t.unbind(0) for t in gpu))
    a = [t.to(dev) for t in (table, lens, refs, weights)]
    t, l, *_ = F.evict_keys(handle, *a, i32(used, dev), 300, first=2, recent=50)
    g = torch.Generator().manual_seed(1)
    q = torch.randn(2, 4, 64, generator=g).half().to(dev)
    pos = l[used] - 1
    got = F.attention(q, None, i32(used, dev), pos, t, *(x[0] for x in gpu))
    for r, s in enumerate(used):
        for h in range(2):
            stay = torch.tensor(R.kept_keys(weights[0, s, h], int(lens[s]), 300, 2, 50))
            page, at = table[s, stay // 128].long(), stay % 128
            k = cache[0][0, page, at, h].double() * cache[2][0, page, at, h].double()
            v = cache[1][0, page, at, h].double() * cache[3][0, page, at, h].double()
            x = q[r, 2 * h:2 * h + 2].double().cpu()
            want = torch.softmax(x @ k.t() / 8, 1) @ v
            off = (got[r].view(4, 64)[2 * h:2 * h + 2].double().cpu() - want).abs()
            assert float(off.max()) <= 2.0 ** -9 * float(v.abs().max())
