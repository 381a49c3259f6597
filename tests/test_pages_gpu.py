"""Copying, forking, freeing and compacting pages of a cache, against the host statements."""
import pytest
import torch

from orinfer_b200.ref import samples_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(cuda):
    return cuda


def state(seed, *, slots, pages, width, lens, kvh=2, d=64, layers=2, share=0):
    """Requests of these lengths in random slots, on random pages; ``share`` more slots hold the
    whole pages of the first.  Everything on the CPU."""
    g = torch.Generator().manual_seed(seed)
    order = (torch.randperm(pages - 1, generator=g) + 1).tolist()
    where = torch.randperm(slots, generator=g).tolist()
    table = torch.zeros(slots, width, dtype=torch.int32)
    length, refs = torch.zeros(slots, dtype=torch.int32), torch.zeros(pages, dtype=torch.int32)
    used = []
    for n in lens:
        s, k = where.pop(), (n + 127) // 128
        mine = [order.pop() for _ in range(k)]
        table[s, :k], length[s] = torch.tensor(mine, dtype=torch.int32), n
        refs[mine] += 1
        used.append(s)
    for _ in range(share):
        s, k = where.pop(), lens[0] // 128
        table[s, :k], length[s] = table[used[0], :k], k * 128
        refs[table[s, :k].long()] += 1
        used.append(s)
    mk = lambda last, dt: torch.randint(-120, 120, (pages, 128, kvh, last), generator=g).to(dt)
    cache = [t for _ in range(layers) for t in (mk(d, torch.int8), mk(d, torch.int8),
                                                mk(d // 64, torch.float16),
                                                mk(d // 64, torch.float16))]
    return table, length, refs, cache, used, where


def _to(dev, *ts):
    return [t.to(dev) for t in ts]


def _unaligned(t, by=1):
    flat = torch.empty(t.numel() + 16, dtype=t.dtype, device=t.device)
    out = flat[by:by + t.numel()].view(t.shape)
    out.copy_(t)
    return out


def i32(v, dev="cpu"):
    return torch.tensor(v, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("kvh,d", [(2, 64), (1, 64), (3, 128), (8, 128), (2, 256)])
@pytest.mark.parametrize("inplace", [False, True])
def test_fork(dev, kvh, d, inplace):
    from orinfer_b200.ops import functional as F
    lens = [1, 127, 128, 129, 300, 511, 640]
    table, length, refs, cache, used, free = state(kvh + d, slots=40, pages=60, width=7, lens=lens,
                                                   kvh=kvh, d=d, share=2)
    parents = [used[i % len(used)] for i in range(20)]
    children = free[:20]
    gpu = _to(dev, *cache)
    tables = _to(dev, table, length, refs)
    before = [t.clone() for t in tables]
    handle = F.CachePages(gpu)
    got = F.fork_pages(handle, *tables, i32(parents, dev), i32(children, dev),
                       out=tables if inplace else None)
    want = R.fork_pages(cache, table, length, refs, i32(parents), i32(children))
    assert want[3] == 0 and int(got[3]) == 0
    for a, b in zip(got[:3], want[:3]):
        assert torch.equal(a.cpu(), b)
    for a, b in zip(gpu, cache):
        assert torch.equal(a.cpu(), b)
    for t, o, a in zip(tables, before, got):
        assert (a is t) if inplace else torch.equal(t, o)


@pytest.mark.parametrize("by", [1, 2, 4, 8])
def test_fork_of_unaligned_tensors(dev, by):
    """Tensors at any address: INT8 ones ``by`` bytes and FP16 ones twice as far past 16."""
    from orinfer_b200.ops import functional as F
    table, length, refs, cache, used, free = state(by, slots=12, pages=30, width=4,
                                                   lens=[100, 333, 127], kvh=1, d=64)
    gpu = [_unaligned(t.to(dev), by) for t in cache]
    args = (i32([used[0], used[1], used[2], used[1]]), i32(free[:4]))
    got = F.fork_pages(F.CachePages(gpu), *_to(dev, table, length, refs), *_to(dev, *args))
    want = R.fork_pages(cache, table, length, refs, *args)
    assert int(got[3]) == want[3] == 0
    for a, b in zip([*got[:3], *gpu], [*want[:3], *cache]):
        assert torch.equal(a.cpu(), b)


def test_fork_of_many_slots_and_pages(dev):
    """More pairs, slots and pages than the planning CTA has threads."""
    from orinfer_b200.ops import functional as F
    lens = [130, 77, 256, 5]
    table, length, refs, cache, used, free = state(7, slots=1500, pages=4000, width=3, lens=lens,
                                                   kvh=1, layers=1)
    refs[1:2500] = refs[1:2500].clamp(min=1)         # the free pages lie behind
    n = 1300
    args = (i32([used[i % 4] for i in range(n)]), i32(free[:n]))
    gpu = _to(dev, *cache)
    got = F.fork_pages(F.CachePages(gpu), *_to(dev, table, length, refs), *_to(dev, *args))
    want = R.fork_pages(cache, table, length, refs, *args)
    assert int(got[3]) == want[3] == 0
    for a, b in zip([*got[:3], *gpu], [*want[:3], *cache]):
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("by", [0, 4, 1])
@pytest.mark.parametrize("lens", [[333, 70], [128, 1, 511], [257]])
def test_children_that_get_their_parents_page_from_one_read(dev, by, lens):
    """More pairs and tensors than have CTAs of their own: a parent's page is read for all of its
    children, whose pages are each of their own."""
    from orinfer_b200.ops import functional as F
    table, length, refs, cache, used, free = state(len(lens), slots=50, pages=60, width=5, lens=lens,
                                                   kvh=8, d=128)
    n = 40
    gpu = [_unaligned(t.to(dev), by) for t in cache]
    handle = F.CachePages(gpu)
    assert n * len(handle.units) > 8 * 148
    args = (i32([used[i * i % len(lens)] for i in range(n)]), i32(free[:n]))
    tables = _to(dev, table, length, refs)
    got = F.fork_pages(handle, *tables, *_to(dev, *args), out=tables)
    want = R.fork_pages(cache, table, length, refs, *args)
    assert int(got[3]) == want[3] == 0
    for a, b in zip([*got[:3], *gpu], [*want[:3], *cache]):
        assert torch.equal(a.cpu(), b)


def test_forks_that_cannot_be_change_nothing(dev):
    from orinfer_b200.ops import functional as F
    table, length, refs, cache, used, free = state(3, slots=12, pages=12, width=4,
                                                   lens=[300, 64, 128])
    a, b, c = used
    bad = table.clone()
    bad[a, 1] = 99                                   # a page that does not exist
    held = refs.clone()
    held[table[a, 0]] = 0                            # a page that nobody holds
    cases = [(table, refs, [a], [a], 2), (table, refs, [a], [b], 2),
             (table, refs, [a, b], [free[0]] * 2, 2), (table, refs, [12], [free[0]], 2),
             (table, refs, [-1], [free[0]], 2), (table, refs, [a], [12], 2),
             (table, refs, [a], [-3], 2), (table, refs, [free[1], a], [free[0], free[1]], 2),
             (bad, refs, [a], [free[0]], 2), (table, held, [a], [free[0]], 2),
             (table, refs, [a] * 8, free[:8], 1), (table, refs, [c] * 8, free[:8], 0),
             (table, refs, [a] * 7, free[:7], 1), (table, refs, [a] * 6, free[:6], 0),
             (table, refs, [free[1]], [free[0]], 0)]
    for t0, r0, parents, children, status in cases:
        gpu = _to(dev, *cache)
        got = F.fork_pages(F.CachePages(gpu), *_to(dev, t0, length, r0), i32(parents, dev),
                           i32(children, dev))
        copy = [x.clone() for x in cache]
        want = R.fork_pages(copy, t0, length, r0, i32(parents), i32(children))
        assert int(got[3]) == status == want[3], (parents, children)
        for x, y in zip([*got[:3], *gpu], [*want[:3], *copy]):
            assert torch.equal(x.cpu(), y)


def test_a_long_length_in_the_table_is_refused(dev):
    from orinfer_b200.ops import functional as F
    table, length, refs, cache, used, free = state(5, slots=6, pages=9, width=2, lens=[200])
    for n in (257, -1, 2 ** 31 - 1):
        length[used[0]] = n
        got = F.fork_pages(F.CachePages(_to(dev, *cache)), *_to(dev, table, length, refs),
                           i32(used, dev), i32(free[:1], dev))
        assert int(got[3]) == 2 and torch.equal(got[0].cpu(), table)


@pytest.mark.parametrize("inplace", [False, True])
def test_free(dev, inplace):
    from orinfer_b200.ops import functional as F
    table, length, refs, cache, used, free = state(9, slots=300, pages=700, width=7,
                                                   lens=[640, 5, 128, 300] * 20, share=30)
    gone = i32(used[:5] + used[40:110:2] + [used[3], used[3], free[0]])
    tables = _to(dev, table, length, refs)
    before = [t.clone() for t in tables]
    got = F.free_pages(*tables, gone.to(dev), out=tables if inplace else None)
    for a, b in zip(got, R.free_pages(table, length, refs, gone)):
        assert torch.equal(a.cpu(), b)
    for t, o, a in zip(tables, before, got):
        assert (a is t) if inplace else torch.equal(t, o)


def test_free_reports_what_is_nobodys(dev):
    from orinfer_b200.ops import functional as F, native
    table, length, refs, cache, used, free = state(2, slots=5, pages=9, width=3, lens=[300])
    wrong = table.clone()
    wrong[used[0], 2] = 77
    twice = refs.clone()
    twice[table[used[0], 1]] = 0
    for t0, r0, slots in ((table, refs, [5]), (table, refs, [-1]), (wrong, refs, used),
                          (table, twice, used)):
        assert native.read_status() == 0
        t, l, r = F.free_pages(*_to(dev, t0, length, r0), i32(slots, dev))
        assert native.read_status() >> 16 == 6       # a rejected index
        native.clear_status()
        assert bool((r >= 0).all())


@pytest.mark.parametrize("pages,live", [(2, 0), (2, 1), (9, 4), (40, 39), (130, 60), (1500, 700),
                                        (2100, 100), (2049, 2000)])
@pytest.mark.parametrize("inplace", [False, True])
def test_compact(dev, pages, live, inplace):
    from orinfer_b200.ops import functional as F
    g = torch.Generator().manual_seed(pages)
    held = (torch.randperm(pages - 1, generator=g) + 1)[:live]
    refs = torch.zeros(pages, dtype=torch.int32)
    refs[held] = torch.randint(1, 4, (live,), generator=g, dtype=torch.int32)
    table = torch.zeros(10, live // 10 + 2, dtype=torch.int32)
    table.view(-1)[:live] = held.int()
    mk = lambda last, dt: torch.randint(-120, 120, (pages, 128, 1, last), generator=g).to(dt)
    cache = [mk(64, torch.int8), mk(1, torch.float16), mk(64, torch.int8), mk(1, torch.float16)]
    gpu = _to(dev, *cache)
    tables = _to(dev, table, refs)
    got = F.compact_pages(F.CachePages(gpu), *tables, out=tables if inplace else None)
    want = R.compact_pages(cache, table, refs)
    for a, b in zip([*got, *gpu], [*want, *cache]):
        assert torch.equal(a.cpu(), b)
    if not inplace:
        assert torch.equal(tables[0].cpu(), table) and torch.equal(tables[1].cpu(), refs)


def test_copy_pages(dev):
    from orinfer_b200.ops import functional as F
    *_, cache, _, _ = state(1, slots=4, pages=20, width=2, lens=[1], kvh=3, d=128)
    gpu = _to(dev, *cache)
    handle = F.CachePages(gpu)
    src, dst, tokens = [3, 3, 7, 19], [1, 2, 5, 0], [128, 1, 77, 0]
    F.copy_pages(handle, i32(src, dev), i32(dst, dev), i32(tokens, dev))
    for t in cache:
        for s, d, n in zip(src, dst, tokens):
            t[d, :n] = t[s, :n]
    assert all(torch.equal(a.cpu(), b) for a, b in zip(gpu, cache))
    F.copy_pages(handle, i32([1], dev), i32([9], dev))
    for t in cache:
        t[9] = t[1]
    assert all(torch.equal(a.cpu(), b) for a, b in zip(gpu, cache))
    F.copy_pages(handle, i32([], dev), i32([], dev))


def test_copy_pages_leaves_out_what_does_not_exist(dev):
    from orinfer_b200.ops import functional as F, native
    *_, cache, _, _ = state(1, slots=4, pages=6, width=2, lens=[1])
    for src, dst, tokens in ((6, 1, 128), (1, 6, 128), (-1, 1, 5), (1, -2, 5), (1, 2, 129)):
        gpu = _to(dev, *cache)
        F.copy_pages(F.CachePages(gpu), i32([src], dev), i32([dst], dev), i32([tokens], dev))
        assert native.read_status() >> 16 == 6
        native.clear_status()
        assert all(torch.equal(a.cpu(), b) for a, b in zip(gpu, cache))


def test_a_pool_with_offsets_past_32_bits(dev):
    from orinfer_b200.ops import functional as F
    pages = (2 ** 31 + 2 ** 28) // (128 * 1024)
    big = torch.zeros(pages, 128, 8, 128, dtype=torch.int8, device=dev)
    big[-1] = torch.randint(-9, 9, (128, 8, 128), dtype=torch.int8)
    F.copy_pages(F.CachePages([big]), i32([pages - 1], dev), i32([pages - 3], dev),
                 i32([100], dev))
    assert torch.equal(big[-3, :100], big[-1, :100]) and bool((big[-3, 100:] == 0).all())


def test_fork_free_and_compact_in_a_graph(dev):
    """A captured round in place: fork, free the parent, compact."""
    from orinfer_b200.ops import functional as F
    table, length, refs, cache, used, free = state(21, slots=16, pages=50, width=6,
                                                   lens=[700, 129, 380])
    parents, children = i32([used[0], used[1], used[0]]), i32(free[:3])
    gone = i32([used[0]])
    first = _to(dev, table, length, refs, *cache)
    live = [t.clone() for t in first]
    t, l, r, gpu = live[0], live[1], live[2], live[3:]
    handle = F.CachePages(gpu)
    d = _to(dev, parents, children, gone)

    def round_():
        F.fork_pages(handle, t, l, r, d[0], d[1], out=(t, l, r))
        F.free_pages(t, l, r, d[2], out=(t, l, r))
        return F.compact_pages(handle, t, r, out=(t, r))[2]

    round_()
    torch.cuda.synchronize()
    wt, wl, wr, status = R.fork_pages(cache, table, length, refs, parents, children)
    wt, wl, wr = R.free_pages(wt, wl, wr, gone)
    wt, wr, _ = R.compact_pages(cache, wt, wr)
    want = [wt, wl, wr, *cache]
    assert status == 0 and all(torch.equal(a.cpu(), b) for a, b in zip(live, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        round_()
    for _ in range(3):
        for a, b in zip(live, first):
            a.copy_(b)
        graph.replay()
        assert all(torch.equal(a.cpu(), b) for a, b in zip(live, want))


def test_refusals(dev):
    from orinfer_b200.ops import functional as F
    from orinfer_b200.ops.native import KernelError
    table, length, refs, cache, used, free = state(1, slots=6, pages=9, width=2, lens=[200])
    gpu = _to(dev, *cache)
    t, l, r = _to(dev, table, length, refs)
    handle = F.CachePages(gpu)
    p, c = i32(used, dev), i32(free[:1], dev)
    for tensors in ([], [gpu[0], gpu[1][:5]], [gpu[0].transpose(2, 3)], [gpu[0][:, :64]],
                    [cache[0]], [torch.zeros(9, device=dev)]):
        with pytest.raises(KernelError):
            F.CachePages(tensors)
    for args in ((t.long(), l, r, p, c), (t, l.long(), r, p, c), (t, l[:-1], r, p, c),
                 (t, l, r[:-1], p, c), (t, l, r, p.long(), c), (t, l, r, p, i32(free[:2], dev)),
                 (t[0], l, r, p, c), (t, l, r, p, c[None]), (table, l, r, p, c)):
        with pytest.raises(KernelError):
            F.fork_pages(handle, *args)
    with pytest.raises(KernelError):
        F.fork_pages(handle, t, l, r, p, c, out=(t, l))
    with pytest.raises(KernelError):
        F.fork_pages(handle, t, l, r, p, c, out=(t, l, r.long()))
    for args in ((t, l, r, p.long()), (t, l, r[None], p), (t, l, r, used)):
        with pytest.raises((KernelError, AttributeError)):
            F.free_pages(*args)
    with pytest.raises(KernelError):
        F.compact_pages(handle, t, r[:-1])
    with pytest.raises(KernelError):
        F.copy_pages(handle, p, i32([1, 2], dev))
