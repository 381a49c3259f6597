"""Attention of rows that share a prefix, at the edges of its tiles, pages and splits, against the
64-bit statement."""
import pytest
import torch

from orinfer_b200.ref import samples_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(cuda):
    return cuda


def _unaligned(t):
    """A contiguous copy whose address is two bytes past a 16-byte boundary."""
    flat = torch.empty(t.numel() + 8, dtype=t.dtype, device=t.device)
    out = flat[1:1 + t.numel()].view(t.shape)
    out.copy_(t)
    return out


def batch(dev, groups, qh, kvh, d, *, seed=0, loners=(), scales=(1e-3, 0.02), gated=False,
          score=1.0, fill=True):
    """A batch of ``groups``, (shared keys, keys of each row) with the shared ones on common pages,
    then rows of no group (``loners``).  Returns (plan's groups, arguments)."""
    g = torch.Generator().manual_seed(seed * 7919 + qh * 31 + d)
    spec, rows, pages = [], [], 1
    width = max([k for _, lens in groups for k in lens] + list(loners) + [1]) // 128 + 2
    for shared, lens in groups:
        spec.append((len(rows), len(lens), shared))
        common = list(range(pages, pages + shared // 128))
        pages += len(common)
        for n in lens:
            mine = max(0, (n + 127) // 128 - len(common))
            if shared % 128 and n > 0:
                mine = max(mine, 1)
            rows.append((n, common + list(range(pages, pages + mine))))
            pages += mine
        if shared % 128:            # the shared keys end inside a page: it is everybody's
            at = shared // 128
            for _, t in rows[spec[-1][0]:]:
                if len(t) > at:
                    t[at] = rows[spec[-1][0]][1][at]
    for n in loners:
        rows.append((n, list(range(pages, pages + (n + 127) // 128))))
        pages += (n + 127) // 128
    order = torch.randperm(pages - 1, generator=g) + 1
    table = torch.zeros(len(rows), width, dtype=torch.int32)
    for r, (_, t) in enumerate(rows):
        table[r, :len(t)] = order[torch.tensor(t, dtype=torch.long) - 1].int() if t else 0
    shape = (pages, 128, kvh)
    code = lambda: torch.randint(-127, 128, (*shape, d), generator=g, dtype=torch.int8).to(dev)
    scale = lambda: (torch.rand(*shape, d // 64, generator=g) * (scales[1] - scales[0])
                     + scales[0]).half()
    kc, vc, ks, vs = code(), code(), scale(), scale()
    if fill:                         # slots that nobody has written hold anything
        reach = torch.zeros(pages, dtype=torch.long)
        for r, (n, t) in enumerate(rows):
            for j in range((n + 127) // 128):
                p = int(table[r, j])
                reach[p] = max(int(reach[p]), min(128, n - 128 * j))
        dead = torch.arange(128)[None, :] >= reach[:, None]
        ks[dead], vs[dead] = float("nan"), float("inf")
    q = (torch.randn(len(rows), qh, d, generator=g) * score).half().to(dev)
    gate = torch.randn(len(rows), qh, d, generator=g).half().to(dev) if gated else None
    perm = torch.randperm(len(rows), generator=g)                  # requests in any order
    req = torch.empty(len(rows), dtype=torch.int32)
    req[:] = perm.int()
    shuffled = torch.empty_like(table)
    shuffled[perm] = table
    pos = torch.tensor([n - 1 for n, _ in rows], dtype=torch.int32)
    return spec, (q, gate, req.to(dev), pos.to(dev), shuffled.to(dev), kc, vc, ks.to(dev),
                  vs.to(dev))


def limit(ref, size, reach):
    """FP16 keys, values and weights at most, each rounded by 2^-11 at most, in sums of FP32: a
    score moves by 2^-11 of its terms' magnitudes, so a weight and the weights' sum by as much, a
    weight by its own rounding, a value by its own; then the result is rounded.  FP32's own part is
    a few 2^-22 of every term, and FP16 ends at 2^-25."""
    u = 2.0 ** -11
    return u * ref.abs() + size * (2.02 * u * reach + 2.02 * u + 2.0 ** -16) + 2.0 ** -24


def check(dev, spec, args, max_kv_len=None, plan=None, out=None):
    from orinfer_b200.ops import functional as F
    q, pos = args[0], args[3]
    if plan is None:
        plan = F.SharedPrefix(spec, q.shape[0], qh=q.shape[1], kvh=args[5].shape[2],
                              head_dim=q.shape[2],
                              max_kv_len=max_kv_len or int(pos.max()) + 1, device=dev,
                              force=True)
    out = F.attention_shared(*args, plan, out=out)
    ref, size, reach = R.attention_rows(*args)
    off = (out.double().view_as(ref) - ref).abs()
    assert bool(out.isfinite().all())
    assert bool((off <= limit(ref, size, reach)).all()), float((off / limit(ref, size, reach)).max())
    return out, ref


HEADS = [(2, 2, 64), (4, 2, 64), (16, 2, 64), (3, 3, 128), (4, 2, 128), (8, 2, 128), (10, 2, 128),
         (8, 1, 128), (2, 1, 256), (8, 1, 256), (8, 2, 256)]


@pytest.mark.parametrize("qh,kvh,d", HEADS)
@pytest.mark.parametrize("aligned", [True, False])
def test_groups_at_block_and_page_edges(dev, qh, kvh, d, aligned):
    """Few and many rows, prefixes of no, one and several pages, own keys from none on, a row that
    sees nothing, rows outside the groups."""
    groups = [(128, [129, 128, 200]), (256, [257] * 2), (0, [1, 40]),
              (640, [640 + n for n in (0, 1, 15, 16, 17, 31, 32, 33, 64, 127, 128, 129, 300)])]
    spec, args = batch(dev, groups, qh, kvh, d, loners=(5, 130, 0), gated=d == 256)
    if not aligned:
        args = (_unaligned(args[0]), None if args[1] is None else _unaligned(args[1]), *args[2:7],
                _unaligned(args[7]), _unaligned(args[8]))
    out, _ = check(dev, spec, args)
    assert bool((out[-1] == 0).all())


@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 130])
@pytest.mark.parametrize("qh,kvh,d", [(8, 2, 128), (2, 2, 64), (8, 1, 256), (10, 2, 128)])
def test_rows_at_tile_edges(dev, rows, qh, kvh, d):
    spec, args = batch(dev, [(384, [384 + 1 + 3 * r % 70 for r in range(rows)])], qh, kvh, d,
                       seed=rows)
    check(dev, spec, args)


@pytest.mark.parametrize("shared", [1, 2, 63, 64, 65, 127, 129, 191, 193, 1000])
@pytest.mark.parametrize("qh,kvh,d", [(8, 2, 128), (4, 2, 64), (8, 1, 256)])
def test_prefixes_that_end_inside_a_page(dev, shared, qh, kvh, d):
    """All keys of the rows are shared, and a row may see fewer of them than its group has."""
    lens = [shared, shared, max(1, shared - 1), max(1, shared // 2), 1, 0]
    spec, args = batch(dev, [(shared, lens)], qh, kvh, d, seed=shared)
    check(dev, spec, args)


def test_verification_rows_of_one_request(dev):
    """Rows at consecutive positions of one request: each sees one key more than the one before."""
    spec, args = batch(dev, [(896, [896 + i for i in range(1, 9)])], 8, 2, 128, seed=4)
    q, gate, req, pos, table, *cache = args
    longest = table[req[7].long()]
    table = table.clone()
    table[:] = longest
    for c in cache[2:]:
        c.nan_to_num_(nan=0.01, posinf=0.01)
    check(dev, spec, (q, gate, req, pos, table, *cache))


@pytest.mark.parametrize("qh,kvh,d", [(32, 8, 128), (40, 8, 128), (32, 4, 128), (16, 2, 256),
                                      (16, 8, 64)])
@pytest.mark.parametrize("rows,groups,shared", [(3, 1, 5120), (70, 3, 1280), (128, 1, 640),
                                                (24, 8, 256)])
def test_serving_geometries(dev, qh, kvh, d, rows, groups, shared):
    per = rows // groups
    spec, args = batch(dev, [(shared - 128 * (g % 2), [shared - 128 * (g % 2) + 1 + (37 * r) % 333
                                                       for r in range(per)])
                             for g in range(groups)],
                       qh, kvh, d, seed=rows + d, scales=(0.015, 0.045), gated=d == 256)
    out, ref = check(dev, spec, args)
    # on average: scores, weights, values and results each rounded once, 2^-11 / sqrt(3) at most
    assert float((out.double() - ref).norm() / ref.norm()) < 2 * 2.0 ** -11 / 3 ** 0.5 * 1.1


@pytest.mark.parametrize("qh,kvh,d", [(64, 8, 128), (32, 8, 256)])
def test_more_pages_to_a_cta_than_a_warp_has_lanes(dev, qh, kvh, d):
    from orinfer_b200.ops import functional as F
    rows = 128 // (qh // kvh) * (148 // (kvh * max(1, d // 128))) + 1
    spec, args = batch(dev, [(128 * 136 + 40, [128 * 136 + 41 + r % 60 for r in range(rows)])], qh, kvh,
                       d, seed=d)
    plan = F.SharedPrefix(spec, rows, qh=qh, kvh=kvh, head_dim=d, max_kv_len=128 * 138, device=dev,
                          force=True)
    keys = (plan.items[:, 3] - plan.items[:, 2]) * (32 if d > 128 else 64)
    assert int(keys.max()) > 32 * 128
    check(dev, spec, args, plan=plan)


def test_scores_that_leap_and_scales_over_many_binades(dev):
    spec, args = batch(dev, [(1024, [1024 + n for n in range(1, 40, 3)]), (512, [700, 701])], 8, 2,
                       128, seed=9, score=6.0, fill=False)
    vs = args[8]
    vs.copy_(torch.exp2(torch.rand(vs.shape, generator=torch.Generator().manual_seed(1)) * 18 - 14)
             .half())
    check(dev, spec, args)


def test_equal_scores_and_a_single_loud_key(dev):
    """Keys of zero give every value the same weight; one key that outweighs all others by far gives
    its value alone, wherever it stands."""
    spec, args = batch(dev, [(512, [600, 513, 640])], 8, 2, 128, seed=2, fill=False)
    q, _, req, pos, table, kc, vc, ks, vs = args
    kc.zero_()
    check(dev, spec, args)
    for key in (0, 100, 127, 128, 511, 512):
        kc.zero_()
        page = table[req[0].long(), key // 128].long()
        kc[page, key % 128] = 127
        q[:] = q.abs() + 1
        out, _ = check(dev, spec, args)


def test_a_long_cache_with_offsets_past_32_bits(dev):
    """A pool of more than 2^31 bytes per tensor, its last pages in use."""
    from orinfer_b200.ops import functional as F
    kvh, d, pages = 8, 128, (2 ** 31 + 2 ** 29) // (128 * 8 * 128)
    kc = torch.zeros(pages, 128, kvh, d, dtype=torch.int8, device=dev)
    vc = torch.zeros_like(kc)
    ks = torch.full((pages, 128, kvh, 2), 0.02, dtype=torch.float16, device=dev)
    table = torch.zeros(3, 4, dtype=torch.int32)
    table[:, :2] = torch.tensor([pages - 1, pages - 2])
    table[:, 2] = torch.tensor([pages - 3, pages - 4, pages - 5])
    g = torch.Generator().manual_seed(5)
    for c in (kc, vc):
        c[-5:] = torch.randint(-127, 128, (5, 128, kvh, d), generator=g, dtype=torch.int8).to(dev)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    q = torch.randn(3, 32, d, generator=g).half().to(dev)
    args = (q, None, i32([0, 1, 2]), i32([299, 256, 383]), table.to(dev), kc, vc, ks, ks)
    check(dev, [(0, 3, 256)], args)
    plan = F.SharedPrefix([], 3, qh=32, kvh=kvh, head_dim=d, max_kv_len=512, device=dev,
                          force=True)
    check(dev, [], args, plan=plan)


def test_one_plan_serves_the_steps_of_a_loop(dev):
    """The plan's bound is above the contexts of its first steps, and the results are those of a
    plan that knows them; the same call twice gives the same bits."""
    from orinfer_b200.ops import functional as F
    spec, args = batch(dev, [(384, [400, 450, 520])], 8, 2, 128, seed=11)
    plan = F.SharedPrefix(spec, 3, qh=8, kvh=2, head_dim=128, max_kv_len=4096, device=dev,
                          force=True)
    first, _ = check(dev, spec, args, plan=plan)
    first = first.clone()
    out = torch.empty_like(first)
    again, _ = check(dev, spec, args, plan=plan, out=out)
    assert again is out and torch.equal(first, again)


@pytest.mark.parametrize("rows,shared,items", [(2, 384, False), (8, 1024, False), (128, 1024, True),
                                               (40, 5120, True)])
def test_what_is_cheaper_read_again_is_not_shared(dev, rows, shared, items):
    from orinfer_b200.ops import functional as F
    spec, args = batch(dev, [(shared, [shared + 1 + 7 * r % 90 for r in range(rows)])], 32, 8, 128,
                       seed=rows)
    plan = F.SharedPrefix(spec, rows, qh=32, kvh=8, head_dim=128, max_kv_len=shared + 90, device=dev)
    assert (plan.items is not None) == items
    check(dev, spec, args, plan=plan)


def test_own_keys_in_parts(dev):
    """Own keys that are long enough to be split, behind a prefix and without one, gated and not."""
    for qh, kvh, d in ((8, 2, 128), (4, 2, 64), (8, 1, 256)):
        spec, args = batch(dev, [(256, [2500, 300, 256])], qh, kvh, d, loners=(1700, 40, 0), seed=d,
                           gated=d == 256)
        from orinfer_b200.ops import functional as F
        plan = F.SharedPrefix(spec, 6, qh=qh, kvh=kvh, head_dim=d, max_kv_len=2600, device=dev,
                              force=True)
        assert plan.splits > 1
        check(dev, spec, args, plan=plan)


def test_on_another_stream_and_in_a_graph(dev):
    from orinfer_b200.ops import functional as F
    spec, args = batch(dev, [(640, [700, 641, 900, 780]), (256, [300, 257])], 32, 8, 128, seed=13)
    plan = F.SharedPrefix(spec, 6, qh=32, kvh=8, head_dim=128, max_kv_len=900, device=dev, force=True)
    want = F.attention_shared(*args, plan).clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = F.attention_shared(*args, plan)
    side.synchronize()
    assert torch.equal(got, want)
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        F.attention_shared(*args, plan, out=out)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)


@pytest.mark.parametrize("rows,shared,qh,kvh,d", [(24, 1024, 8, 2, 128), (70, 512, 4, 2, 64),
                                                  (9, 640, 16, 2, 256)])
def test_steps_that_follow_each_other_without_a_wait(dev, rows, shared, qh, kvh, d):
    """A decode loop writes the queries of each step over those of the last and its keys behind
    theirs.  In one graph the row kernels run beside the prefix's kernel, and the next step's beside
    them; with a wait after every call they cannot.  The results have the same bits."""
    from orinfer_b200.ops import functional as F
    steps, g = 24, torch.Generator().manual_seed(rows)
    width = (shared + 128) // 128
    spec, args = batch(dev, [(shared, [shared + 1] * rows)], qh, kvh, d, seed=rows)
    _, _, row_req, _, table, kc, vc, ks, vs = args
    assert table.shape[1] >= width
    qkv = torch.randn(steps, rows, (qh + 2 * kvh) * d, generator=g).half().to(dev)
    pos = (torch.arange(steps, dtype=torch.int32)[:, None] + shared
           + torch.zeros(rows, dtype=torch.int32)).to(dev)
    plan = F.SharedPrefix(spec, rows, qh=qh, kvh=kvh, head_dim=d, max_kv_len=shared + steps,
                          device=dev, force=True)
    q = torch.empty(rows, qh, d, dtype=torch.float16, device=dev)
    cos, sin = (torch.empty(rows, d // 2, dtype=torch.float32, device=dev) for _ in range(2))
    caches = [t.clone() for t in (kc, vc, ks, vs)]

    def loop(out, wait):
        for t, first in zip((kc, vc, ks, vs), caches):
            t.copy_(first)
        for s in range(steps):
            F.rope_table(pos[s], d, 1e6, cos, sin, rows=rows)
            F.qk_rope_kv(qkv[s], None, None, cos, sin, row_req, pos[s], table, kc, vc, ks, vs, qh=qh,
                         kvh=kvh, head_dim=d, gated=False, eps=1e-6, zero_centered=False, q_out=q,
                         gate_out=None, rows=rows)
            wait()
            F.attention_shared(q, None, row_req, pos[s], table, kc, vc, ks, vs, plan, out=out[s])
            wait()

    want, got = (torch.empty(steps, rows, qh * d, dtype=torch.float16, device=dev) for _ in range(2))
    loop(want, torch.cuda.synchronize)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loop(got, lambda: None)
    for _ in range(3):
        got.zero_()
        graph.replay()
        assert torch.equal(got, want)
    assert float(want.float().abs().max()) > 0 and not torch.equal(want[0], want[1])


def test_refusals(dev):
    from orinfer_b200.ops import functional as F
    from orinfer_b200.ops.native import KernelError
    mk = lambda groups, rows=6, **kw: F.SharedPrefix(
        groups, rows, **{**dict(qh=8, kvh=2, head_dim=128, max_kv_len=1024, device=dev), **kw})
    for groups in ([(0, 7, 128)], [(-1, 2, 128)], [(0, 2, -1)], [(0, 2, 2048)],
                   [(0, 3, 128), (2, 2, 128)]):
        with pytest.raises(KernelError):
            mk(groups)
    for kw in (dict(head_dim=96), dict(qh=6), dict(qh=7), dict(qh=10, head_dim=64),
               dict(rows=-1), dict(max_kv_len=-1), dict(kvh=0)):
        with pytest.raises(KernelError):
            mk([], **kw)
    spec, args = batch(dev, [(256, [300, 280])], 8, 2, 128)
    plan = F.SharedPrefix(spec, 2, qh=8, kvh=2, head_dim=128, max_kv_len=300, device=dev)
    F.attention_shared(*args, plan)
    bad = {0: [args[0].float(), args[0][:1], args[0].transpose(0, 1).contiguous().transpose(0, 1),
               args[0].cpu()],
           1: [args[0].float(), args[0][:1]], 2: [args[2].long(), args[2][:1]],
           3: [args[3].long()], 4: [args[4].long(), args[4][0], args[4].t()],
           5: [args[5].short(), args[5][:, :64], args[5][..., :64]],
           6: [args[6][:-1]], 7: [args[7].float(), args[7][..., :1]], 8: [args[8][:-1]]}
    for at, values in bad.items():
        for v in values:
            with pytest.raises(KernelError):
                F.attention_shared(*args[:at], v, *args[at + 1:], plan)
    with pytest.raises(KernelError):
        F.attention_shared(*args, mk(spec, 3))
    with pytest.raises(KernelError):
        F.attention_shared(*args, plan, out=torch.empty(2, 8, 128, device=dev))


def test_no_rows(dev):
    from orinfer_b200.ops import functional as F
    spec, args = batch(dev, [(128, [130])], 8, 2, 128)
    plan = F.SharedPrefix([], 0, qh=8, kvh=2, head_dim=128, max_kv_len=10, device=dev)
    out = F.attention_shared(args[0][:0], None, args[2][:0], args[3][:0], *args[4:], plan)
    assert out.shape == (0, 1024)
