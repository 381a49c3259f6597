"""The weight that prefill chunks give to every key, against the 64-bit statement."""
import pytest
import torch

from orinfer_b200.ref import eviction_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(cuda):
    return cuda


def packet(dev, spans, qh, kvh, d, *, seed=0, score=1.0, gap=0, extra=1):
    """Chunks of (rows, position of the first), each of a request of its own, with ``gap`` rows of nobody
    behind each; what no row sees holds numbers that are none."""
    g = torch.Generator().manual_seed(seed * 7919 + qh * 31 + d)
    lens = [n + p for n, p in spans]
    counts = [-(-n // 128) for n in lens]
    pages = sum(counts) + 1
    order, at = torch.randperm(pages - 1, generator=g) + 1, 0
    slots = torch.randperm(len(spans), generator=g).tolist()
    table = torch.zeros(len(spans), max(counts) + extra, dtype=torch.int32)
    kc = torch.randint(-127, 128, (pages, 128, kvh, d), generator=g, dtype=torch.int8)
    ks = (torch.rand(pages, 128, kvh, d // 64, generator=g) * 0.019 + 1e-3).half()
    ks[0] = float("nan")
    chunks, row = [], 0
    for (n, p), slot, k in zip(spans, slots, counts):
        table[slot, :k] = order[at:at + k].int()
        at += k
        if (n + p) % 128:
            ks[table[slot, k - 1], (n + p) % 128:] = float("nan")
        chunks.append([row, n, p, slot])
        row += n + gap
    q = (torch.randn(max(row, 1), qh, d, generator=g) * score).half()
    for first, n, _, _ in chunks:
        q[first + n:first + n + gap] = float("nan")
    return (q.to(dev), torch.tensor(chunks, dtype=torch.int32, device=dev), max(n for n, _ in spans),
            table.to(dev), kc.to(dev), ks.to(dev))


def near(got, base, args, chunks=None):
    """A score is off by what its FP32 sums of 64 products at a time can be (64 steps of 2^-23 of its
    terms' magnitudes and eight roundings), a weight by that of its score and of the row's sum, and the
    roundings of both exponentials, of the sum (a chain of four and of the key steps of a row) and of the
    logarithm, whose result is as large as a score; a sum of weights by its parts' chains (sixteen
    weights, four parts to a unit, the units of a tile)."""
    q, all_chunks, _, table, kc, ks = args
    chunks = all_chunks.tolist() if chunks is None else chunks
    rows, req, pos = (t.to(q.device) for t in R.chunk_rows(chunks))
    added, reach = R.key_weights(q[rows], req, pos, table, kc, ks)
    steps = max([(p + n) // 64 for _, n, p, _ in chunks] + [1])
    tiles = sum(-(-n * q.shape[1] // kc.shape[2] // 100) for _, n, _, _ in chunks)
    rel = (2 * (64 * 2 + 8) * reach + 8 + 8 + steps + 4 * (reach + 20) + 24 + tiles) * 2.0 ** -24
    want = base.double()
    want[..., :added.shape[-1]] += added
    limit = 2.0 ** -23 * want * len(chunks)
    limit[..., :added.shape[-1]] += added * rel
    off = (got.double() - want).abs()
    assert bool((off <= limit).all()), f"{float((off / limit.clamp(min=1e-30)).max())} of the limit"


def sums(dev, args, seed=3):
    g = torch.Generator().manual_seed(seed)
    table, kvh = args[3], args[4].shape[2]
    return torch.rand(table.shape[0], kvh, table.shape[1] * 128, generator=g).to(dev)


def check(dev, args, **kw):
    from orinfer_b200.ops import functional as F
    base = sums(dev, args)
    weights = base.clone()
    F.prefill_weights(*args, weights, **kw)
    near(weights, base, args)
    return base, weights


GEOMETRIES = [(4, 2, 64), (16, 8, 64), (4, 4, 64), (16, 1, 64), (32, 8, 128), (40, 8, 128), (2, 2, 128),
              (8, 1, 128), (16, 2, 256), (3, 3, 256), (6, 2, 256), (16, 1, 256), (9, 3, 128)]


@pytest.mark.parametrize("qh,kvh,d", GEOMETRIES)
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 127, 128, 129, 300])
def test_one_chunk(dev, qh, kvh, d, n):
    check(dev, packet(dev, [(n, 0)], qh, kvh, d))


@pytest.mark.parametrize("qh,kvh,d", GEOMETRIES)
@pytest.mark.parametrize("before", [1, 63, 64, 127, 128, 500])
def test_behind_others(dev, qh, kvh, d, before):
    check(dev, packet(dev, [(70, before)], qh, kvh, d, seed=before))


@pytest.mark.parametrize("qh,kvh,d", GEOMETRIES)
def test_ragged_chunks(dev, qh, kvh, d):
    """Rows between the chunks are nobody's and hold no numbers."""
    spans = [(1, 0), (129, 0), (200, 300), (1, 1000), (64, 64), (33, 7), (2, 255)]
    check(dev, packet(dev, spans, qh, kvh, d, gap=3))


@pytest.mark.parametrize("qh,kvh,d", [(4, 2, 64), (32, 8, 128), (40, 8, 128), (16, 2, 256)])
@pytest.mark.parametrize("spans", [[(1100, 0)], [(64, 6000)], [(700, 900), (5, 3000)]])
def test_tiles_of_many_ctas(dev, qh, kvh, d, spans):
    check(dev, packet(dev, spans, qh, kvh, d))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("score", [0.0, 8.0, 40.0])
def test_equal_and_leaping_scores(dev, d, score):
    check(dev, packet(dev, [(200, 100), (90, 1000)], 8, 2, d, score=score))


def test_many_chunks(dev):
    check(dev, packet(dev, [(1 + i % 5, i % 140) for i in range(300)], 2, 2, 64))


def test_chunks_of_one_request_add_up(dev):
    """In their order, the same bits every time."""
    from orinfer_b200.ops import functional as F
    q, _, longest, table, kc, ks = packet(dev, [(400, 300), (100, 0)], 8, 2, 128)
    slot = int(packet(dev, [(400, 300), (100, 0)], 8, 2, 128)[1][0, 3])
    chunks = torch.tensor([[0, 150, 300, slot], [400, 100, 0, 1 - slot], [150, 250, 450, slot],
                           [0, 400, 300, slot]], dtype=torch.int32, device=dev)
    args = (q, chunks, longest, table, kc, ks)
    base, weights = check(dev, args)
    for _ in range(3):
        again = base.clone()
        F.prefill_weights(*args, again)
        assert torch.equal(again, weights)


def test_the_last_rows_of_a_prompt(dev):
    args = list(packet(dev, [(500, 0)], 8, 2, 128))
    args[1] = torch.tensor([[468, 32, 468, 0]], dtype=torch.int32, device=dev)
    args[2] = 32
    check(dev, args)


def test_a_row_at_a_time_and_a_prompt_at_once(dev):
    """Chunked or not, a prompt's rows give what single rows give."""
    from orinfer_b200.ops import functional as F
    q, chunks, n, table, kc, ks = packet(dev, [(150, 0)], 8, 2, 128)
    whole = torch.zeros(1, 2, table.shape[1] * 128, device=dev)
    F.prefill_weights(q, chunks, n, table, kc, ks, whole)
    rows = torch.zeros_like(whole)
    v, vs = torch.zeros_like(kc), torch.ones_like(ks)
    i32 = lambda *a: torch.arange(*a, dtype=torch.int32, device=dev)
    F.attention_weighed(q, None, i32(150) * 0, i32(150), table, kc, v, ks, vs, rows)
    args = (q, chunks, n, table, kc, ks)
    near(whole, torch.zeros_like(whole), args)
    near(rows, torch.zeros_like(whole), args)


def test_strided_sums_and_a_buffer_of_their_own(dev):
    from orinfer_b200.ops import functional as F
    args = packet(dev, [(200, 30), (10, 700)], 4, 2, 128)
    whole = torch.rand(5, 3, 4, args[3].shape[1] * 128 + 3, device=dev)
    view = whole[1:3, 0, 1:3]
    before, keep = view.clone(), whole.clone()
    other = torch.full_like(before, -1.0)
    F.prefill_weights(*args, view, weights_out=other)
    assert torch.equal(whole, keep)
    for _, n, p, slot in args[1].tolist():
        assert bool((other[slot, :, n + p:] == -1.0).all())
        near_other = other[slot, :, :n + p].clone()
        assert bool((near_other >= 0).all())
    F.prefill_weights(*args, view)
    near(view, before, args)
    for _, n, p, slot in args[1].tolist():
        assert torch.equal(view[slot, :, :n + p], other[slot, :, :n + p])
    keep[1:3, 0, 1:3] = view
    assert torch.equal(whole, keep)


def test_bounds_given_by_the_host(dev):
    """The longest context is known, rows behind the packet are in the buffer."""
    args = list(packet(dev, [(200, 30), (10, 700)], 4, 2, 128, extra=30))
    q = torch.full((300, 4, 128), float("nan"), dtype=torch.float16, device=dev)
    q[:210] = args[0]
    args[0] = q
    check(dev, args, max_kv_len=710, total_rows=210)


@pytest.mark.parametrize("wrong", [[0, 201, 0, 0], [151, 60, 0, 0], [-1, 5, 0, 0], [0, 5, -1, 0], [0, 5, 0, 2],
                                   [0, 5, 0, -1], [0, 5, 252, 0], [0, -3, 0, 0]])
def test_chunks_that_cannot_be_are_left_out(dev, wrong):
    from orinfer_b200.ops import functional as F, native
    q, chunks, n, table, kc, ks = packet(dev, [(200, 30), (10, 100)], 4, 2, 64, extra=0)
    chunks = torch.cat([chunks[1:], torch.tensor([wrong], dtype=torch.int32, device=dev)])
    base = torch.rand(2, 2, 256, device=dev)
    weights = base.clone()
    F.prefill_weights(q, chunks, 200, table, kc, ks, weights)
    assert native.read_status() >> 16 == 6
    native.clear_status()
    near(weights, base, (q, chunks, n, table, kc, ks), chunks.tolist()[:1])


def test_pages_that_are_none_are_reported(dev):
    from orinfer_b200.ops import functional as F, native
    q, chunks, n, table, kc, ks = packet(dev, [(200, 30)], 4, 2, 64)
    for bad in (kc.shape[0], -1):
        broken = table.clone()
        broken[0, 0] = bad
        F.prefill_weights(q, chunks, n, broken, kc, ks, torch.zeros(1, 2, table.shape[1] * 128, device=dev))
        assert native.read_status() >> 16 == 6
        native.clear_status()


def test_nothing_to_weigh(dev):
    from orinfer_b200.ops import functional as F
    q, chunks, n, table, kc, ks = packet(dev, [(20, 3)], 4, 2, 64)
    weights = torch.rand(1, 2, table.shape[1] * 128, device=dev)
    before = weights.clone()
    F.prefill_weights(q, chunks[:0], n, table, kc, ks, weights)
    F.prefill_weights(q[:0], chunks * 0, 0, table, kc, ks, weights)
    F.prefill_weights(q, chunks * 0, n, table, kc, ks, weights)
    assert torch.equal(weights, before)


def test_captured_and_on_another_stream(dev):
    from orinfer_b200.ops import functional as F
    args = packet(dev, [(200, 30), (10, 700)], 8, 2, 128)
    base, want = check(dev, args)
    weights = base.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        F.prefill_weights(*args, weights)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(weights, want)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            F.prefill_weights(*args, weights)
        graphs.append(g)
    for g in graphs:
        weights.copy_(base)
        g.replay()
        assert torch.equal(weights, want)
