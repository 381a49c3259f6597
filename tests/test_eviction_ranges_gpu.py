"""The operators of a bounded cache where a cache passes 32 bits, on two streams at once, and in turns on
the same keys."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture
def dev(cuda):
    return cuda


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def cache(g, pages, kvh, d, dev):
    k, v = (torch.randint(-127, 128, (pages, 128, kvh, d), generator=g, dtype=torch.int8) for _ in range(2))
    ks, vs = ((torch.rand(pages, 128, kvh, d // 64, generator=g) * 0.02).half() for _ in range(2))
    return [t.to(dev) for t in (k, v, ks, vs)]


def calls(F, parts, table, lens, refs, q, weights, slots):
    """A prompt's weights, a step's, a cut and a step behind it."""
    kvh, d = parts[0].shape[2:]
    dev, n = q.device, int(lens[0])
    F.prefill_weights(q, i32([[0, 40, n - 40, 0]], dev), 40, table, parts[0], parts[2], weights[0])
    outs = [F.attention_weighed(q[40:42], None, i32([0, 1], dev), i32([n - 1, 299], dev), table, *parts,
                                weights[0], splits=3, max_kv_len=n)]
    handle = F.KeyCache(*([t] for t in parts))
    *_, status = F.evict_keys(handle, table, lens, refs, weights, slots, 200, first=3, recent=20,
                              out=(table, lens, refs))
    outs.append(F.attention_weighed(q[42:44], None, i32([0, 1], dev), i32([199, 199], dev), table, *parts,
                                    weights[0], max_kv_len=384))
    return [*outs, status]


@pytest.mark.parametrize("kvh,d", [(8, 128), (2, 256)])
def test_pages_beyond_32_bits(dev, kvh, d):
    """The same requests on the first pages of a small cache and behind byte 2^32 of a large one."""
    from orinfer_b200.ops import functional as F
    g = torch.Generator().manual_seed(d)
    near = cache(g, 12, kvh, d, dev)
    base = (1 << 32) // (128 * kvh * d) + 1
    far = [torch.empty(base + 12, *t.shape[1:], dtype=t.dtype, device=dev) for t in near]
    for a, b in zip(near, far):
        b[base:] = a
    assert far[0].stride(0) * base > 1 << 32
    table = i32([[1, 2, 3], [4, 5, 6]], dev)
    refs = i32([0] + [1] * 6 + [0] * 5, dev)
    q = torch.randn(44, kvh * 4, d, generator=g).half().to(dev)
    got = []
    for parts, up in ((near, 0), (far, base)):
        t = torch.where(table > 0, table + up, table).int()
        held = torch.ones(up + 12, dtype=torch.int32, device=dev)
        held[up:] = refs
        held[up] = 1 if up else 0
        state = [t, i32([384, 300], dev), held, torch.zeros(1, 2, kvh, 384, device=dev)]
        outs = calls(F, parts, state[0], state[1], state[2], q, state[3], i32([0, 1], dev))
        assert int(outs[2]) == 0
        assert torch.equal(state[0], i32([[7 + up, 8 + up, 0], [9 + up, 10 + up, 0]], dev))
        got.append([*outs[:2], state[1], state[3], state[2][up + 1:], *(p[up + 7:up + 11] for p in parts)])
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_two_streams_at_once(dev):
    """Each stream has a cache of its own; calls share no workspace, so neither sees the other."""
    from orinfer_b200.ops import functional as F
    g = torch.Generator().manual_seed(5)
    kvh, d, n = 4, 128, 384
    sides = []
    for side in range(2):
        parts = cache(g, 12, kvh, d, dev)
        q = torch.randn(44, kvh * 4, d, generator=g).half().to(dev)
        sides.append((parts, q))

    def state():
        return (i32([[1, 2, 3], [4, 5, 6]], dev), i32([n, 300], dev), i32([0] + [1] * 6 + [0] * 5, dev),
                torch.zeros(1, 2, kvh, n, device=dev))

    want = []
    for parts, q in sides:
        mine, s = [p.clone() for p in parts], state()
        want.append([*calls(F, mine, *s[:3], q, s[3], i32([0, 1], dev)), *s, *mine])
    streams = [torch.cuda.Stream() for _ in sides]
    for _ in range(10):
        held = [([p.clone() for p in parts], state(), q) for parts, q in sides]
        slots = i32([0, 1], dev)
        torch.cuda.synchronize()
        got = []
        for stream, (mine, s, q) in zip(streams, held):
            with torch.cuda.stream(stream):
                got.append([*calls(F, mine, *s[:3], q, s[3], slots), *s, *mine])
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_graphs_that_take_turns(dev):
    """A step and a cut captured into a graph each, replayed in turns while the request grows back: every
    state is that of the same calls without graphs."""
    from orinfer_b200.ops import functional as F
    g = torch.Generator().manual_seed(6)
    kvh, d = 2, 64
    parts = cache(g, 9, kvh, d, dev)
    mine = [p.clone() for p in parts]
    q = torch.randn(1, 8, d, generator=g).half().to(dev)

    def make(parts):
        table, lens, refs = i32([[1, 2, 3]], dev), i32([384], dev), i32([0, 1, 1, 1, 0, 0, 0, 0, 0], dev)
        weights, slots, pos = torch.zeros(1, 1, kvh, 384, device=dev), i32([0], dev), i32([383], dev)
        handle = F.KeyCache(*([t] for t in parts))
        step = lambda: F.attention_weighed(q, None, slots, pos, table, *parts, weights[0], splits=2)
        cut = lambda: F.evict_keys(handle, table, lens, refs, weights, slots, 300, recent=8,
                                   out=(table, lens, refs))[3]
        return step, cut, (table, lens, refs, weights, pos)

    def turns(step, cut, state):
        table, lens, refs, weights, pos = state
        seen = []
        for turn in range(4):
            pos.fill_(383)
            seen.append(step().clone())
            seen += [cut().clone(), *(t.clone() for t in state)]
            pos.fill_(299)
            seen.append(step().clone())
            lens.fill_(384)                          # (it has grown back: the page has the room)
        return seen

    step, cut, state = make(parts)
    want = turns(step, cut, state)
    step, cut, state = make(mine)
    initial = [t.clone() for t in (*state, *mine)]
    step(), cut()                                    # (warm-up outside the graphs)
    for t, was in zip((*state, *mine), initial):
        t.copy_(was)
    graphs, outs = [], []
    for call in (step, cut):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call())
        graphs.append(graph)
    for t, was in zip((*state, *mine), initial):
        t.copy_(was)
    replay = lambda i: (graphs[i].replay(), outs[i])[1]
    got = turns(lambda: replay(0), lambda: replay(1), state)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    assert all(torch.equal(a, b) for a, b in zip(parts, mine))


@pytest.mark.parametrize("qh,kvh,d", [(8, 2, 64), (16, 4, 128), (8, 1, 256)])
def test_a_row_of_one_key_and_a_cut_to_one(dev, qh, kvh, d):
    """The shortest there is: the only key has the weight of all heads, and stays."""
    from orinfer_b200.ops import functional as F
    g = torch.Generator().manual_seed(7)
    parts = cache(g, 4, kvh, d, dev)
    q = torch.randn(3, qh, d, generator=g).half().to(dev)
    table, weights = i32([[1]], dev), torch.zeros(1, 1, kvh, 128, device=dev)
    F.prefill_weights(q, i32([[0, 1, 0, 0]], dev), 1, table, parts[0], parts[2], weights[0])
    F.attention_weighed(q[1:2], None, i32([0], dev), i32([0], dev), table, *parts, weights[0])
    # exp(score - lse) of a score that is the lse but for its roundings: four sums of at most 16 (eight
    # deviations) in each of two orders, 2 * 4 * 16 * 2^-24 = 2^-17
    assert float((weights[0, 0, :, 0] - 2 * qh // kvh).abs().max()) <= 2 * qh // kvh * 2.0 ** -17
    assert bool((weights[..., 1:] == 0).all())
    F.attention_weighed(q[2:3], None, i32([0], dev), i32([1], dev), table, *parts, weights[0])
    lens, refs = i32([2], dev), i32([0, 1, 0, 0], dev)
    handle = F.KeyCache(*([t] for t in parts))
    *_, status = F.evict_keys(handle, table, lens, refs, weights, i32([0], dev), 1,
                              out=(table, lens, refs))
    assert int(status) == 0 and table.tolist() == [[2]] and refs.tolist() == [0, 0, 1, 0]
    assert torch.equal(parts[0][2, 0], parts[0][1, 0]) and torch.equal(parts[3][2, 0], parts[3][1, 0])
    out = F.attention_weighed(q[2:3], None, i32([0], dev), i32([0], dev), table, *parts, weights[0])
    v = parts[1][2, 0].double().view(kvh, d // 64, 64) * parts[3][2, 0].double()[..., None]
    want = v.reshape(kvh, 1, d).expand(kvh, qh // kvh, d).reshape(qh * d)
    # a weight of one in 2^20, and the FP16 result's rounding of half a step (and the least number's)
    assert bool(((out[0].double() - want).abs() <= want.abs() * (2.0 ** -11 + 2.0 ** -19) + 2.0 ** -25).all())
