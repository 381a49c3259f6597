"""Decode attention that weighs its keys, given rows that name what is not there: nothing outside the
caller's tensors is read or written, the other rows are served, and the status word says so."""
import pytest
import torch

from test_attention_weighed_gpu import batch, near, sums

pytestmark = pytest.mark.gpu
BAD_INDEX = 6


@pytest.fixture(scope="module")
def dev(cuda):
    return cuda


def status():
    from orinfer_b200.ops import native
    word = native.read_status()
    native.clear_status()
    return word >> 16, word & 0xffff


# geometry, splits: both forms of the row kernel, with heads of their own and with four to a CTA
FORMS = [(4, 2, 64, 1), (32, 8, 128, 1), (32, 8, 128, 3), (16, 2, 256, 2), (40, 8, 128, 1)]


@pytest.mark.parametrize("qh,kvh,d,splits", FORMS)
@pytest.mark.parametrize("long", [False, True])
def test_rows_of_requests_that_do_not_exist(dev, qh, kvh, d, splits, long):
    """Sums lie inside a larger buffer, whose other places stay as they were."""
    from orinfer_b200.ops import functional as F
    lens = [3000, 700, 1500, 90] if long else [61, 130, 5, 300]
    args = list(batch(dev, lens, qh, kvh, d, seed=4, gated=d == 256))
    whole = torch.rand(10, kvh, args[4].shape[1] * 128, device=dev)
    before, view = whole.clone(), whole[3:7]
    want = F.attention(*args, splits=splits)
    good = args[2].clone()
    args[2] = torch.tensor([0, 4, -1, 3], dtype=torch.int32, device=dev)     # of four requests
    out = F.attention_weighed(*args, view, splits=splits)
    assert status() == (BAD_INDEX, 0x61)
    assert torch.equal(out[[0, 3]], want[[0, 3]]) and bool((out[[1, 2]] == 0).all())
    assert torch.equal(whole[:3], before[:3]) and torch.equal(whole[7:], before[7:])
    assert torch.equal(view[1:3], before[4:6])
    args[2], args[3] = good, args[3].masked_fill(torch.tensor([0, 1, 1, 0], device=dev).bool(), -1)
    near(view, before[3:7], args)


def test_many_rows_of_requests_that_do_not_exist(dev):
    """More rows than a CTA looks at at once, four heads to a CTA; indices far away among them."""
    from orinfer_b200.ops import functional as F
    args = list(batch(dev, [1 + i % 60 for i in range(300)], 8, 8, 64, seed=5))
    gone = torch.arange(300, device=dev) % 7 == 3
    good, args[2] = args[2], args[2].masked_fill(gone, 2**31 - 1)
    args[2][3] = -2**31
    base = sums(dev, args)
    weights = base.clone()
    out = F.attention_weighed(*args, weights)
    assert status() == (BAD_INDEX, 0x61)
    args[2], args[3] = good, args[3].masked_fill(gone, -1)
    assert torch.equal(out, F.attention(*args))
    near(weights, base, args)


def test_padding_of_any_request_is_no_fault(dev):
    from orinfer_b200.ops import functional as F
    args = list(batch(dev, [200, 90, 77], 4, 2, 128))
    args[2] = torch.tensor([0, 99, -5], dtype=torch.int32, device=dev)
    args[3] = torch.tensor([199, -1, -1], dtype=torch.int32, device=dev)
    out = F.attention_weighed(*args, sums(dev, args), splits=2)
    assert status() == (0, 0) and bool((out[1:] == 0).all())


@pytest.mark.parametrize("qh,kvh,d,splits", FORMS + [(32, 8, 128, 32)])
@pytest.mark.parametrize("far", [3 * 128, 10**6, 2**31 - 2, 2**31 - 1])
def test_positions_behind_the_row_of_the_table(dev, qh, kvh, d, splits, far):
    """Such a row sees nothing, another row of its request what it did; the last one's keys would end
    behind the table."""
    from orinfer_b200.ops import functional as F
    args = list(batch(dev, [3 * 128, 100, 3 * 128], qh, kvh, d, per=2, seed=6))
    args[4] = args[4][:, :3].contiguous()
    want = F.attention(*args, splits=splits)
    base = sums(dev, args)
    weights, good = base.clone(), args[3]
    gone = torch.tensor([1, 0, 0, 0, 0, 1], device=dev).bool()
    args[3] = good.masked_fill(gone, far)
    out = F.attention_weighed(*args, weights, splits=splits)
    assert status() == (BAD_INDEX, 0x61)
    assert torch.equal(out[~gone], want[~gone]) and bool((out[gone] == 0).all())
    args[3] = good.masked_fill(gone, -1)
    near(weights, base, args, 2)


@pytest.mark.parametrize("qh,kvh,d,splits", FORMS)
@pytest.mark.parametrize("bad", [-1, 10**9, "first"])
def test_pages_that_the_cache_does_not_have(dev, qh, kvh, d, splits, bad):
    """Page 0 is read for them; here it has the keys of the page that the table should name."""
    from orinfer_b200.ops import functional as F
    args = list(batch(dev, [5000, 700, 90], qh, kvh, d, seed=7))
    for row, column in ((0, 20), (0, 39), (1, 5), (2, 0)):
        table = args[4]
        for cache in args[5:]:
            cache[0] = cache[int(table[row, column])]
        want = F.attention(*args, splits=splits)
        base = sums(dev, args)
        given, weights = list(args), base.clone()
        given[4] = table.clone()
        given[4][row, column] = args[5].shape[0] if bad == "first" else bad
        out = F.attention_weighed(*given, weights, splits=splits)
        assert status() == (BAD_INDEX, 0x62)
        assert torch.equal(out, want)
        near(weights, base, args)


@pytest.mark.parametrize("most", [1, 97, 98, 99, 100])
@pytest.mark.parametrize("over", [0, 1, 2])
def test_the_bound_of_keys_is_met_to_the_key(dev, most, over):
    """Keys behind ``max_kv_len`` get nothing and are reported, wherever it lies among four."""
    from orinfer_b200.ops import functional as F
    args = batch(dev, [most + over, 1], 4, 2, 64)
    base = sums(dev, args)
    weights = base.clone()
    F.attention_weighed(*args, weights, max_kv_len=most)
    assert status() == ((BAD_INDEX, 0x60) if over else (0, 0))
    want = base.clone()
    F.attention_weighed(*args, want)
    assert status() == (0, 0)
    assert torch.equal(weights[..., :most], want[..., :most])
    assert torch.equal(weights[..., most:], base[..., most:])


@pytest.mark.parametrize("order", [(0, 1, 2), (1, 0, 2)])
def test_weights_and_sums_in_turns_in_one_buffer(dev, order):
    """Two buffers line by line in one, and weights that are read from one line for all slots."""
    from orinfer_b200.ops import functional as F
    args = batch(dev, [200, 700, 90], 4, 2, 128)
    keys = args[4].shape[1] * 128
    shape = [3, 2, keys]
    inv = [order.index(i) for i in range(3)]
    base = torch.zeros(*[shape[i] for i in order[:2]], 2, keys, device=dev)
    one, two = (base[:, :, i].permute(*inv) for i in (0, 1))
    one.copy_(sums(dev, args))
    before = one.clone()
    want = before.clone()
    F.attention_weighed(*args, want, splits=2)
    F.attention_weighed(*args, one, splits=2, weights_out=two)
    seen = torch.arange(keys, device=dev)[None, :] <= args[3][:, None]
    seen = seen[:, None].expand(shape)
    assert torch.equal(one, before) and torch.equal(two[seen], want[seen])
    line = sums(dev, args)[:1, :1].expand(shape)
    want = line.clone()
    F.attention_weighed(*args, want, splits=2)
    F.attention_weighed(*args, line, splits=2, weights_out=two)
    assert torch.equal(two[seen], want[seen])
