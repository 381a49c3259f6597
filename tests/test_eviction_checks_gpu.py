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
