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
