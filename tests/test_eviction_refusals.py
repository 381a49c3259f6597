"""The operators of a cache with a bound refuse what they cannot serve before anything is launched;
their host statement on small cases."""
import math

import pytest
import torch

from orinfer_b200.ops import functional as F, native
from orinfer_b200.ref import eviction_ref as R
from test_samples_devices import On, nothing_runs  # noqa: F401


@pytest.fixture(autouse=True)
def device_0(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)


def weighed(index=0, changed=None, **kw):
    """A call of ``attention_weighed`` on tensors that say they lie on a GPU."""
    rows, qh, kvh, d, pages = 3, 4, 2, 64, 5
    ints = lambda *s: torch.zeros(*s, dtype=torch.int32)
    half = lambda *s: torch.zeros(*s, dtype=torch.float16)
    given = dict(q=half(rows, qh, d), gate=None, row_req=ints(rows), row_pos=ints(rows),
                 page_table=ints(2, 3), kcache=torch.zeros(pages, 128, kvh, d, dtype=torch.int8),
                 vcache=torch.zeros(pages, 128, kvh, d, dtype=torch.int8),
                 kscale=half(pages, 128, kvh, 1), vscale=half(pages, 128, kvh, 1),
                 weights=torch.zeros(2, kvh, 384))
    given = {k: v if v is None else On.gpu(index, v) for k, v in given.items()}
    for k, v in (changed or {}).items():
        given[k] = v if v is None or isinstance(v, On) or not isinstance(v, torch.Tensor) else On.gpu(index, v)
    return F.attention_weighed(*given.values(), **kw)


@pytest.mark.parametrize("changed", [
    dict(q=torch.zeros(3, 4, 64)), dict(q=torch.zeros(3, 4, 128, dtype=torch.float16)),
    dict(q=torch.zeros(3, 5, 64, dtype=torch.float16)),
    dict(q=torch.zeros(3, 64, 4, dtype=torch.float16).transpose(1, 2)),
    dict(row_req=torch.zeros(2, dtype=torch.int32)), dict(row_pos=torch.zeros(3, dtype=torch.int64)),
    dict(page_table=torch.zeros(2, 3)), dict(page_table=torch.zeros(3, 3, dtype=torch.int32)),
    dict(kscale=torch.zeros(5, 128, 2, 2, dtype=torch.float16)),
    dict(kcache=torch.zeros(5, 64, 2, 64, dtype=torch.int8)),
    dict(vcache=torch.zeros(4, 128, 2, 64, dtype=torch.int8)),
    dict(weights=torch.zeros(2, 3, 384)), dict(weights=torch.zeros(2, 2, 384, dtype=torch.float64)),
    dict(weights=torch.zeros(2, 384, 2).transpose(1, 2)), dict(weights=torch.zeros(1, 2, 384)),
    dict(gate=torch.zeros(3, 4, 32, dtype=torch.float16)),
])
def test_attention_weighed_refuses(nothing_runs, changed):  # noqa: F811
    with pytest.raises(native.KernelError):
        weighed(changed=changed)


@pytest.mark.parametrize("kw", [dict(splits=0), dict(splits=33), dict(rows=4), dict(rows=-1),
                                dict(weights_out=On.gpu(0, torch.zeros(2, 2, 383))),
                                dict(weights_out=On.gpu(1, torch.zeros(2, 2, 384))),
                                dict(out=On.gpu(0, torch.zeros(3, 256)))])
def test_attention_weighed_refuses_options(nothing_runs, kw):  # noqa: F811
    with pytest.raises(native.KernelError):
        weighed(**kw)


def test_another_device_than_the_current_one(nothing_runs):  # noqa: F811
    with pytest.raises(native.KernelError, match="current"):
        weighed(index=1)
    with pytest.raises(native.KernelError, match="current"):
        evict(index=1)


def key_cache(index=0):
    cache = object.__new__(F.KeyCache)
    cache.device, cache.layers, cache.pages = torch.device("cuda", index), 2, 9
    cache.kvh, cache.head_dim = 2, 64
    cache.bases = On.gpu(index, torch.zeros(8, dtype=torch.int64))
    return cache


def evict(index=0, keep=100, **changed):
    ints = lambda *s: torch.zeros(*s, dtype=torch.int32)
    given = dict(table=ints(4, 3), lens=ints(4), refs=ints(9), weights=torch.zeros(2, 4, 2, 384),
                 slots=ints(2))
    given.update({k: changed.pop(k) for k in list(changed) if k in given})
    given = {k: v if isinstance(v, On) else On.gpu(index, v) for k, v in given.items()}
    return F.evict_keys(key_cache(index), *given.values(), keep, **changed)


@pytest.mark.parametrize("changed", [
    dict(keep=0), dict(keep=385), dict(first=60, recent=41), dict(first=-1), dict(recent=-1),
    dict(weights=torch.zeros(2, 4, 2, 383)), dict(weights=torch.zeros(1, 4, 2, 384)),
    dict(weights=torch.zeros(2, 4, 2, 768)[..., ::2]), dict(weights=torch.zeros(2, 4, 384)),
    dict(weights=torch.zeros(2, 4, 2, 384).half()), dict(refs=torch.zeros(8, dtype=torch.int32)),
    dict(lens=torch.zeros(3, dtype=torch.int32)), dict(slots=torch.zeros(2, dtype=torch.int64)),
    dict(slots=On.gpu(1, torch.zeros(2, dtype=torch.int32))),
    dict(weights=On.gpu(1, torch.zeros(2, 4, 2, 384))),
    dict(weights_out=On.gpu(0, torch.zeros(2, 4, 2, 385))), dict(out=()),
])
def test_evict_keys_refuses(nothing_runs, changed):  # noqa: F811
    with pytest.raises(native.KernelError):
        evict(**changed)


def test_key_cache_refuses():
    one = lambda **kw: {**dict(k=torch.zeros(3, 128, 2, 64, dtype=torch.int8),
                               v=torch.zeros(3, 128, 2, 64, dtype=torch.int8),
                               ks=torch.zeros(3, 128, 2, 1, dtype=torch.float16),
                               vs=torch.zeros(3, 128, 2, 1, dtype=torch.float16)), **kw}
    with pytest.raises(native.KernelError):
        F.KeyCache([], [], [], [])
    with pytest.raises(native.KernelError, match="CPU"):
        F.KeyCache(*([t] for t in one().values()))


def test_kept_keys():
    w = torch.tensor([0.1, 5.0, math.nan, 0.2, 5.0, -math.inf, 0.3, 0.0])
    assert R.kept_keys(w, 8, 3, 0, 0) == [1, 4, 6]
    assert R.kept_keys(w, 8, 3, 1, 1) == [0, 1, 7]
    assert R.kept_keys(w, 8, 7, 0, 0) == [0, 1, 3, 4, 5, 6, 7]
    assert R.kept_keys(w, 3, 3, 0, 0) == [0, 1, 2]


def test_weights_of_a_row_add_up_to_its_heads():
    g = torch.Generator().manual_seed(0)
    k = torch.randint(-99, 99, (4, 128, 2, 64), generator=g, dtype=torch.int8)
    s = torch.rand(4, 128, 2, 1, generator=g).half() * 0.01
    q = torch.randn(3, 6, 64, generator=g).half()
    table = torch.tensor([[1, 2], [3, 0]], dtype=torch.int32)
    got, _ = R.key_weights(q, torch.tensor([0, 1, 0]), torch.tensor([200, 5, -1]), table, k, s)
    assert torch.allclose(got.sum(2), torch.full((2, 2), 3.0, dtype=torch.float64))
    assert bool((got[0, :, 201:] == 0).all()) and bool((got[1, :, 6:] == 0).all())


def prefill(index=0, longest=3, **changed):
    ints = lambda *s: torch.zeros(*s, dtype=torch.int32)
    given = dict(q=torch.zeros(3, 4, 64, dtype=torch.float16), chunks=ints(1, 4), table=ints(2, 3),
                 k=torch.zeros(5, 128, 2, 64, dtype=torch.int8),
                 ks=torch.zeros(5, 128, 2, 1, dtype=torch.float16), weights=torch.zeros(2, 2, 384))
    given.update({k: changed.pop(k) for k in list(changed) if k in given})
    given = {k: v if isinstance(v, On) else On.gpu(index, v) for k, v in given.items()}
    q, chunks, table, k, ks, weights = given.values()
    return F.prefill_weights(q, chunks, longest, table, k, ks, weights, **changed)


@pytest.mark.parametrize("changed", [
    dict(q=torch.zeros(3, 4, 64)), dict(q=torch.zeros(3, 4, 128, dtype=torch.float16)),
    dict(q=torch.zeros(3, 5, 64, dtype=torch.float16)),
    dict(q=torch.zeros(3, 34, 64, dtype=torch.float16)),         # 17 query heads to a KV head
    dict(q=torch.zeros(3 * 256 + 1, dtype=torch.float16)[1:].view(3, 4, 64)),
    dict(chunks=torch.zeros(1, 4)), dict(chunks=torch.zeros(1, 3, dtype=torch.int32)),
    dict(chunks=torch.zeros(4, 2, dtype=torch.int32).t()),
    dict(chunks=torch.zeros(513, 4, dtype=torch.int32)),
    dict(chunks=On.gpu(1, torch.zeros(1, 4, dtype=torch.int32))),
    dict(table=torch.zeros(3, 3, dtype=torch.int32)), dict(k=torch.zeros(4, 128, 2, 64, dtype=torch.int8)),
    dict(k=torch.zeros(5 * 128 * 128 + 1, dtype=torch.int8)[1:].view(5, 128, 2, 64)),
    dict(ks=torch.zeros(5, 128, 2, 2, dtype=torch.float16)), dict(weights=torch.zeros(2, 1, 384)),
    dict(weights=torch.zeros(2, 2, 384).double()), dict(weights=On.gpu(1, torch.zeros(2, 2, 384))),
    dict(weights_out=On.gpu(0, torch.zeros(2, 2, 383))), dict(total_rows=4), dict(total_rows=-1),
    dict(longest=-1),
])
def test_prefill_weights_refuses(nothing_runs, changed):  # noqa: F811
    with pytest.raises(native.KernelError):
        prefill(**changed)


@pytest.mark.parametrize("changed", [dict(longest=0), dict(total_rows=0), dict(max_kv_len=0),
                                     dict(chunks=torch.zeros(0, 4, dtype=torch.int32))])
def test_prefill_weights_of_nothing_launches_nothing(nothing_runs, changed):  # noqa: F811
    assert prefill(**changed) is None


def test_prefill_weights_on_another_device_than_the_current_one(nothing_runs):  # noqa: F811
    with pytest.raises(native.KernelError, match="current"):
        prefill(index=1)


def test_the_plain_runner_turns_keys_where_it_is_told_and_counts_nothing():
    from orinfer_b200.config import PRESETS
    from orinfer_b200.models.runner import KVPool, Packet
    from orinfer_b200.models.torch_runner import TorchRunner
    from orinfer_b200.models.weights import random_model
    cfg = PRESETS["tiny"]
    runner = TorchRunner(random_model(cfg, seed=1), KVPool.allocate(cfg, 3, "cpu"), max_rows=8)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)
    ids, table, keys = i32([5, 9, 11]), i32([[1], [2]]), []
    for slot, pos, rope in ((0, [7, 8, 9], None), (1, [2, 3, 4], i32([7, 8, 9]))):
        runner.logits(Packet(ids, i32([slot] * 3), i32(pos), table, 3, 10, rope_pos=rope))
        keys.append(runner.kv.k[0][slot + 1, pos])
    assert torch.equal(*keys)
    with pytest.raises(ValueError):
        runner.logits(Packet(ids, i32([0] * 3), i32([0, 1, 2]), table, 3, 3,
                             weights=torch.zeros(cfg.layers, 2, cfg.kv_heads, 128)))
