"""Calls of a bounded cache's operators that must not reach a kernel: seen on the host."""
import ctypes

import pytest
import torch

from orinfer_b200.ops import native
from test_eviction_refusals import device_0, evict, prefill, weighed  # noqa: F401
from test_samples_devices import On, nothing_runs  # noqa: F401


@pytest.mark.parametrize("which", ["kcache", "vcache"])
@pytest.mark.parametrize("by", [1, 4, 8])
def test_attention_weighed_refuses_a_cache_off_16_bytes(nothing_runs, which, by):  # noqa: F811
    """Its kernels copy keys and values 16 bytes at a time."""
    raw = torch.zeros(5 * 128 * 2 * 64 + 32, dtype=torch.int8)
    raw = raw[-raw.data_ptr() % 16:]
    with pytest.raises(native.KernelError, match="16-byte"):
        weighed(changed={which: raw[by:by + 5 * 128 * 2 * 64].view(5, 128, 2, 64)})


@pytest.mark.parametrize("kc,vc", [(1, 0), (0, 8), (4, 4)])
def test_the_entries_refuse_a_cache_off_16_bytes(kc, vc):
    """Both entries answer before they look at a GPU."""
    place = 1 << 20                                  # (nothing is read there)
    at = ctypes.c_void_p(place)
    cache = [ctypes.c_void_p(place + kc), ctypes.c_void_p(place + vc)]
    lib = native.lib()
    assert lib.orinfer_attention(at, None, at, at, at, 1, *cache, at, at, at, 1, 2, 1, 128, 1, None, 0,
                                 None) == -1
    assert lib.orinfer_attention_weighed(at, None, at, at, at, 1, 1, *cache, at, at, 1, at, at, 256, 128,
                                         at, 256, 128, 128, 1, 2, 1, 128, 1, 128, at, 0, None) == -1


def test_the_plain_runner_refuses_before_anything_changes():
    from orinfer_b200.config import PRESETS
    from orinfer_b200.models.runner import KVPool, Packet
    from orinfer_b200.models.torch_runner import TorchRunner
    from orinfer_b200.models.weights import random_model
    cfg = PRESETS["tiny-hybrid"]
    assert not cfg.is_full_attention(0)
    runner = TorchRunner(random_model(cfg, seed=1), KVPool.allocate(cfg, 3, "cpu"), max_rows=8)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)
    for kw in (dict(weights=torch.zeros(1, 2, cfg.kv_heads, 128)),
               dict(rope_pos=i32([7]), mrope=i32([[7]] * 3))):
        with pytest.raises(ValueError):
            runner.logits(Packet(i32([5]), i32([0]), i32([0]), i32([[1]]), 1, 1, **kw))
        assert not hasattr(runner, "_gdn_pool")
        assert all(bool((t == 0).all()) for t in (*runner.kv.k, *runner.kv.v))


@pytest.fixture
def on_the_host(monkeypatch):
    """What a call allocates on the way to the library."""
    monkeypatch.setattr(torch, "empty", lambda *shape, **kw: torch.zeros(1))


def lines(slots, heads, slot_stride, head_stride, offset=0, size=4096, base=None):
    """[slots, heads, 384] at these strides of a buffer."""
    base = torch.zeros(size) if base is None else base
    return base.as_strided((slots, heads, 384), (slot_stride, head_stride, 1), offset)


SHARED_PLACES = [(0, 384), (768, 0), (0, 0), (768, 383), (767, 384), (384, 384), (383, 768)]
OWN_PLACES = [(768, 384), (384, 768), (1000, 500), (390, 800), (1152, 768)]


@pytest.mark.parametrize("strides", SHARED_PLACES)
def test_sums_that_share_places_are_refused(nothing_runs, strides):  # noqa: F811
    for kw in (dict(changed=dict(weights=lines(2, 2, *strides))),
               dict(weights_out=On.gpu(0, lines(2, 2, *strides)))):
        with pytest.raises(native.KernelError, match="place"):
            weighed(**kw)
    with pytest.raises(native.KernelError, match="place"):
        prefill(weights=lines(2, 2, *strides))


@pytest.mark.parametrize("strides", OWN_PLACES)
def test_sums_in_places_of_their_own_are_served(nothing_runs, on_the_host, strides):  # noqa: F811
    """(What is not refused reaches the library.)"""
    with pytest.raises(AssertionError, match="library"):
        weighed(changed=dict(weights=lines(2, 2, *strides)))
    with pytest.raises(AssertionError, match="library"):        # weights that are only read may be expanded
        weighed(changed=dict(weights=torch.zeros(1, 1, 384).expand(2, 2, 384)),
                weights_out=On.gpu(0, lines(2, 2, *strides)))


def test_two_buffers_in_one(nothing_runs, on_the_host):  # noqa: F811
    """Slot by slot or head by head a buffer may hold both the weights and the sums; shifted by less than a
    line it may not."""
    base = torch.zeros(8192)
    for strides, apart in (((1536, 384), 768), ((1536, 768), 384), ((768, 384), 1536), ((768, 1536), 384)):
        one = lambda at: lines(2, 2, *strides, at, base=base)
        with pytest.raises(AssertionError, match="library"):
            weighed(changed=dict(weights=one(0)), weights_out=On.gpu(0, one(apart)))
        with pytest.raises(AssertionError, match="library"):
            weighed(changed=dict(weights=one(5)), weights_out=On.gpu(0, one(5)))
        for by in (1, 383, apart - 1, apart + (1 if apart < 1536 else -384)):
            for a, b in ((0, by), (by, 0)):
                with pytest.raises(native.KernelError, match="place"):
                    weighed(changed=dict(weights=one(a)), weights_out=On.gpu(0, one(b)))


def test_evicted_weights_overlap_nothing(nothing_runs, on_the_host):  # noqa: F811
    shape, n = (2, 4, 2, 384), 2 * 4 * 2 * 384
    base = torch.zeros(3 * n)
    at = lambda i: base[i:i + n].view(shape)
    same = [On.gpu(0, torch.zeros(*s, dtype=torch.int32)) for s in ((4, 3), (4,), (9,))]
    for a, b in ((0, 1), (1, 0), (0, n - 1), (n - 1, 0), (n, 384)):
        with pytest.raises(native.KernelError, match="apart"):
            evict(weights=at(a), weights_out=On.gpu(0, at(b)), out=same)
    for a, b in ((0, n), (n, 0), (7, 7)):
        with pytest.raises(AssertionError, match="library"):
            evict(weights=at(a), weights_out=On.gpu(0, at(b)), out=same)
