"""Calls of a bounded cache's operators that must not reach a kernel: seen on the host."""
import ctypes

import pytest
import torch

from orinfer_b200.ops import native
from test_eviction_refusals import device_0, weighed  # noqa: F401
from test_samples_devices import nothing_runs  # noqa: F401


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
