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
