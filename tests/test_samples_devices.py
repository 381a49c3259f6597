"""The operators for several samples refuse tensors of different GPUs before anything is launched."""
import pytest
import torch

from orinfer_b200.ops import functional as F, native


class On(torch.Tensor):
    """A CPU tensor that says it lies on a GPU."""

    @staticmethod
    def gpu(index, t):
        out = t.as_subclass(On)
        out.index_of_gpu = index
        return out

    @property
    def device(self):
        return torch.device("cuda", self.index_of_gpu)

    @property
    def is_cuda(self):
        return True


@pytest.fixture
def nothing_runs(monkeypatch):
    def lib():
        raise AssertionError("the library was called")
    monkeypatch.setattr(native, "lib", lib)


def cache_on(index):
    cache = object.__new__(F.CachePages)
    cache.pages, cache.device, cache._args = 9, torch.device("cuda", index), ()
    return cache


def i32(index, *shape):
    return On.gpu(index, torch.zeros(*shape, dtype=torch.int32))


@pytest.mark.parametrize("elsewhere", range(5))
def test_fork(nothing_runs, elsewhere):
    on = [int(i == elsewhere) for i in range(5)]
    with pytest.raises(native.KernelError, match="GPU"):
        F.fork_pages(cache_on(0), i32(on[0], 4, 3), i32(on[1], 4), i32(on[2], 9), i32(on[3], 1),
                     i32(on[4], 1))


def test_a_cache_on_another_gpu(nothing_runs):
    with pytest.raises(native.KernelError, match="GPU"):
        F.fork_pages(cache_on(1), i32(0, 4, 3), i32(0, 4), i32(0, 9), i32(0, 1), i32(0, 1))
    with pytest.raises(native.KernelError, match="GPU"):
        F.compact_pages(cache_on(1), i32(0, 4, 3), i32(0, 9))
    with pytest.raises(native.KernelError, match="GPU"):
        F.copy_pages(cache_on(1), i32(0, 2), i32(0, 2))
    with pytest.raises(native.KernelError, match="GPU"):
        F.copy_pages(cache_on(1), i32(1, 2), i32(1, 2), i32(0, 2))


def test_free(nothing_runs):
    with pytest.raises(native.KernelError, match="GPU"):
        F.free_pages(i32(0, 4, 3), i32(0, 4), i32(0, 9), i32(1, 2))


@pytest.mark.parametrize("name", ["history", "history_len", "repetition", "presence", "frequency",
                                  "bias_start", "bias_ids", "bias_values", "mask", "mask_rows", "out",
                                  "flags"])
def test_logits(nothing_runs, name):
    rows, vocab = 2, 40
    f64 = lambda n: torch.zeros(n, dtype=torch.float64)
    ints = lambda *s: torch.zeros(*s, dtype=torch.int32)
    given = dict(history=ints(rows, 5), history_len=ints(rows), repetition=f64(rows),
                 presence=f64(rows), frequency=f64(rows), bias_start=ints(rows + 1), bias_ids=ints(3),
                 bias_values=f64(3), mask=ints(rows, 2), mask_rows=ints(rows),
                 out=torch.zeros(rows, vocab), flags=ints(rows))
    given = {k: On.gpu(int(k == name), v) for k, v in given.items()}
    with pytest.raises(native.KernelError, match="GPU"):
        F.process_logits(On.gpu(0, torch.zeros(rows, vocab)), **given)
