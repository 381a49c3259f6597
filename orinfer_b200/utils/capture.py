"""Recording of CUDA graphs."""

from __future__ import annotations

import contextlib
import gc

import torch


@contextlib.contextmanager
def recording(graph: "torch.cuda.CUDAGraph"):
    """``torch.cuda.graph`` with Python's cycle collector at rest.  A dead engine is held by cycles
    until a collection finds it, and one that destroys the engine's graphs in the midst of a capture
    ends that capture with an error."""
    collects = gc.isenabled()
    gc.disable()
    try:
        with torch.cuda.graph(graph):
            yield
    finally:
        if collects:
            gc.enable()
