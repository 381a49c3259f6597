"""Requests whose text outgrows their cache, decoded together on one GPU: keys that got little
attention are given up (random weights: the tokens are noise, the operators are those of serving).

    PYTHONPATH=. python examples/bounded-cache.py [preset] [requests] [tokens of a request]
"""
import sys
import time

import torch

from orinfer_b200.config import PRESETS
from orinfer_b200.core.sampling import SamplingOptions
from orinfer_b200.models.bounded import BoundedRequests
from orinfer_b200.models.runner import KVPool, ModelRunner
from orinfer_b200.models.weights import random_model


def main(preset="tiny", requests=4, tokens=64):
    cfg = PRESETS[preset]
    device = torch.device("cuda")
    pages = 1 + 7 * requests
    runner = ModelRunner(random_model(cfg, device=device), KVPool.allocate(cfg, pages, device),
                         max_rows=512)
    pool = BoundedRequests(runner, slots=requests, bound=640, keep=384, first=4, recent=64)
    words = torch.Generator().manual_seed(0)
    slots = [pool.add(torch.randint(0, cfg.vocab, (500 + 300 * i,), generator=words).tolist())
             for i in range(requests)]
    torch.cuda.synchronize()
    start = time.perf_counter()
    drawn = pool.generate(slots, [SamplingOptions(temperature=0.8, top_k=40, seed=i)
                                  for i in range(requests)], tokens)
    seconds = time.perf_counter() - start
    for s, got, held in zip(slots, drawn, pool.lens.tolist()):
        print(f"request {s}: {len(pool.text[s])} tokens of text, {held} in the cache, {got[:8]}")
    print(f"{requests * tokens / seconds:.0f} tok/s, {pool.held} of {pages - 1} pages held")
    return drawn


if __name__ == "__main__":
    main(*sys.argv[1:2], *(int(a) for a in sys.argv[2:4]))
