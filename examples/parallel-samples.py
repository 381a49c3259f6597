"""Several samples of each of two prompts, decoded together on one GPU (random weights: the tokens
are noise, the operators are those of serving).

    PYTHONPATH=. python examples/parallel-samples.py [preset] [samples of a prompt] [tokens of a sample]
"""
import sys
import time

import torch

from orinfer_b200.config import PRESETS
from orinfer_b200.core.sampling import SamplingOptions
from orinfer_b200.models.runner import KVPool, ModelRunner
from orinfer_b200.models.samples import PromptSamples
from orinfer_b200.models.weights import random_model


def main(preset="tiny", samples=8, tokens=32):
    cfg = PRESETS[preset]
    device = torch.device("cuda")
    runner = ModelRunner(random_model(cfg, device=device), KVPool.allocate(cfg, 256, device),
                         max_rows=512)
    pool = PromptSamples(runner, slots=2 * samples + 2, max_tokens=2048)
    text = torch.Generator().manual_seed(0)
    prompts = [pool.add(torch.randint(0, cfg.vocab, (n,), generator=text).tolist())
               for n in (1000, 700)]
    options = [[SamplingOptions(temperature=0.8, top_k=40, top_p=0.95, repetition_penalty=1.1,
                                presence_penalty=0.2, seed=100 * p + i) for i in range(samples)]
               for p in prompts]
    print(f"{pool.held} pages hold two prompts")
    torch.cuda.synchronize()
    start = time.perf_counter()
    drawn = pool.sample(prompts, options, tokens)
    seconds = time.perf_counter() - start
    for p, group in zip(prompts, drawn):
        for tokens_of in group:
            print(p, tokens_of[:12])
    print(f"{2 * samples} samples of {tokens} tokens: {2 * samples * tokens / seconds:.0f} tok/s")
    pool.drop(prompts[0])
    print(f"{pool.compact()} pages hold the second prompt, from the first page on")
    again = pool.sample(prompts[1:], options[1:], tokens)[0]
    print(f"{sum(len(s) for s in again)} more tokens of it")
    return drawn, again


if __name__ == "__main__":
    main(*sys.argv[1:2], *(int(a) for a in sys.argv[2:4]))
