"""Several samples of a prompt on one GPU.

A prompt is prefilled once and keeps its pages.  Every batch of samples forks it: whole pages of the
prompt are shared, the page that is not full is copied.  The samples decode together: the shared
pages are read once for all of them (``Packet.shared``), penalties, biases and masks are applied to
the logits on the device, and the device sampler draws.  A sample that ends gives its pages back, and
``compact`` moves what is held to the front of the cache, so that its tail can be given up.
"""

from __future__ import annotations

from typing import Callable, Dict, List, Optional, Sequence

import numpy as np
import torch

from ..config import PAGE_TOKENS
from ..core import sampling as S
from ..ops import functional as F
from .runner import ModelRunner, Packet
from .slots import SlotPages


class PromptSamples(SlotPages):
    """Prompts and their samples in the cache of ``runner``, which nothing else uses meanwhile.
    ``slots`` bounds the prompts held and the samples decoded at once, ``max_tokens`` the length of
    each."""

    def __init__(self, runner: ModelRunner, slots: int, max_tokens: int):
        super().__init__(runner, slots, max_tokens)
        self.cache = runner.kv.cache_pages()
        self._prompts: Dict[int, tuple] = {}            # slot -> (tokens, last logits, recurrent state)

    def compact(self) -> int:
        """Moves the pages that are held to the front; returns how many there are."""
        F.compact_pages(self.cache, self.table, self.refs, out=(self.table, self.refs))
        return self.held

    # ---------------------------------------------------------------- prompts
    def add(self, prompt: Sequence[int]) -> int:
        """Prefills a prompt and keeps it; returns its slot."""
        prompt = [int(t) for t in prompt]
        if not 0 < len(prompt) <= self.max_tokens:
            raise ValueError(f"a prompt of {len(prompt)} tokens, of 1 to {self.max_tokens}")
        if not self._free:
            raise MemoryError("no free slot")
        columns = range(-(-len(prompt) // PAGE_TOKENS))
        self._take([self._free[-1]] * len(columns), columns)
        slot = self._free.pop()
        self.lens[slot] = len(prompt)
        try:
            logits = self._prefill(slot, prompt)
        except BaseException:
            self._release([slot])
            raise
        state = None
        if self.runner.cfg.arch == "hybrid":
            state = self.runner.gdn_snapshot(slot)
        self._prompts[slot] = (prompt, logits, state)
        return slot

    def _prefill(self, slot: int, prompt: List[int]) -> torch.Tensor:
        """Logits behind the prompt, whose keys and values go to the slot's pages."""
        i32, most = self._i32, self.runner.ws.max_rows
        for at in range(0, len(prompt), most):
            ids = prompt[at:at + most]
            n, end = len(ids), at + len(ids)
            p = Packet(i32(ids), i32([slot] * n), i32(list(range(at, end))), self.table, n, end,
                       torch.tensor([n - 1], device=self.device),
                       chunks=i32([[0, n, at, slot]]), max_q_len=n, max_chunk_kv=end)
            if end == len(prompt):
                return self.runner.logits(p)[0]
            self.runner.forward_hidden(p)

    def drop(self, slot: int) -> None:
        """Gives up a prompt."""
        del self._prompts[slot]
        self._release([slot])

    # ---------------------------------------------------------------- samples
    def sample(self, prompts: Sequence[int], options: Sequence[Sequence[S.SamplingOptions]],
               max_new: int, *, mask: Optional[np.ndarray] = None,
               stop: Optional[Callable[[Sequence[int]], bool]] = None, force: bool = False,
               on_step=None) -> List[List[List[int]]]:
        """``options[i]`` has the options of every sample of prompt (slot) ``prompts[i]``; returns
        the tokens of each.  ``mask``: the words of a token mask (bit set = permitted) that binds
        all samples.  A sample ends at ``max_new`` tokens or where ``stop(tokens)`` says so.
        ``force`` shares prefixes that are cheaper read again.  ``on_step(rows, logits, tokens)``
        sees each step's sample numbers, raw logits and tokens."""
        for slot in prompts:
            if slot not in self._prompts:
                raise ValueError(f"slot {slot} holds no prompt")
            if len(self._prompts[slot][0]) + max_new - 1 > self.max_tokens:
                raise ValueError(f"{max_new} tokens do not fit behind the prompt of slot {slot}")
        of = [i for i, o in enumerate(options) for _ in o]
        if len(of) > min(len(self._free), self.runner.ws.max_rows):
            raise MemoryError(f"{len(of)} samples, {len(self._free)} free slots")
        flat = [o for group in options for o in group]
        for o in flat:
            o.validate()
        got: List[List[int]] = [[] for _ in flat]
        if flat and max_new > 0:
            run = _Run(self, [prompts[i] for i in of], flat, max_new, mask, force)
            try:
                run.decode(got, stop, on_step)
            finally:
                run.end(run.live)
        out: List[List[List[int]]] = [[] for _ in prompts]
        for i, tokens in zip(of, got):
            out[i].append(tokens)
        return out


class _Run:
    """The samples that are decoded together.  Row r of a step is sample ``live[r]``; the tensors of
    a step have its rows and shrink as samples end."""

    def __init__(self, pool: PromptSamples, parents: List[int], options, max_new, mask, force):
        dev, i32 = pool.device, pool._i32
        self.pool, self.runner, self.parents, self.options = pool, pool.runner, parents, options
        self.max_new, self.force, self.mask = max_new, force, mask
        n = len(parents)
        self.live: List[int] = []
        self.slots = [pool._free[-1 - i] for i in range(n)]
        texts = [pool._prompts[p][0] for p in parents]
        self.prompt_len = [len(t) for t in texts]
        history = torch.zeros(n, max(self.prompt_len) + max_new, dtype=torch.int32)
        for r, t in enumerate(texts):
            history[r, :len(t)] = torch.tensor(t, dtype=torch.int32)
        f64 = lambda v: torch.tensor(v, dtype=torch.float64, device=dev)
        self.rows = dict(
            slot=i32(self.slots), history=history.to(dev), history_len=i32(self.prompt_len),
            repetition=f64([o.repetition_penalty for o in options]),
            presence=f64([o.presence_penalty for o in options]),
            frequency=f64([o.frequency_penalty for o in options]),
            top_k=i32([min(max(o.top_k, 1), 64) for o in options]),
            temperature=f64([max(o.temperature, 1e-5) for o in options]),
            top_p=f64([o.top_p for o in options]))
        self.uniforms = [[S.counter_uniform(o.seed, 0, t) for o in options] for t in range(max_new)]
        # what the device sampler draws; the host law serves the others, and the flagged rows
        self.on_device = [o.temperature >= 1e-5 and 1 <= o.top_k <= 64 for o in options]
        self.mask_words = None
        if mask is not None:
            words = np.ascontiguousarray(mask, dtype=np.uint32).view(np.int32)
            self.mask_words = torch.from_numpy(words.copy()).to(dev).view(1, -1)
        *_, status = F.fork_pages(pool.cache, pool.table, pool.lens, pool.refs, i32(parents),
                                  i32(self.slots), out=(pool.table, pool.lens, pool.refs))
        if int(status) != 0:
            raise MemoryError("not enough free pages for the samples")
        del pool._free[-n:]
        self.live = list(range(n))
        for s, parent in zip(self.slots, parents):
            if pool._prompts[parent][2] is not None:
                self.runner.gdn_restore(s, pool._prompts[parent][2], pool.slots)

    def end(self, samples: Sequence[int]) -> None:
        if samples:
            self.pool._release([self.slots[i] for i in samples])

    def _rows_changed(self) -> None:
        """Plan, biases and masks of the rows that are left."""
        cfg, pool, live = self.runner.cfg, self.pool, self.live
        groups, first = [], 0
        for r in range(1, len(live) + 1):
            if r == len(live) or self.parents[live[r]] != self.parents[live[first]]:
                whole = self.prompt_len[live[first]] // PAGE_TOKENS * PAGE_TOKENS
                if r - first > 1 and whole:
                    groups.append((first, r - first, whole))
                first = r
        self.plan = None
        if groups:
            self.plan = F.SharedPrefix(groups, len(live), qh=cfg.q_heads, kvh=cfg.kv_heads,
                                       head_dim=cfg.head_dim, device=pool.device, force=self.force,
                                       max_kv_len=[self.prompt_len[i] + self.max_new for i in live])
        biases = [sorted(self.options[i].logit_bias.items()) for i in live]
        self.extra = {}
        if any(biases):
            starts = np.cumsum([0] + [len(b) for b in biases]).tolist()
            self.extra.update(bias_start=pool._i32(starts),
                              bias_ids=pool._i32([t for b in biases for t, _ in b]),
                              bias_values=torch.tensor([v for b in biases for _, v in b],
                                                       dtype=torch.float64, device=pool.device))
        if self.mask_words is not None:
            self.extra.update(mask=self.mask_words, mask_rows=pool._i32([0] * len(live)))

    def _draw(self, logits, step: int, got) -> torch.Tensor:
        t, live = self.rows, self.live
        scores, refused = F.process_logits(logits, history=t["history"], history_len=t["history_len"],
                                     repetition=t["repetition"], presence=t["presence"],
                                     frequency=t["frequency"], **self.extra)
        uniform = torch.tensor([self.uniforms[step][i] for i in live], dtype=torch.float64,
                               device=logits.device)
        token, flag = F.sample_topk(scores, t["top_k"], t["temperature"], t["top_p"], uniform)
        flags = (flag | refused).tolist()
        for r, i in enumerate(live):
            if flags[r] or not self.on_device[i]:
                history = self.pool._prompts[self.parents[i]][0] + got[i]
                token[r] = S.sample(logits[r].cpu().numpy(), history, self.options[i],
                                    self.uniforms[step][i], self.mask)
        return token

    def decode(self, got: List[List[int]], stop, on_step) -> None:
        pool, t = self.pool, self.rows
        logits = torch.stack([pool._prompts[p][1] for p in self.parents])
        self._rows_changed()
        for step in range(self.max_new):
            token = self._draw(logits, step, got)
            for i, tok in zip(self.live, token.tolist()):
                got[i].append(tok)
            if on_step is not None:
                on_step(list(self.live), logits, token)
            over = [step + 1 == self.max_new or (stop is not None and stop(got[i]))
                    for i in self.live]
            t["history"].scatter_(1, t["history_len"].long()[:, None], token[:, None])
            t["history_len"] += 1
            if any(over):
                ended = [i for i, o in zip(self.live, over) if o]
                self.live = [i for i, o in zip(self.live, over) if not o]
                self.end(ended)
                if not self.live:
                    return
                keep = torch.tensor([r for r, o in enumerate(over) if not o], device=pool.device)
                for k in t:
                    t[k] = t[k].index_select(0, keep)
                token = token.index_select(0, keep)
                self._rows_changed()
            at = {i: self.prompt_len[i] + step for i in self.live}
            new = [i for i in self.live if at[i] % PAGE_TOKENS == 0]
            if new:
                pool._take([self.slots[i] for i in new], [at[i] // PAGE_TOKENS for i in new])
            p = Packet(token, t["slot"], t["history_len"] - 1, pool.table, len(self.live),
                       max(at.values()) + 1, shared=self.plan)
            logits = self.runner.logits(p)
            pool.lens[t["slot"].long()] += 1
