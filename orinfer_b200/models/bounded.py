"""Requests of any length whose cache has a bound, on one GPU.

Every row that is computed adds the attention weight that it gives to the keys it sees, layer by
layer and KV head by KV head.  A request that reaches the bound is cut down to ``keep`` tokens: in
each layer and head the first and the latest keys stay, and of the others those that got the most
weight.  What stays keeps the rotary angle that it was written with, so rows take their rotary
position from the text (``Packet.rope_pos``) and their place in the cache from what is left.
"""

from __future__ import annotations

from typing import Callable, Dict, List, Optional, Sequence

import torch

from ..config import PAGE_TOKENS
from ..core import sampling as S
from ..ops import functional as F
from .runner import ModelRunner, Packet
from .slots import SlotPages


class BoundedRequests(SlotPages):
    """Up to ``slots`` requests in the cache of ``runner``, which nothing else uses meanwhile.  A
    request holds at most ``bound`` tokens and is cut down to ``keep`` of them, the ``first`` and the
    last ``recent`` among them, when the next would not fit.  ``last_rows``: how many rows at the end
    of each piece of a prompt count for the weights (default: all)."""

    def __init__(self, runner: ModelRunner, slots: int, bound: int, keep: int, *, first: int = 4,
                 recent: int = 64, last_rows: Optional[int] = None):
        if not (0 < keep < bound and first >= 0 and recent >= 0 and first + recent <= keep):
            raise ValueError(f"{bound} tokens cut down to {keep} with {first} first and {recent} last")
        if last_rows is not None and last_rows < 1:
            raise ValueError("last_rows: at least one")
        super().__init__(runner, slots, bound)
        cfg = runner.cfg
        layers = sum(cfg.is_full_attention(i) for i in range(cfg.layers))
        self.cache = runner.kv.key_cache(layers)
        self.bound, self.keep, self.first, self.recent = bound, keep, first, recent
        self.last_rows = last_rows
        self.weights = torch.zeros(layers, slots, cfg.kv_heads, self.table.shape[1] * PAGE_TOKENS,
                                   device=self.device)
        self.text: Dict[int, List[int]] = {}            # slot -> its tokens
        self.logits: Dict[int, torch.Tensor] = {}       # slot -> logits behind them
        self._len: Dict[int, int] = {}                  # slot -> tokens in the cache

    # ---------------------------------------------------------------- cache
    def cut(self, slots: Sequence[int]) -> None:
        """Cuts those of the slots down that have more than ``keep`` tokens."""
        self._known(slots)
        slots = [s for s in slots if self._len[s] > self.keep]
        # all at once, or one after the other where free pages are too few for that
        if not self._cut(slots) and not all(self._cut([s]) for s in slots):
            raise MemoryError("not enough free pages for the kept keys")

    def _cut(self, slots: List[int]) -> bool:
        if not slots:
            return True
        *_, status = F.evict_keys(self.cache, self.table, self.lens, self.refs, self.weights,
                                  self._i32(slots), self.keep, first=self.first,
                                  recent=self.recent, out=(self.table, self.lens, self.refs))
        if int(status) == 2:
            raise RuntimeError("the page table and the lengths do not agree")
        if int(status) == 0:
            self._len.update(dict.fromkeys(slots, self.keep))
        return int(status) == 0

    def _grow(self, slots: Sequence[int], tokens: int):
        """Pages for ``tokens`` more tokens of each slot; returns what was taken, or None."""
        at = [(s, c) for s in slots for c in range(-(-self._len[s] // PAGE_TOKENS),
                                                   -(-(self._len[s] + tokens) // PAGE_TOKENS))]
        return self._take([s for s, _ in at], [c for _, c in at]) if at else None

    def _wrote(self, slots: Sequence[int], tokens: int) -> None:
        self.lens[torch.tensor(list(slots), device=self.device)] += tokens
        for s in slots:
            self._len[s] += tokens

    # ---------------------------------------------------------------- requests
    def add(self, prompt: Sequence[int]) -> int:
        """Prefills a prompt of any length; returns its slot."""
        prompt = [int(t) for t in prompt]
        if not prompt:
            raise ValueError("a prompt has tokens")
        if not self._free:
            raise MemoryError("no free slot")
        slot = self._free.pop()
        self._len[slot] = 0
        try:
            at = 0
            while at < len(prompt):
                if self._len[slot] == self.bound:
                    self.cut([slot])
                n = min(len(prompt) - at, self.runner.ws.max_rows, self.bound - self._len[slot])
                self.logits[slot] = self._prefill(slot, prompt, at, n)
                at += n
        except BaseException:
            self._give_up(slot)
            raise
        self.text[slot] = prompt
        return slot

    def _prefill(self, slot: int, prompt: List[int], at: int, n: int) -> torch.Tensor:
        i32, before = self._i32, self._len[slot]
        self._grow([slot], n)
        count = min(n, self.last_rows or n)
        p = Packet(i32(prompt[at:at + n]), i32([slot] * n), i32(list(range(before, before + n))),
                   self.table, n, before + n, torch.tensor([n - 1], device=self.device),
                   chunks=i32([[0, n, before, slot]]), max_q_len=n, max_chunk_kv=before + n,
                   weights=self.weights, rope_pos=i32(list(range(at, at + n))),
                   weigh_chunks=i32([[n - count, count, before + n - count, slot]]))
        logits = self.runner.logits(p)[0]
        self._wrote([slot], n)
        return logits

    def step(self, tokens: Dict[int, int]) -> torch.Tensor:
        """Appends a token to each of the given slots; returns their logits, in that order.  Where the
        forward raises, the requests are as they were before it, though cut down if they were at the
        bound, and the step may be taken again; those of a model with recurrent layers, whose states have
        moved on, are given up."""
        slots = list(tokens)
        self._known(slots)
        if not 0 < len(slots) <= self.runner.ws.max_rows:
            raise ValueError(f"{len(slots)} requests, at most {self.runner.ws.max_rows} at once")
        self.cut([s for s in slots if self._len[s] == self.bound])
        at = [self._len[s] for s in slots]
        p = Packet(self._i32([int(tokens[s]) for s in slots]), self._i32(slots), self._i32(at),
                   self.table, len(slots), max(at) + 1, weights=self.weights,
                   rope_pos=self._i32([len(self.text[s]) for s in slots]))
        rows = torch.tensor(slots, device=self.device)
        before = self.weights[:, rows, :, :max(at) + 1]      # (a copy)
        taken = self._grow(slots, 1)
        try:
            logits = self.runner.logits(p)
            self._wrote(slots, 1)
        except BaseException:
            self.weights[:, rows, :, :max(at) + 1] = before
            if taken is not None:
                self._put_back(taken)
            if self.runner.cfg.arch == "hybrid":
                for s in slots:
                    self.drop(s)
            raise
        for r, s in enumerate(slots):
            self.text[s].append(int(tokens[s]))
            self.logits[s] = logits[r]
        return logits

    def generate(self, slots: Sequence[int], options: Sequence[S.SamplingOptions], max_new: int, *,
                 stop: Optional[Callable[[Sequence[int]], bool]] = None) -> List[List[int]]:
        """Up to ``max_new`` tokens of each slot, drawn by the host law; a request ends early where
        ``stop(tokens)`` says so, and may go on with another call."""
        if len(slots) != len(options) or len(set(slots)) != len(slots):
            raise ValueError("options for each slot, a slot once")
        self._known(slots)
        for o in options:
            o.validate()
        got: Dict[int, List[int]] = {s: [] for s in slots}
        live = list(zip(slots, options))
        for _ in range(max_new):
            if not live:
                break
            drawn = {s: int(S.sample(self.logits[s].cpu().numpy(), self.text[s], o,
                                     S.counter_uniform(o.seed, 0, len(self.text[s]))))
                     for s, o in live}
            self.step(drawn)
            for s, token in drawn.items():
                got[s].append(token)
            live = [(s, o) for s, o in live if stop is None or not stop(got[s])]
        return [got[s] for s in slots]

    def drop(self, slot: int) -> None:
        """Gives up a request."""
        self._known([slot])
        del self.text[slot]
        self._give_up(slot)

    def _known(self, slots: Sequence[int]) -> None:
        for s in slots:
            if s not in self._len:
                raise ValueError(f"slot {s} holds no request")

    def _give_up(self, slot: int) -> None:
        self.logits.pop(slot, None)
        del self._len[slot]
        self.weights[:, slot].zero_()
        self._release([slot])
