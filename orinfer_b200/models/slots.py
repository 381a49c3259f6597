"""Slots of requests in a model's paged cache on one GPU, and the pages that they hold."""

from __future__ import annotations

from typing import Sequence

import torch

from ..config import PAGE_TOKENS
from ..ops import functional as F
from .runner import ModelRunner


class SlotPages:
    """``slots`` requests of up to ``max_tokens`` cached tokens each in the cache of ``runner``, which
    nothing else uses meanwhile: their page table, lengths and the references of the pages."""

    def __init__(self, runner: ModelRunner, slots: int, max_tokens: int):
        self.runner, self.device, self.slots = runner, runner.device, slots
        self.max_tokens = max_tokens
        width = -(-max_tokens // PAGE_TOKENS)
        zeros = lambda *s: torch.zeros(*s, dtype=torch.int32, device=self.device)
        self.table, self.lens, self.refs = zeros(slots, width), zeros(slots), zeros(runner.kv.pages)
        self._free = list(range(slots - 1, -1, -1))

    def _i32(self, v):
        return torch.tensor(v, dtype=torch.int32, device=self.device)

    def _take(self, slots: Sequence[int], columns: Sequence[int]):
        """Gives each slot a free page at a column of its row, the lowest pages first; returns what
        ``_put_back`` needs."""
        held = self.refs.cpu()
        pages = [p for p in range(1, len(held)) if held[p] == 0][:len(slots)]
        if len(pages) < len(slots):
            raise MemoryError(f"{len(slots)} pages wanted, {len(pages)} free")
        at, where = torch.tensor(pages, device=self.device), (
            torch.tensor(slots, device=self.device), torch.tensor(columns, device=self.device))
        self.refs[at] = 1
        self.table[where] = at.int()
        return at, where

    def _put_back(self, taken) -> None:
        """Undoes a ``_take`` whose pages nothing has been forked from."""
        at, where = taken
        self.table[where] = 0
        self.refs[at] = 0

    def _release(self, slots: Sequence[int]) -> None:
        F.free_pages(self.table, self.lens, self.refs, self._i32(list(slots)),
                     out=(self.table, self.lens, self.refs))
        self._free += list(slots)

    @property
    def held(self) -> int:
        """Pages that a slot holds."""
        return int((self.refs > 0).sum())
