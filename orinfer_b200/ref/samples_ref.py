"""64-bit statements of the operators for several samples of one prompt: attention of rows that
share a prefix, the pages of their cache, and what is done to their logits before a draw.

Written from the definitions, page by page and token by token, for tests of the kernels in
``csrc/kernels/attention_shared.cu``, ``pages.cu`` and ``logits.cu``.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

PAGE = 128


def attention_rows(q, gate, row_req, row_pos, page_table, kcache, vcache, kscale, vscale):
    """fp64 [rows, qh * D]: row r against keys 0..row_pos[r] of page-table row row_req[r].  Also
    returns, per row and channel, sum_j p_j |v_j|, and per row and head max_j sum_c |q_c k_jc| /
    sqrt(D): what bounds the effect of roundings of V, and of K on the scores."""
    rows, qh, d = q.shape
    kvh = kcache.shape[2]
    out = torch.zeros(rows, qh, d, dtype=torch.float64, device=q.device)
    size, reach = torch.zeros_like(out), torch.zeros(rows, qh, 1, dtype=torch.float64,
                                                     device=q.device)
    for r, (req, pos) in enumerate(zip(row_req.tolist(), row_pos.tolist())):
        n = pos + 1
        if n <= 0:
            continue
        pages = page_table[req, :(n + PAGE - 1) // PAGE].long()

        def read(codes, scales):
            x = codes[pages].reshape(-1, kvh, d // 64, 64)[:n].double()
            return (x * scales[pages].reshape(-1, kvh, d // 64, 1)[:n].double()) \
                .reshape(n, kvh, d).repeat_interleave(qh // kvh, 1)

        k, v, qr = read(kcache, kscale), read(vcache, vscale), q[r].double()
        p = torch.softmax(torch.einsum("hd,thd->ht", qr, k) / math.sqrt(d), 1)
        out[r] = torch.einsum("ht,thd->hd", p, v)
        size[r] = torch.einsum("ht,thd->hd", p, v.abs())
        reach[r, :, 0] = torch.einsum("hd,thd->ht", qr.abs(), k.abs()).amax(1) / math.sqrt(d)
    if gate is not None:
        g = torch.sigmoid(gate.double().view_as(out))
        out, size = out * g, size * g
    return out.view(rows, -1), size.view(rows, -1), reach.expand(-1, -1, d).reshape(rows, -1)


def fork_pages(tensors, table, lens, refs, parents, children):
    """(table, lens, refs, status) as ``ops.functional.fork_pages``; the cache ``tensors`` are
    changed in place.  Everything on the CPU."""
    table, lens, refs = table.clone(), lens.clone(), refs.clone()
    slots, width = table.shape
    pages = refs.shape[0]
    pairs = list(zip(parents.tolist(), children.tolist()))
    named = [c for _, c in pairs]
    for p, c in pairs:
        if not (0 <= p < slots and 0 <= c < slots) or p in named or named.count(c) > 1:
            return table, lens, refs, 2
        if lens[c] != 0 or not 0 <= lens[p] <= width * PAGE:
            return table, lens, refs, 2
        for j in range((int(lens[p]) + PAGE - 1) // PAGE):
            if not 0 < table[p, j] < pages or refs[table[p, j]] <= 0:
                return table, lens, refs, 2
    free = [p for p in range(1, pages) if refs[p] <= 0]
    if sum(int(lens[p]) % PAGE > 0 for p, _ in pairs) > len(free):
        return table, lens, refs, 1
    for p, c in pairs:
        full, tail = divmod(int(lens[p]), PAGE)
        table[c] = 0
        table[c, :full] = table[p, :full]
        for page in table[c, :full].tolist():
            refs[page] += 1
        if tail:
            page = free.pop(0)
            table[c, full], refs[page] = page, 1
            for t in tensors:
                t[page, :tail] = t[int(table[p, full]), :tail]
        lens[c] = lens[p]
    return table, lens, refs, 0


def free_pages(table, lens, refs, slots):
    table, lens, refs = table.clone(), lens.clone(), refs.clone()
    for s in dict.fromkeys(slots.tolist()):
        for page in table[s].tolist():
            if page:
                refs[page] -= 1
        table[s], lens[s] = 0, 0
    return table, lens, refs


def compact_pages(tensors, table, refs):
    """(table, refs, moved); the cache ``tensors`` are changed in place."""
    live = [p for p in range(1, refs.shape[0]) if refs[p] > 0]
    count = len(live)
    holes = [p for p in range(1, count + 1) if refs[p] <= 0]
    moved = torch.arange(refs.shape[0], dtype=torch.int32)
    refs_out = torch.zeros_like(refs)
    for p in live:
        if p > count:
            to = holes.pop(0)
            moved[p] = to
            for t in tensors:
                t[to] = t[p]
        refs_out[moved[p]] = refs[p]
    return moved[table.long()], refs_out, moved


def process_logits(logits, history=None, repetition=1.0, presence=0.0, frequency=0.0,
                   bias=(), permitted: Optional[torch.Tensor] = None, masked=-1e30):
    """One row: (fp64 scores [vocab], flag).  ``bias``: (token, value) in order; ``permitted``: bool
    [vocab]."""
    s = logits.double().clone()
    wrong = not bool(s.isfinite().all())
    count = torch.zeros_like(s)
    for t in [] if history is None else history:
        if 0 <= t < s.shape[0]:
            count[t] += 1
    if repetition != 1.0 or presence != 0.0 or frequency != 0.0:
        seen = torch.where(s < 0, s * repetition, s / repetition) - presence
        s = torch.where(count > 0, seen, s) - frequency * count
    added = torch.zeros_like(s)
    for t, v in bias:
        if 0 <= t < s.shape[0]:
            added[t] = v
    s = s + added
    allowed = torch.ones_like(s, dtype=torch.bool) if permitted is None else permitted
    wrong = wrong or not bool(s.float()[allowed].isfinite().all())
    return s.masked_fill(~allowed, masked), 2 if wrong else int(not bool(allowed.any()))
