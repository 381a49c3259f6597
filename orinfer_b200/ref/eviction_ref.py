"""64-bit statements of the operators of a cache with a bound: the weight that attention gives to
every key, and which keys stay when a request is cut down.

Written from the definitions, row by row and key by key, for tests of ``attention_weighed``,
``prefill_weights`` and ``evict_keys`` (``csrc/kernels/attention.cu``, ``weigh.cu``, ``evict.cu``).
"""

from __future__ import annotations

import math

import torch

PAGE = 128


def key_weights(q, row_req, row_pos, page_table, kcache, kscale, slots=None):
    """(fp64 [slots, KV heads, keys], reach): the softmax weights that every key gets from the rows,
    row r seeing keys 0..row_pos[r] of table row row_req[r], summed over rows and the query heads of a
    KV head; and the largest sum_c |q_c k_jc| / sqrt(D), which bounds the effect of roundings."""
    rows, qh, d = q.shape
    kvh = kcache.shape[2]
    sums = torch.zeros(slots or page_table.shape[0], kvh, page_table.shape[1] * PAGE,
                       dtype=torch.float64, device=q.device)
    reach = 0.0
    for r, (req, pos) in enumerate(zip(row_req.tolist(), row_pos.tolist())):
        n = pos + 1
        if n <= 0:
            continue
        pages = page_table[req, :(n + PAGE - 1) // PAGE].long()
        k = kcache[pages].reshape(-1, kvh, d // 64, 64)[:n].double()
        k = (k * kscale[pages].reshape(-1, kvh, d // 64, 1)[:n].double()).reshape(n, kvh, d)
        x = q[r].double().view(kvh, qh // kvh, d) / math.sqrt(d)
        p = torch.softmax(torch.einsum("gid,tgd->git", x, k), 2)
        sums[req, :, :n] += p.sum(1)
        reach = max(reach, float(torch.einsum("gid,tgd->git", x.abs(), k.abs()).max()))
    return sums, reach


def chunk_rows(chunks):
    """(rows of q, row_req, row_pos) of the rows of prefill chunks [(first row, rows, position, slot)]."""
    at = [(first + i, slot, pos + i) for first, n, pos, slot in chunks for i in range(n)]
    return tuple(torch.tensor(v, dtype=torch.int64) for v in zip(*at)) if at else \
        (torch.zeros(0, dtype=torch.int64),) * 3


def kept_keys(weights, length, keep, first, recent):
    """Indices of the keys of a head that stay, in order; ``weights`` [at least length]."""
    if length <= keep:
        return list(range(length))
    w = [float(x) for x in weights[:length]]
    w = [-math.inf if math.isnan(x) else x for x in w]
    number = [not math.isnan(float(x)) for x in weights[:length]]
    between = sorted(range(first, length - recent), key=lambda i: (-w[i], not number[i], i))
    return sorted([*range(first), *between[:keep - first - recent], *range(length - recent, length)])


def evict_keys(k, v, ks, vs, table, lens, refs, weights, slots, keep, first=0, recent=0):
    """(table, lens, refs, weights, status) as ``ops.functional.evict_keys``; the layers' caches ``k``,
    ``v``, ``ks``, ``vs`` are changed in place.  Everything on the CPU."""
    before = table, lens, refs, weights
    table, lens, refs, weights = (t.clone() for t in before)
    total, width = table.shape
    pages, kept = refs.shape[0], (keep + PAGE - 1) // PAGE
    named = list(dict.fromkeys(slots.tolist()))
    for s in named:
        if not 0 <= s < total or not 0 <= lens[s] <= width * PAGE:
            return (*before, 2)
        if lens[s] > keep:
            row = table[s].tolist()
            for j, p in enumerate(row):
                if not 0 <= p < pages or (j * PAGE < lens[s] and p == 0) or (p and refs[p] <= 0):
                    return (*before, 2)
    cut = [s for s in named if lens[s] > keep]
    free = [p for p in range(1, pages) if refs[p] <= 0]
    if len(free) < kept * len(cut):
        return (*before, 1)
    for s in cut:
        fresh, free = free[:kept], free[kept:]
        old = before[0][s].tolist()
        for layer, tensors in enumerate(zip(k, v, ks, vs)):
            for h in range(k[0].shape[2]):
                stay = kept_keys(before[3][layer, s, h], int(lens[s]), keep, first, recent)
                for i, j in enumerate(stay):
                    for t in tensors:
                        t[fresh[i // PAGE], i % PAGE, h] = t[old[j // PAGE], j % PAGE, h]
                weights[layer, s, h] = 0
                weights[layer, s, h, :keep] = before[3][layer, s, h, stay]
        for p in old:
            if p:
                refs[p] -= 1
        table[s] = 0
        table[s, :kept] = torch.tensor(fresh, dtype=table.dtype)
        refs[fresh] = 1
        lens[s] = keep
    return table, lens, refs, weights, 0
