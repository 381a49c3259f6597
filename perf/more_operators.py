"""Operators of a cache with a bound: what they cost at the sizes that serving meets.

``attention_weighed`` is decode attention that also adds up the attention weight of every key,
``prefill_weights`` adds up the weights that a prompt's rows give, and ``evict_keys`` keeps the
keys with the most weight and gives the pages of the others back.  ``run`` makes the framework's
calls where ``own`` is set and states them in elementary torch operations otherwise; ``exact``
states them in 64 bits.  Geometries are the presets of ``orinfer_b200.config``.
"""

from __future__ import annotations

import math

import torch

own = False

PAGE = 128                  # tokens of a cache page


# ------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one chat under a small budget, the smallest step there is
        dict(name="step_one", kind="step", rows=1, per=1, keys=300, pad=0, qh=32, kvh=8, d=128),
        # a full decode batch of short requests, with padded rows of a captured step
        dict(name="step_batch", kind="step", rows=125, per=1, keys=640, pad=3, qh=32, kvh=8,
             d=128),
        # a few long requests: the cache is read at the memory's rate
        dict(name="step_long", kind="step", rows=6, per=1, keys=24000, pad=0, qh=32, kvh=8, d=128),
        # gated heads of 256 channels, four rows of each request verified together
        dict(name="step_gated", kind="step", rows=36, per=4, keys=3000, pad=1, qh=16, kvh=2, d=256),
        # a short question on the smallest geometry
        dict(name="prompt_short", kind="prompt", chunks=1, rows=61, before=0, qh=4, kvh=2, d=64),
        # a long prompt
        dict(name="prompt_full", kind="prompt", chunks=1, rows=4096, before=0, qh=32, kvh=8, d=128),
        # two chunks of prompts that are prefilled in pieces, gated heads of 256 channels
        dict(name="prompt_chunks", kind="prompt", chunks=2, rows=777, before=3000, qh=16, kvh=2,
             d=256),
        # the last rows of long prompts weigh all of their keys
        dict(name="prompt_window", kind="prompt", chunks=6, rows=64, before=20000, qh=32, kvh=8,
             d=128),
        # one request of the smallest geometry: latency
        dict(name="evict_one", kind="evict", slots=1, table=32, len=700, keep=256, first=4,
             recent=32, share=0, layers=2, kvh=2, d=64),
        # a batch that has reached its budget, on all layers of a 4B-class model
        dict(name="evict_batch", kind="evict", slots=11, table=64, len=1450, keep=1000, first=4,
             recent=100, share=0, layers=36, kvh=8, d=128),
        # two long prompts are cut down to a sixth
        dict(name="evict_long", kind="evict", slots=2, table=32, len=12000, keep=2000, first=0,
             recent=64, share=0, layers=36, kvh=8, d=128),
        # samples of one prompt, whose pages they share, heads of 256 channels
        dict(name="evict_samples", kind="evict", slots=17, table=128, len=2100, keep=1100, first=16,
             recent=256, share=1500, layers=12, kvh=2, d=256),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["step", "prompt", "evict"])
    qh, kvh, d = rng.choice([(32, 8, 128), (40, 8, 128), (32, 4, 128), (16, 2, 256), (16, 8, 64),
                             (4, 2, 64)])
    if kind == "step":
        rows = _log(rng, 1, 128)
        keys = 700000 * 8 * 128 // (rows * kvh * d)            # the plain form's memory
        return dict(kind=kind, rows=rows, per=rng.choice([1, 1, 1, rng.randint(2, 8)]),
                    keys=_log(rng, 8, max(9, min(24000, keys))),
                    pad=rng.choice([0, 0, rng.randint(1, 5)]), qh=qh, kvh=kvh, d=d)
    if kind == "prompt":
        chunks = _log(rng, 1, 8)
        most = 4096 * 2048 * 32 * 128 // (chunks * qh * d)     # (row, key) pairs of a chunk
        rows = _log(rng, 1, min(4096, int(math.sqrt(2 * most))))
        before = min(20000, most // rows - rows // 2)
        return dict(kind=kind, chunks=chunks, rows=rows, qh=qh, kvh=kvh, d=d,
                    before=0 if before < 2 else rng.choice([0, _log(rng, 1, before)]))
    slots, layers = _log(rng, 1, 32), _log(rng, 1, 36)
    most = 11000 * 36 * 8 * 128 // (layers * kvh * d * slots)  # keys kept of a slot
    length = _log(rng, 16, min(12000, 2 * most))
    keep = max(2, min(most, int(length * rng.uniform(0.1, 0.95))))
    recent = rng.randint(0, keep // 2)
    return dict(kind=kind, slots=slots, table=slots + rng.randint(0, 100), len=length, keep=keep,
                first=rng.randint(0, min(64, keep - recent)), recent=recent,
                share=rng.choice([0, 0, length // 2]), layers=layers, kvh=kvh, d=d)


# ----------------------------------------------------------------------------- inputs
class _Rand:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(1000003 * (seed % 1000000007) + 41)

    def normal(self, *shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=self.g, device="cuda") * std).to(dtype)

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.g, device="cuda")

    def order(self, n):
        return torch.randperm(n, generator=self.g, device="cuda")

    def cache(self, *lead, kvh, d):
        """INT8 values as quantised Gaussian keys have them, and their FP16 group scales."""
        codes = lambda: (self.normal(*lead, PAGE, kvh, d, dtype=torch.float16) * 33) \
            .clamp_(-127, 127).round_().to(torch.int8)
        scales = lambda: ((self.uniform(*lead, PAGE, kvh, d // 64) + 0.5) / 33).to(torch.float16)
        return dict(k=codes(), v=codes(), ks=scales(), vs=scales())


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _spread(i, lo, hi):
    """A number from lo to hi for item i of a ragged batch; the first gets hi."""
    return lo + int(round((hi - lo) * (1.0 - (0.618034 * i) % 1.0)))


def _page_table(lens, width, r):
    """Rows of a page table whose pages lie in random order, and how many pages there are."""
    counts = [-(-n // PAGE) for n in lens]
    order = (r.order(sum(counts)) + 1).cpu().tolist()
    table, at = [[0] * width for _ in lens], 0
    for row, n in zip(table, counts):
        row[:n] = order[at:at + n]
        at += n
    return table, sum(counts) + 1


def _weights(r, *shape):
    """Sums of attention weights: few keys with much, most with little."""
    return r.uniform(*shape) ** 8 * 0.2


def _step_requests(c):
    """Keys that the last row of each request of a decode batch sees."""
    n = -(-c["rows"] // c["per"])
    return [max(c["per"], _spread(i, max(1, c["keys"] // 2), c["keys"])) for i in range(n)]


def _inputs_step(c, r):
    lens, per = _step_requests(c), c["per"]
    req = [i // per for i in range(c["rows"])]
    pos = [lens[i // per] - per + i % per for i in range(c["rows"])]
    table, pages = _page_table(lens, -(-max(lens) // PAGE), r)
    total = c["rows"] + c["pad"]
    gated = c["d"] == 256
    q = r.normal(total, c["qh"], c["d"], dtype=torch.float16)
    weights = _weights(r, len(lens), c["kvh"], len(table[0]) * PAGE)
    return dict(q=q, gate=r.normal(*q.shape, dtype=torch.float16) if gated else None,
                req=_i32(req + [0] * c["pad"]), pos=_i32(pos + [-1] * c["pad"]),
                table=_i32(table), max_len=max(lens), weights=weights, sums=weights.clone(),
                **r.cache(pages, kvh=c["kvh"], d=c["d"]))


def _prompt_chunks(c):
    """(rows, position of the first) of every chunk."""
    return [(_spread(i, max(1, c["rows"] // 2), c["rows"]),
             _spread(i, c["before"] // 2, c["before"])) for i in range(c["chunks"])]


def _inputs_prompt(c, r):
    spans = _prompt_chunks(c)
    lens = [n + p for n, p in spans]
    table, pages = _page_table(lens, -(-max(lens) // PAGE), r)
    chunks, at = [], 0
    for i, (n, p) in enumerate(spans):
        chunks.append([at, n, p, i])
        at += n
    cache = r.cache(pages, kvh=c["kvh"], d=c["d"])
    weights = _weights(r, len(lens), c["kvh"], len(table[0]) * PAGE)
    return dict(q=r.normal(at, c["qh"], c["d"], dtype=torch.float16), chunks=_i32(chunks),
                longest=max(n for n, _ in spans), max_len=max(lens), table=_i32(table),
                k=cache["k"], ks=cache["ks"], weights=weights, sums=weights.clone())


def _evict_slots(c):
    """(tokens, whole pages shared) of every slot; the last of several may be within its budget."""
    lens = [_spread(i, max(1, c["len"] // 2, c["keep"] - 20), c["len"]) for i in range(c["slots"])]
    return [(n, min(n, c["share"]) // PAGE) for n in lens]


def _inputs_evict(c, r):
    spans, kept = _evict_slots(c), -(-c["keep"] // PAGE)
    common = max(s for _, s in spans)
    counts = [-(-n // PAGE) - s for n, s in spans]
    total = common + sum(counts) + kept * c["slots"] + 2
    order = (r.order(total - 1) + 1).cpu().tolist()
    front, at = order[:common], common
    width = -(-c["len"] // PAGE) + 1
    place = r.order(c["table"])[:c["slots"]].cpu().tolist()
    table, lens = [[0] * width for _ in range(c["table"])], [0] * c["table"]
    refs = [0] * total
    for slot, (n, s), more in zip(place, spans, counts):
        row = front[:s] + order[at:at + more]
        at += more
        table[slot][:len(row)] = row
        lens[slot] = n
        for p in row:
            refs[p] += 1
    weights = _weights(r, c["layers"], c["table"], c["kvh"], width * PAGE)
    return dict(table=_i32(table), lens=_i32(lens), refs=_i32(refs), slots=_i32(place),
                keep=c["keep"], first=c["first"], recent=c["recent"], weights=weights,
                sums=weights.clone(), **r.cache(c["layers"], total, kvh=c["kvh"], d=c["d"]))


_INPUTS = dict(step=_inputs_step, prompt=_inputs_prompt, evict=_inputs_evict)


def prepare(case, seed):
    st = dict(_INPUTS[case["kind"]](case, _Rand(seed)), kind=case["kind"])
    if own:
        # what a program keeps: the handle of its cache, the splits of its batch
        from orinfer_b200.ops import functional as F, native
        native.init()
        if case["kind"] == "evict":
            st["cache"] = F.KeyCache(*(list(st[name].unbind(0)) for name in ("k", "v", "ks", "vs")))
        elif case["kind"] == "step":
            st["splits"] = F.attention_splits(st["max_len"], st["q"].shape[0], case["kvh"])
    return st


# ----------------------------------------------------------------------------- one pass
def run(st):
    return (_OWN if own else _PLAIN)[st["kind"]](st)


def _own_step(st):
    from orinfer_b200.ops import functional as F
    out = F.attention_weighed(st["q"], st["gate"], st["req"], st["pos"], st["table"], st["k"],
                              st["v"], st["ks"], st["vs"], st["weights"], splits=st["splits"],
                              max_kv_len=st["max_len"], weights_out=st["sums"])
    return dict(out=out, weights=st["sums"])


def _own_prompt(st):
    from orinfer_b200.ops import functional as F
    F.prefill_weights(st["q"], st["chunks"], st["longest"], st["table"], st["k"], st["ks"],
                      st["weights"], max_kv_len=st["max_len"], weights_out=st["sums"])
    return dict(weights=st["sums"])


def _own_evict(st):
    from orinfer_b200.ops import functional as F
    table, lens, refs, status = F.evict_keys(
        st["cache"], st["table"], st["lens"], st["refs"], st["weights"], st["slots"], st["keep"],
        first=st["first"], recent=st["recent"], weights_out=st["sums"])
    return dict(table=table, lens=lens, refs=refs, status=status, weights=st["sums"], k=st["k"],
                v=st["v"], ks=st["ks"], vs=st["vs"])


def _read(codes, scales, pages):
    """FP32 [requests, keys, KV heads, D] of the pages of each."""
    x = codes[pages].float()
    n, w, _, kvh, d = x.shape
    x = x.view(n, w * PAGE, kvh, d // 64, 64)
    x *= scales[pages].float().view(n, w * PAGE, kvh, d // 64, 1)
    return x.view(n, w * PAGE, kvh, d)


def _plain_step(st):
    rows, qh, d = st["q"].shape
    kvh = st["k"].shape[2]
    pages = st["table"].long()[st["req"].long()]
    keys = pages.shape[1] * PAGE
    q = st["q"].float().view(rows, kvh, qh // kvh, d) * d ** -0.5
    s = torch.einsum("rgid,rtgd->rgit", q, _read(st["k"], st["ks"], pages))
    dead = torch.arange(keys, device="cuda")[None, :] > st["pos"][:, None]
    s = s.masked_fill(dead[:, None, None], -1e30)
    p = (s - s.amax(-1, keepdim=True)).exp().masked_fill(dead[:, None, None], 0.0)
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = torch.einsum("rgit,rtgd->rgid", p, _read(st["v"], st["vs"], pages)).reshape(rows, qh * d)
    if st["gate"] is not None:
        o = o / (1 + (-st["gate"].float().view(rows, qh * d)).exp())
    sums = st["sums"].copy_(st["weights"])
    sums.index_add_(0, st["req"].long(), p.sum(2))
    return dict(out=o.to(torch.float16), weights=sums)


def _plain_prompt(st):
    total, qh, d = st["q"].shape
    kvh = st["k"].shape[2]
    first, n, before, slot = st["chunks"].long().unbind(1)
    chunks, longest = first.shape[0], st["longest"]
    at = torch.arange(longest, device="cuda")
    there = at[None, :] < n[:, None]
    q = st["q"][(first[:, None] + at[None, :]).clamp(max=total - 1)].float() * d ** -0.5
    k = _read(st["k"], st["ks"], st["table"].long()[slot])
    s = torch.einsum("crgid,ctgd->cgirt", q.view(chunks, longest, kvh, qh // kvh, d), k)
    sees = torch.arange(k.shape[1], device="cuda")[None, None, :] <= (before[:, None] + at)[..., None]
    sees &= there[..., None]
    s = s.masked_fill(~sees[:, None, None], -1e30)
    s = (s - s.amax(-1, keepdim=True)).exp_().masked_fill_(~sees[:, None, None], 0.0)
    s /= s.sum(-1, keepdim=True).clamp(min=1e-30)
    sums = st["sums"].copy_(st["weights"])
    sums.index_add_(0, slot, s.sum((2, 3)))
    return dict(weights=sums)


def _plain_evict(st):
    table, lens, refs = st["table"].clone(), st["lens"].clone(), st["refs"].clone()
    keep, first, recent = st["keep"], st["first"], st["recent"]
    slots = st["slots"].long()
    n = lens[slots]
    cut = n > keep
    old = table[slots].long()
    width, kept = table.shape[1], -(-keep // PAGE)
    # pages: the lowest free ones, in the order of the slots
    used = (refs > 0).int()
    used[0] = 1
    free = torch.sort(used, stable=True).indices
    place = ((cut.long().cumsum(0) - 1).clamp(min=0) * kept)[:, None] \
        + torch.arange(width, device="cuda")
    inside = torch.arange(width, device="cuda")[None, :] < kept
    fresh = torch.where(inside, free[place.clamp(max=free.shape[0] - 1)], 0)
    short = (cut.sum() * kept > (refs[1:] <= 0).sum()).int()
    rows = torch.where(cut[:, None], fresh, old)
    table[slots] = rows.int()
    lens[slots] = torch.where(cut, keep, n).int()
    refs.index_add_(0, old.reshape(-1), -(cut[:, None] & (old > 0)).int().reshape(-1))
    refs.index_add_(0, fresh.reshape(-1), (cut[:, None] & inside).int().reshape(-1))
    # keys: the first, the last and the heaviest of the others
    w = st["weights"][:, slots]
    cap = w.shape[-1]
    at = torch.arange(cap, device="cuda")[None, :]
    always = (at < first) | (at >= n[:, None] - recent)
    rank = w.masked_fill(always[:, None], math.inf).masked_fill((at >= n[:, None])[:, None],
                                                                -math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    source = torch.sort(order, dim=-1).values
    to = torch.arange(keep, device="cuda")
    source = torch.where(cut[:, None, None], source, to)              # [layers, slots, heads, keep]
    layers, _, kvh, _ = source.shape
    layer = torch.arange(layers, device="cuda")[:, None, None, None]
    slot = torch.arange(slots.shape[0], device="cuda")[None, :, None, None]
    head = torch.arange(kvh, device="cuda")[None, None, :, None]
    page, target = old[slot, source // PAGE], rows[slot, (to // PAGE)]

    def move(x):
        x[layer, target, to % PAGE, head] = x[layer, page, source % PAGE, head]
        return x

    moved = torch.where(cut[:, None, None], torch.nn.functional.pad(w.gather(-1, source),
                                                                   (0, cap - keep)), w)
    sums = st["sums"].copy_(st["weights"])
    sums[:, slots] = moved
    return dict(table=table, lens=lens, refs=refs, status=short.view(1), weights=sums,
                k=move(st["k"]), v=move(st["v"]), ks=move(st["ks"]), vs=move(st["vs"]))


_OWN = dict(step=_own_step, prompt=_own_prompt, evict=_own_evict)
_PLAIN = dict(step=_plain_step, prompt=_plain_prompt, evict=_plain_evict)


# ----------------------------------------------------------------------------- work
def work(case):
    c = case
    key = c["kvh"] * (c["d"] + 2 * (c["d"] // 64))             # bytes of a key, or a value
    if c["kind"] == "step":
        lens, per = _step_requests(c), c["per"]
        seen = sum(lens[i // per] - per + i % per + 1 for i in range(c["rows"]))
        io = (c["rows"] + c["pad"]) * c["qh"] * c["d"] * 2 * (3 if c["d"] == 256 else 2)
        return dict(bytes=sum(lens) * (2 * key + 8 * c["kvh"]) + io,
                    flops=4 * c["qh"] * c["d"] * seen)
    if c["kind"] == "prompt":
        spans = _prompt_chunks(c)
        seen = sum(n * p + n * (n + 1) // 2 for n, p in spans)
        return dict(bytes=sum(n + p for n, p in spans) * (key + 8 * c["kvh"])
                    + sum(n for n, _ in spans) * c["qh"] * c["d"] * 2,
                    flops=2 * c["qh"] * c["d"] * seen)
    width = -(-c["len"] // PAGE) + 1
    lens = [n for n, _ in _evict_slots(c)]
    cut = sum(n > c["keep"] for n in lens)
    sums = sum(4 * n + 4 * width * PAGE for n in lens)
    return dict(bytes=c["layers"] * (4 * cut * c["keep"] * key + c["kvh"] * sums)
                + 8 * c["table"] * (width + 1), flops=0)


# ----------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    if case["kind"] == "evict":
        return None                                   # copies and whole numbers: nothing to round
    st = _INPUTS[case["kind"]](case, _Rand(seed))
    return (_exact_step if case["kind"] == "step" else _exact_prompt)(st)


def _read64(st, which, slot, head, n):
    """fp64 [n, D]: what a KV head has of the first ``n`` tokens of a request."""
    pages = st["table"][slot, :(n + PAGE - 1) // PAGE].long()
    codes = st[which][pages][:, :, head].reshape(-1, st["k"].shape[3])[:n].double()
    scales = st[which + "s"][pages][:, :, head].reshape(-1, st["ks"].shape[3])[:n].double()
    return codes * scales.repeat_interleave(64, 1)


def _exact_step(st):
    """Row by row and head by head."""
    rows, qh, d = st["q"].shape
    kvh = st["k"].shape[2]
    rep = qh // kvh
    out = torch.zeros(rows, qh, d, dtype=torch.float64, device="cuda")
    sums = st["weights"].double()
    for r, (slot, last) in enumerate(zip(st["req"].tolist(), st["pos"].tolist())):
        n = last + 1
        for g in range(kvh if n > 0 else 0):
            mine = slice(g * rep, (g + 1) * rep)
            p = torch.softmax(st["q"][r, mine].double() @ _read64(st, "k", slot, g, n).t()
                              / math.sqrt(d), 1)
            out[r, mine] = p @ _read64(st, "v", slot, g, n)
            sums[slot, g, :n] += p.sum(0)
    if st["gate"] is not None:
        out = out * torch.sigmoid(st["gate"].double())
    return dict(out=out.view(rows, qh * d), weights=sums)


def _exact_prompt(st):
    """Chunk by chunk and head by head."""
    d, kvh = st["q"].shape[2], st["k"].shape[2]
    rep = st["q"].shape[1] // kvh
    sums = st["weights"].double()
    for first, n, before, slot in st["chunks"].tolist():
        sees = torch.ones(n, n + before, dtype=torch.bool, device="cuda").tril(before)
        for g in range(kvh):
            k = _read64(st, "k", slot, g, n + before)
            for h in range(g * rep, (g + 1) * rep):
                s = st["q"][first:first + n, h].double() @ k.t() / math.sqrt(d)
                sums[slot, g, :n + before] += torch.softmax(s.masked_fill(~sees, -math.inf), 1).sum(0)
    return dict(weights=sums)
