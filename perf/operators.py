"""Operators for several samples of one prompt: what they cost at the sizes that serving meets.

``attention_shared`` decodes a batch whose rows share a prefix, ``fork_pages`` / ``free_pages`` /
``compact_pages`` move their paged cache, and ``process_logits`` applies penalties, biases and
grammar masks before a draw.  ``run`` makes the framework's calls where ``own`` is set and states
them in elementary torch operations otherwise; ``exact`` states them in 64 bits.  Geometries are
the presets of ``orinfer_b200.config``.
"""

from __future__ import annotations

import math

import torch

own = False

PAGE = 128                  # tokens of a cache page


# ------------------------------------------------------------------------------- the cases
def listed():
    return [
        # a pair of samples of a short question, the smallest call there is to share
        dict(name="shared_pair", kind="attention", rows=2, groups=1, shared=384, own_keys=40,
             pad=0, qh=32, kvh=8, d=128),
        # a full decode batch under five system prompts, with padded rows of a captured step
        dict(name="shared_prompts", kind="attention", rows=125, groups=5, shared=3840,
             own_keys=700, pad=3, qh=32, kvh=8, d=128),
        # many continuations of a long document
        dict(name="shared_document", kind="attention", rows=64, groups=1, shared=16384,
             own_keys=250, pad=0, qh=32, kvh=4, d=128),
        # the same for gated heads of 256 channels
        dict(name="shared_gated", kind="attention", rows=37, groups=2, shared=6016, own_keys=150,
             pad=1, qh=16, kvh=2, d=256),
        # one request forked into four on the smallest geometry: latency
        dict(name="fork_four", kind="fork", parents=1, per=4, ctx=333, slots=32, spare=40,
             layers=2, kvh=2, d=64),
        # a beam: eight requests, eight branches each, on all layers of a 4B-class model
        dict(name="fork_beams", kind="fork", parents=8, per=8, ctx=1500, slots=128, spare=80,
             layers=36, kvh=8, d=128),
        # one sample of two has ended
        dict(name="free_one", kind="free", parents=1, per=2, ctx=700, slots=32, spare=40),
        # most samples of a full table give their pages back
        dict(name="free_samples", kind="free", parents=16, per=8, ctx=9000, slots=256, spare=500),
        # a small pool with a few holes: latency
        dict(name="compact_few", kind="compact", pages=64, live=0.9, slots=32, layers=2, kvh=2,
             d=64),
        # a fragmented pool of a 4B-class model is made dense
        dict(name="compact_pool", kind="compact", pages=256, live=0.5, slots=128, layers=36,
             kvh=8, d=128),
        # one chat under a repetition penalty
        dict(name="logits_one", kind="logits", rows=1, vocab=151936, history=900, biases=0, masked=0.0),
        # the largest batch: long histories, biases, half of the rows bound by a grammar
        dict(name="logits_full", kind="logits", rows=256, vocab=151936, history=16000, biases=300,
             masked=0.5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "fork", "free", "compact", "logits",
                       "logits"])
    if kind == "attention":
        qh, kvh, d = rng.choice([(32, 8, 128), (40, 8, 128), (32, 4, 128), (16, 2, 256),
                                 (16, 8, 64)])
        rows = _log(rng, 2, 128)
        keys = 1000000 // rows * 4 // kvh // (d // 64) * 2     # the plain form's memory
        shared = PAGE * _log(rng, 1, max(2, min(16384, keys) // PAGE))
        return dict(kind=kind, rows=rows, groups=rng.randint(1, max(1, min(8, rows // 2))),
                    shared=shared, own_keys=_log(rng, 1, min(2000, max(2, keys // 4))),
                    pad=rng.choice([0, 0, rng.randint(1, 5)]), qh=qh, kvh=kvh, d=d)
    kvh, d = rng.choice([(8, 128), (4, 128), (2, 256), (8, 64), (2, 64)])
    layers = rng.randint(1, 36)
    if kind in ("fork", "free"):
        parents = _log(rng, 1, 16)
        per = _log(rng, 1, 64 // parents)
        if kind == "free":
            return dict(kind=kind, parents=parents, per=max(2, per), ctx=_log(rng, 1, 9000),
                        slots=rng.randint(80, 256), spare=rng.randint(0, 500))
        return dict(kind=kind, parents=parents, per=per, ctx=_log(rng, 1, 1500),
                    slots=rng.randint(80, 256), spare=parents * per + rng.randint(0, 30),
                    layers=layers, kvh=kvh, d=d)
    if kind == "compact":
        return dict(kind=kind, pages=_log(rng, 4, 256), live=round(rng.uniform(0.05, 0.95), 3),
                    slots=rng.randint(8, 200), layers=layers, kvh=kvh, d=d)
    return dict(kind=kind, rows=_log(rng, 1, 256), vocab=rng.choice(
                    [151936, 8192, rng.randint(1000, 151936)]), history=_log(rng, 1, 16000),
                biases=rng.choice([0, _log(rng, 1, 300)]),
                masked=rng.choice([0.0, round(rng.uniform(0.1, 1.0), 3)]))


# ----------------------------------------------------------------------------- inputs
class _Rand:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(1000003 * (seed % 1000000007) + 29)

    def normal(self, *shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=self.g, device="cuda") * std).to(dtype)

    def uniform(self, *shape, dtype=torch.float32):
        return torch.rand(*shape, generator=self.g, device="cuda", dtype=dtype)

    def ints(self, lo, hi, shape, dtype=torch.int32):
        return torch.randint(lo, hi, shape, generator=self.g, device="cuda", dtype=dtype)

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


def _groups(c):
    """(first row, rows, shared keys) of every group: ragged, the first with the longest prefix."""
    base, more = divmod(c["rows"], c["groups"])
    out, at = [], 0
    for i in range(c["groups"]):
        n = base + (1 if i < more else 0)
        out.append((at, n, PAGE * _spread(i, min(1, c["shared"] // PAGE), c["shared"] // PAGE)))
        at += n
    return out


def _inputs_attention(c, r):
    groups, total = _groups(c), c["rows"] + c["pad"]
    own_len = [_spread(i, 1, c["own_keys"]) for i in range(c["rows"])]
    shared_of = [s for _, n, s in groups for _ in range(n)]
    lens = [s + n for s, n in zip(shared_of, own_len)]
    width = max((n + PAGE - 1) // PAGE for n in lens)
    pages = sum(s // PAGE for _, _, s in groups) + sum((n + PAGE - 1) // PAGE for n in own_len)
    order = (r.order(pages) + 1).cpu().tolist()
    table, at = [[0] * width for _ in range(total)], 0
    for first, n, s in groups:
        front = order[at:at + s // PAGE]
        at += len(front)
        for i in range(first, first + n):
            back = (own_len[i] + PAGE - 1) // PAGE
            table[i][:len(front) + back] = front + order[at:at + back]
            at += back
    gated = c["d"] == 256
    return dict(q=r.normal(total, c["qh"], c["d"], dtype=torch.float16),
                gate=r.normal(total, c["qh"], c["d"], dtype=torch.float16) if gated else None,
                req=_i32(list(range(total))), pos=_i32([n - 1 for n in lens] + [-1] * c["pad"]),
                table=_i32(table), max_len=max(lens), groups=groups,
                **r.cache(pages + 1, kvh=c["kvh"], d=c["d"]))


def _inputs_slots(c, r):
    """Slots of requests that share their prompts' pages: ``parents`` prompts with, for ``free``,
    ``per`` samples each, on pages in random order with ``spare`` free ones among them."""
    samples = c["per"] if c["kind"] == "free" else 1
    lens = [_spread(i, max(1, c["ctx"] // 2), c["ctx"]) for i in range(c["parents"])]
    full = [n // PAGE for n in lens]
    used = sum(full) + sum(samples for n in lens if n % PAGE)
    total, width = used + c["spare"] + 1, (c["ctx"] + PAGE - 1) // PAGE + 2
    order = (r.order(total - 1) + 1).cpu().tolist()
    slot = r.order(c["slots"]).cpu().tolist()
    table, length = [[0] * width for _ in range(c["slots"])], [0] * c["slots"]
    refs, at, taken = [0] * total, 0, []
    for i, n in enumerate(lens):
        front = order[at:at + full[i]]
        at += full[i]
        for j in range(samples):
            s = slot[len(taken)]
            row = list(front)
            if n % PAGE:
                row.append(order[at])
                at += 1
            table[s][:len(row)] = row
            length[s] = n
            taken.append(s)
            for p in row:
                refs[p] += 1
    return dict(table=_i32(table), lens=_i32(length), refs=_i32(refs), taken=taken,
                unused=slot[len(taken):], pages=total)


def _inputs_fork(c, r):
    st = _inputs_slots(c, r)
    pairs = [(st["taken"][i % c["parents"]], st["unused"][i])
             for i in range(c["parents"] * c["per"])]
    return dict(table=st["table"], lens=st["lens"], refs=st["refs"],
                parents=_i32([p for p, _ in pairs]), children=_i32([k for _, k in pairs]),
                **r.cache(c["layers"], st["pages"], kvh=c["kvh"], d=c["d"]))


def _inputs_free(c, r):
    st = _inputs_slots(c, r)
    gone = [s for i, s in enumerate(st["taken"]) if i % 3]
    return dict(table=st["table"], lens=st["lens"], refs=st["refs"], gone=_i32(gone))


def _inputs_compact(c, r):
    live = min(c["pages"] - 1, max(1, int(c["live"] * c["pages"])))
    used = (r.order(c["pages"] - 1)[:live] + 1).to(torch.int32)
    width = (live + c["slots"] - 1) // c["slots"] + 1
    table = torch.zeros(c["slots"], width, dtype=torch.int32, device="cuda")
    n = c["slots"] * (width - 1)
    table[:, :-1] = torch.nn.functional.pad(used, (0, n - live)).view(width - 1, c["slots"]).t()
    refs = torch.zeros(c["pages"], dtype=torch.int32, device="cuda")
    refs[used.long()] = 1
    return dict(table=table, refs=refs, **r.cache(c["layers"], c["pages"], kvh=c["kvh"], d=c["d"]))


def _inputs_logits(c, r):
    rows, vocab, hist = c["rows"], c["vocab"], c["history"]
    lens = [_spread(i, min(1, hist), hist) for i in range(rows)]
    # tokens of a text: few ids many times, some seen once
    ids = (vocab * r.uniform(rows, hist) ** 6).to(torch.int32).clamp_(max=vocab - 1)
    f64 = lambda lo, hi: r.uniform(rows, dtype=torch.float64) * (hi - lo) + lo
    every = torch.arange(rows, device="cuda") % 4
    st = dict(logits=r.normal(rows, vocab, std=3.0), history=ids, history_len=_i32(lens),
              repetition=torch.where(every == 3, 1.0, f64(1.0, 1.3)),
              presence=torch.where(every >= 2, 0.0, f64(-0.5, 1.5)),
              frequency=torch.where(every >= 2, 0.0, f64(0.0, 0.5)),
              bias_start=None, bias_ids=None, bias_values=None, mask=None, mask_rows=None)
    if c["biases"]:
        count = [_spread(i, 0, c["biases"]) for i in range(rows)]
        total = sum(count)
        start = [sum(count[:i]) for i in range(rows + 1)]
        st.update(bias_start=_i32(start),
                  bias_ids=torch.cat([r.order(vocab)[:n] for n in count]).to(torch.int32),
                  bias_values=r.uniform(total, dtype=torch.float64) * 20 - 10)
    if c["masked"]:
        n = max(1, int(c["masked"] * rows))
        # a grammar permits a handful of tokens or most of them
        share = torch.where(torch.arange(n, device="cuda") % 2 == 0, 0.001, 0.9)
        words = (vocab + 31) // 32
        st["mask"] = torch.zeros(n, words, dtype=torch.int32, device="cuda")
        for bit in range(32):
            on = r.uniform(n, words) < share[:, None]
            st["mask"] |= on.to(torch.int32) << bit
        st["mask"][:, 7] |= 1                       # always something
        which = [-1] * rows
        for i in range(n):
            which[i * 7919 % rows] = i
        st["mask_rows"] = _i32(which)
    return st


_INPUTS = dict(attention=_inputs_attention, fork=_inputs_fork, free=_inputs_free,
               compact=_inputs_compact, logits=_inputs_logits)


def prepare(case, seed):
    st = dict(_INPUTS[case["kind"]](case, _Rand(seed)), kind=case["kind"])
    if own:
        # what a program keeps from step to step: the plan of its batch, the handle of its cache
        from orinfer_b200.ops import functional as F, native
        native.init()
        if case["kind"] == "attention":
            st["plan"] = F.SharedPrefix(st["groups"], case["rows"] + case["pad"], qh=case["qh"],
                                        kvh=case["kvh"], head_dim=case["d"],
                                        max_kv_len=st["max_len"], device="cuda")
        elif case["kind"] in ("fork", "compact"):
            st["cache"] = F.CachePages([t for name in ("k", "v", "ks", "vs")
                                        for t in st[name].unbind(0)])
    return st


# ----------------------------------------------------------------------------- one pass
def run(st):
    return (_OWN if own else _PLAIN)[st["kind"]](st)


def _own_attention(st):
    from orinfer_b200.ops import functional as F
    return F.attention_shared(st["q"], st["gate"], st["req"], st["pos"], st["table"], st["k"],
                              st["v"], st["ks"], st["vs"], st["plan"])


def _own_fork(st):
    from orinfer_b200.ops import functional as F
    table, lens, refs, status = F.fork_pages(st["cache"], st["table"], st["lens"], st["refs"],
                                             st["parents"], st["children"])
    return dict(table=table, lens=lens, refs=refs, status=status, k=st["k"], v=st["v"],
                ks=st["ks"], vs=st["vs"])


def _own_free(st):
    from orinfer_b200.ops import functional as F
    table, lens, refs = F.free_pages(st["table"], st["lens"], st["refs"], st["gone"])
    return dict(table=table, lens=lens, refs=refs)


def _own_compact(st):
    from orinfer_b200.ops import functional as F
    table, refs, moved = F.compact_pages(st["cache"], st["table"], st["refs"])
    return dict(table=table, refs=refs, moved=moved, k=st["k"], v=st["v"], ks=st["ks"],
                vs=st["vs"])


def _own_logits(st):
    from orinfer_b200.ops import functional as F
    out, flags = F.process_logits(
        st["logits"], history=st["history"], history_len=st["history_len"],
        repetition=st["repetition"], presence=st["presence"], frequency=st["frequency"],
        bias_start=st["bias_start"], bias_ids=st["bias_ids"], bias_values=st["bias_values"],
        mask=st["mask"], mask_rows=st["mask_rows"], masked=-math.inf)
    return dict(out=out, flags=flags)


def _plain_attention(st):
    rows, qh, d = st["q"].shape
    kvh = st["k"].shape[2]
    pages = st["table"].long()
    keys = pages.shape[1] * PAGE

    def gather(codes, scales):
        x = codes[pages].float().view(rows, keys, kvh, d // 64, 64)
        x *= scales[pages].float().view(rows, keys, kvh, d // 64, 1)
        return x.view(rows, keys, kvh, d)

    q = st["q"].float().view(rows, kvh, qh // kvh, d) * d ** -0.5
    s = torch.einsum("rgid,rtgd->rgit", q, gather(st["k"], st["ks"]))
    dead = torch.arange(keys, device="cuda")[None, :] > st["pos"][:, None]
    s = s.masked_fill(dead[:, None, None], -1e30)
    p = (s - s.amax(-1, keepdim=True)).exp().masked_fill(dead[:, None, None], 0.0)
    total = p.sum(-1, keepdim=True)
    o = torch.einsum("rgit,rtgd->rgid", p, gather(st["v"], st["vs"])) / total.clamp(min=1e-30)
    o = o.reshape(rows, qh * d)
    if st["gate"] is not None:
        o = o / (1 + (-st["gate"].float().view(rows, qh * d)).exp())
    return o.to(torch.float16)


def _free_pages(refs):
    """Free pages from the lowest up, as far as there are any (page 0 is nobody's)."""
    used = (refs > 0).int()
    used[0] = 1
    return torch.sort(used, stable=True).indices


def _plain_fork(st):
    table, lens, refs = st["table"].clone(), st["lens"].clone(), st["refs"].clone()
    parents, children = st["parents"].long(), st["children"].long()
    n, tail = lens[parents], lens[parents] % PAGE
    full, fresh = n // PAGE, (tail > 0)
    free = _free_pages(refs)
    mine = torch.where(fresh, free[(fresh.cumsum(0) - 1).clamp(min=0)], 0)
    short = (fresh.sum() > (refs[1:] <= 0).sum()).int()
    at = torch.arange(table.shape[1], device="cuda")[None, :]
    kept = at < full[:, None]
    source = table[parents]
    rows = torch.where(kept, source, torch.where((at == full[:, None]) & fresh[:, None],
                                                 mine[:, None].int(), 0))
    table[children] = rows
    lens[children] = n
    refs.index_add_(0, rows.reshape(-1).long(), (rows > 0).reshape(-1).int())
    last = torch.where(fresh, source.gather(1, full[:, None].long().clamp(max=table.shape[1] - 1))
                       [:, 0].long(), 0)
    live = torch.arange(PAGE, device="cuda")[None, :] < tail[:, None]

    def copy(x):
        x[:, mine] = torch.where(live[None, :, :, None, None], x[:, last], x[:, mine])
        return x

    return dict(table=table, lens=lens, refs=refs, status=short.view(1), k=copy(st["k"]),
                v=copy(st["v"]), ks=copy(st["ks"]), vs=copy(st["vs"]))


def _plain_free(st):
    table, lens, refs = st["table"].clone(), st["lens"].clone(), st["refs"].clone()
    gone = st["gone"].long()
    pages = table[gone].reshape(-1).long()
    refs.index_add_(0, pages, -(pages > 0).int())
    table[gone] = 0
    lens[gone] = 0
    return dict(table=table, lens=lens, refs=refs)


def _plain_compact(st):
    refs = st["refs"]
    pages = torch.arange(refs.shape[0], device="cuda")
    live = (refs > 0) & (pages > 0)
    count = live.sum()
    holes, tops = ~live & (pages > 0) & (pages <= count), live & (pages > count)
    # the k-th page above the count goes to the k-th hole; at most half of the pages move
    most = refs.shape[0] // 2
    source = torch.sort((~tops).int(), stable=True).indices[:most]
    target = torch.sort((~holes).int(), stable=True).indices[:most]
    source, target = torch.where(tops[source], source, 0), torch.where(holes[target], target, 0)
    moved = pages.scatter(0, source, target)
    refs_out = torch.zeros_like(refs).index_add_(0, moved, torch.where(live, refs, 0))

    def copy(x):
        x[:, target] = x[:, source]
        return x

    return dict(table=moved.int()[st["table"].long()], refs=refs_out, moved=moved.int(),
                k=copy(st["k"]), v=copy(st["v"]), ks=copy(st["ks"]), vs=copy(st["vs"]))


def _plain_logits(st):
    x = st["logits"]
    rows, vocab = x.shape
    seen = torch.arange(st["history"].shape[1], device="cuda")[None, :] < st["history_len"][:, None]
    count = torch.zeros(rows, vocab, device="cuda")
    count.scatter_add_(1, st["history"].long(), seen.float())
    col = lambda name: st[name].float()[:, None]
    s = torch.where(count > 0, torch.where(x < 0, x * col("repetition"), x / col("repetition"))
                    - col("presence"), x) - col("frequency") * count
    if st["bias_ids"] is not None:
        at = torch.arange(st["bias_ids"].shape[0], device="cuda", dtype=torch.int32)
        row = torch.searchsorted(st["bias_start"], at, right=True) - 1
        bias = torch.zeros(rows, vocab, device="cuda")
        bias[row, st["bias_ids"].long()] = st["bias_values"].float()
        s = s + bias
    allowed = torch.ones_like(x, dtype=torch.bool)
    if st["mask"] is not None:
        bits = (st["mask"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        allowed = bits.view(bits.shape[0], -1)[:, :vocab] > 0
        allowed = allowed[st["mask_rows"].long().clamp(min=0)] | (st["mask_rows"] < 0)[:, None]
    wrong = (~x.isfinite() | (allowed & ~s.isfinite())).any(1)
    flags = torch.where(wrong, 2, (~allowed.any(1)).int())
    s = s.masked_fill(~allowed, -math.inf)
    return dict(out=s, flags=flags.int())


_OWN = dict(attention=_own_attention, fork=_own_fork, free=_own_free, compact=_own_compact,
            logits=_own_logits)
_PLAIN = dict(attention=_plain_attention, fork=_plain_fork, free=_plain_free,
              compact=_plain_compact, logits=_plain_logits)


# ----------------------------------------------------------------------------- work
def _lengths(c):
    """(shared keys, own keys) of every row of an attention case."""
    shared = [s for _, n, s in _groups(c) for _ in range(n)]
    return [(s, _spread(i, 1, c["own_keys"])) for i, s in enumerate(shared)]


def work(case):
    c = case
    if c["kind"] == "attention":
        per_key = c["kvh"] * (2 * c["d"] + 4 * (c["d"] // 64))
        rows, keys = _lengths(c), sum(s for _, _, s in _groups(c))
        io = (c["rows"] + c["pad"]) * c["qh"] * c["d"] * 2 * (3 if c["d"] == 256 else 2)
        return dict(bytes=per_key * (keys + sum(n for _, n in rows)) + io,
                    flops=4 * c["qh"] * c["d"] * sum(s + n for s, n in rows))
    token = 0 if "layers" not in c else c["layers"] * c["kvh"] * (2 * c["d"] + 4 * (c["d"] // 64))
    if c["kind"] in ("fork", "free"):
        lens = [_spread(i, max(1, c["ctx"] // 2), c["ctx"]) for i in range(c["parents"])]
        width = (c["ctx"] + PAGE - 1) // PAGE + 2
        samples = c["per"] if c["kind"] == "free" else 1
        pages = sum(n // PAGE for n in lens) + samples * sum(n % PAGE > 0 for n in lens) \
            + c["spare"] + 1
        moved = c["per"] * sum(n % PAGE for n in lens) * token if c["kind"] == "fork" else 0
        return dict(bytes=2 * moved + 8 * (c["slots"] * (width + 1) + pages), flops=0)
    if c["kind"] == "compact":
        live = min(c["pages"] - 1, max(1, int(c["live"] * c["pages"])))
        # pages in random order: this share of the live ones lies above their number
        moves = live * (c["pages"] - 1 - live) / max(1, c["pages"] - 1)
        width = (live + c["slots"] - 1) // c["slots"] + 1
        return dict(bytes=2 * moves * PAGE * token + 8 * c["slots"] * width + 12 * c["pages"],
                    flops=0)
    masks = int(c["masked"] * c["rows"]) * c["vocab"] // 8
    history = sum(_spread(i, min(1, c["history"]), c["history"]) for i in range(c["rows"]))
    return dict(bytes=8 * c["rows"] * c["vocab"] + masks + 4 * history, flops=0)


# ----------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    if case["kind"] not in ("attention", "logits"):
        return None                                   # whole numbers: there is nothing to round
    st = _INPUTS[case["kind"]](case, _Rand(seed))
    return (_exact_attention if case["kind"] == "attention" else _exact_logits)(st)


def _exact_attention(st):
    """Row by row, key by key group: the definition, without a shared part or a table of masks."""
    rows, qh, d = st["q"].shape
    kvh = st["k"].shape[2]
    out = torch.zeros(rows, qh, d, dtype=torch.float64, device="cuda")
    for r, last in enumerate(st["pos"].tolist()):
        n = last + 1
        if n <= 0:
            continue
        pages = st["table"][r, :(n + PAGE - 1) // PAGE].long()

        def read(codes, scales):
            x = codes[pages].reshape(-1, kvh, d // 64, 64)[:n].double()
            return (x * scales[pages].reshape(-1, kvh, d // 64)[:n].double()[..., None]) \
                .reshape(n, kvh, d)

        k, v = read(st["k"], st["ks"]), read(st["v"], st["vs"])
        for h in range(kvh):
            mine = slice(h * (qh // kvh), (h + 1) * (qh // kvh))
            weights = torch.softmax(st["q"][r, mine].double() @ k[:, h].t() / math.sqrt(d), 1)
            out[r, mine] = weights @ v[:, h]
    if st["gate"] is not None:
        out = out * torch.sigmoid(st["gate"].double())
    return out.view(rows, qh * d)


def _exact_logits(st):
    x = st["logits"].double()
    for r, n in enumerate(st["history_len"].tolist()):
        ids, count = torch.unique(st["history"][r, :n].long(), return_counts=True)
        s, rep = x[r, ids], st["repetition"][r]
        x[r, ids] = torch.where(s < 0, s * rep, s / rep) - st["presence"][r] \
            - st["frequency"][r] * count
        if st["bias_ids"] is not None:
            lo, hi = st["bias_start"][r:r + 2].tolist()
            x[r, st["bias_ids"][lo:hi].long()] += st["bias_values"][lo:hi]
        which = -1 if st["mask"] is None else int(st["mask_rows"][r])
        if which >= 0:
            at = torch.arange(x.shape[1], device="cuda")
            x[r, (st["mask"][which][at // 32] >> (at % 32)) & 1 == 0] = -math.inf
    return dict(out=x, flags=None)
