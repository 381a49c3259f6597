"""Tensor-level wrappers of the CUDA kernels (one function per device op).

Every wrapper validates shapes/dtypes, takes optional preallocated outputs (so a
captured CUDA graph owns static buffers) and launches on the current stream.
The matching fp32 PyTorch statement of each op lives in ``orinfer_b200.ref.ops_ref``.
"""

from __future__ import annotations

from typing import Optional, Sequence, Tuple, Union

import torch

from . import native
from .native import FMT, check, count_launches, ptr, stream


def _cuda(*tensors):
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise native.KernelError("device op called with a CPU tensor")


def _need(ok: bool, what: str):
    if not ok:
        raise native.KernelError(what)


def embed_w8(ids: torch.Tensor, table_q: torch.Tensor, table_s: torch.Tensor,
             out: Optional[torch.Tensor] = None) -> torch.Tensor:
    _cuda(ids, table_q, table_s)
    rows, hidden = ids.shape[0], table_q.shape[1]
    assert ids.dtype == torch.int32 and table_q.dtype == torch.int8 and table_s.dtype == torch.float16
    if out is None:
        out = torch.empty(rows, hidden, dtype=torch.float16, device=ids.device)
    check(native.lib().orinfer_embed_w8(ptr(ids), ptr(table_q), ptr(table_s), ptr(out), rows,
                                        hidden, table_q.shape[0], stream()), "embed_w8")
    count_launches(1)
    return out


def act_prep(x: Optional[torch.Tensor], resid: Optional[torch.Tensor],
             norm_w: Optional[torch.Tensor], signs: Optional[torch.Tensor], *, eps: float = 1e-6,
             zero_centered: bool = False, swiglu: bool = False, rows: Optional[int] = None,
             q_out: Optional[torch.Tensor] = None, scale_out: Optional[torch.Tensor] = None,
             y_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """residual add (in place into ``resid``) -> RMSNorm -> (SwiGLU) -> rotation -> A8."""
    _cuda(x, resid, norm_w, signs)
    ref = x if x is not None else resid
    rows = ref.shape[0] if rows is None else rows
    k = ref.shape[1] // 2 if swiglu else ref.shape[1]
    if x is not None:
        assert x.dtype == torch.float16 and x.is_contiguous()
    if resid is not None:
        assert resid.dtype == torch.float32 and resid.is_contiguous() and not swiglu
    if q_out is None:
        q_out = torch.empty(ref.shape[0], k, dtype=torch.int8, device=ref.device)
    if scale_out is None:
        scale_out = torch.empty(ref.shape[0], dtype=torch.float32, device=ref.device)
    check(native.lib().orinfer_act_prep(ptr(x), ptr(resid), ptr(norm_w), ptr(signs), ptr(q_out),
                                        ptr(scale_out), ptr(y_out), rows, k, float(eps),
                                        int(zero_centered), int(swiglu), stream()), "act_prep")
    count_launches(1)
    return q_out, scale_out


def act_prep_limited(x: torch.Tensor, signs: Optional[torch.Tensor], row_limit: torch.Tensor, *,
                     swiglu: bool, rows: int, q_out: torch.Tensor,
                     scale_out: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``act_prep`` (no residual / norm) for a launch sized for the worst case: only rows below
    the device-side count ``row_limit[0]`` are processed."""
    _cuda(x, signs, row_limit)
    k = x.shape[1] // 2 if swiglu else x.shape[1]
    assert x.dtype == torch.float16 and x.is_contiguous() and row_limit.dtype == torch.int32
    check(native.lib().orinfer_act_prep_limited(ptr(x), ptr(signs), ptr(q_out), ptr(scale_out),
                                                rows, k, int(swiglu), ptr(row_limit), stream()),
          "act_prep_limited")
    count_launches(1)
    return q_out, scale_out


def rope_table(positions: torch.Tensor, head_dim: int, theta: float,
               cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None,
               rows: Optional[int] = None):
    _cuda(positions)
    assert positions.dtype == torch.int32
    n = positions.shape[0]
    if cos is None:
        cos = torch.empty(n, head_dim // 2, dtype=torch.float32, device=positions.device)
        sin = torch.empty_like(cos)
    check(native.lib().orinfer_rope_table(ptr(positions), ptr(cos), ptr(sin),
                                          n if rows is None else rows, head_dim, float(theta),
                                          stream()), "rope_table")
    count_launches(1)
    return cos, sin


def qk_rope_kv(qkv: torch.Tensor, wq: Optional[torch.Tensor], wk: Optional[torch.Tensor],
               cos: torch.Tensor, sin: torch.Tensor, row_req: torch.Tensor, row_pos: torch.Tensor,
               page_table: torch.Tensor, kcache: torch.Tensor, vcache: torch.Tensor,
               kscale: torch.Tensor, vscale: torch.Tensor, *, qh: int, kvh: int, head_dim: int,
               gated: bool = False, eps: float = 1e-6, zero_centered: bool = False,
               q_out: Optional[torch.Tensor] = None, gate_out: Optional[torch.Tensor] = None,
               rows: Optional[int] = None):
    """Per-head RMSNorm of q/k, NeoX RoPE, and the INT8 group-64 write of K/V into
    the paged cache ``[pages, 128, kvh, D]`` (scales ``[pages, 128, kvh, D/64]``)."""
    _cuda(qkv, cos, row_req, page_table, kcache)
    n = qkv.shape[0]
    assert qkv.dtype == torch.float16 and qkv.is_contiguous()
    assert row_req.dtype == torch.int32 and row_pos.dtype == torch.int32
    assert page_table.dtype == torch.int32 and page_table.dim() == 2
    if q_out is None:
        q_out = torch.empty(n, qh, head_dim, dtype=torch.float16, device=qkv.device)
    if gated and gate_out is None:
        gate_out = torch.empty_like(q_out)
    check(native.lib().orinfer_qk_rope_kv(
        ptr(qkv), ptr(wq), ptr(wk), ptr(cos), ptr(sin), ptr(row_req), ptr(row_pos),
        ptr(page_table), page_table.shape[1], n if rows is None else rows, qh, kvh, head_dim,
        int(gated), float(eps), int(zero_centered), ptr(q_out), ptr(gate_out), ptr(kcache),
        ptr(vcache), ptr(kscale), ptr(vscale), kcache.shape[0], stream()), "qk_rope_kv")
    count_launches(1)
    return q_out, gate_out


def qgemm(a: torch.Tensor, a_scale: torch.Tensor, codes: torch.Tensor, w_scale: torch.Tensor,
          fmt: str, n: int, *, out: Optional[torch.Tensor] = None, out_f32: bool = False,
          rows: Optional[int] = None, path: int = 0) -> torch.Tensor:
    """out[m, n] = (sum_k a[m,k] * W[n,k]) * w_scale[n] * a_scale[m].

    ``path``: 0 auto, 1 SIMT dp4a kernel, 2 tcgen05 tensor-core kernel."""
    _cuda(a, a_scale, codes, w_scale)
    m, k = a.shape
    assert a.dtype == torch.int8 and a.is_contiguous() and a_scale.dtype == torch.float32
    assert w_scale.dtype == torch.float16 and codes.is_contiguous()
    if out is None:
        out = torch.empty(m, n, dtype=torch.float32 if out_f32 else torch.float16, device=a.device)
    else:
        assert out.dtype == (torch.float32 if out_f32 else torch.float16)
    mm = m if rows is None else rows
    check(native.lib().orinfer_qgemm(FMT[fmt], ptr(a), ptr(a_scale), ptr(codes), ptr(w_scale),
                                     ptr(out), mm, n, k, int(out_f32), path, stream()), "qgemm")
    count_launches(native.lib().orinfer_qgemm_launches_fmt(FMT[fmt], mm, n, k, int(out_f32), path))
    return out


PRE_NORM, PRE_PLAIN, PRE_SWIGLU = 1, 2, 3


def qgemv_fused(pre: int, x: Optional[torch.Tensor], resid: Optional[torch.Tensor],
                norm_w: Optional[torch.Tensor], signs: Optional[torch.Tensor], codes: torch.Tensor,
                w_scale: torch.Tensor, fmt: str, n: int, k: int, rows: int, *, eps: float = 1e-6,
                zero_centered: bool = False, out: Optional[torch.Tensor] = None,
                resid_accum: Optional[torch.Tensor] = None, y_out: Optional[torch.Tensor] = None,
                q_out: Optional[torch.Tensor] = None,
                scale_out: Optional[torch.Tensor] = None) -> bool:
    """Projection of at most 8 rows with the row preparation fused into the kernel
    (``pre``: PRE_NORM = resid (+ x) -> RMSNorm -> rotation -> A8; PRE_PLAIN = x -> rotation ->
    A8; PRE_SWIGLU = SwiGLU(x [rows, 2k]) -> rotation -> A8) and, with ``resid_accum``, the
    FP16-rounded result added into an FP32 matrix.  Same bits as ``act_prep`` followed by
    ``qgemm``.  Returns False when the shape does not fit (the caller then runs the separate
    kernels); E8P weights only."""
    if rows > 8 or fmt not in ("q4", "q2"):
        return False
    code = native.lib().orinfer_qgemv_fused(
        FMT[fmt], pre, ptr(x), ptr(resid), ptr(norm_w), ptr(signs), float(eps),
        int(zero_centered), ptr(q_out), ptr(scale_out), ptr(y_out), ptr(codes), ptr(w_scale),
        ptr(out), ptr(resid_accum), rows, n, k, stream())
    if code == -1:
        return False
    check(code, "qgemv_fused")
    count_launches(1)
    return True


def attention_splits(max_kv_len: int, rows: int, kvh: int) -> int:
    """Split the key axis when there are too few (row, kv head) CTAs to fill 148 SMs: about
    three CTAs per SM, at least 64 keys per split.  An ``attention`` entry of the tuning table
    (``tuning/tables.py``) replaces the first rule for its row and context range."""
    if max_kv_len <= 128:
        return 1
    from ..tuning import tables
    tuned = tables.attention_lookup(max_kv_len, rows, kvh)      # a tuned table overrides
    want = tuned if tuned is not None else max(1, (148 * 3) // max(rows * kvh, 1))
    return int(max(1, min(want, (max_kv_len + 63) // 64, 32)))


def attention(q: torch.Tensor, gate: Optional[torch.Tensor], row_req: torch.Tensor,
              row_pos: torch.Tensor, page_table: torch.Tensor, kcache: torch.Tensor,
              vcache: torch.Tensor, kscale: torch.Tensor, vscale: torch.Tensor, *, splits: int = 1,
              scratch: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
              rows: Optional[int] = None, max_kv_len: Optional[int] = None) -> torch.Tensor:
    """Attention of single rows over the paged cache, row r against keys 0..row_pos[r].
    ``max_kv_len``: keys that any row sees at most, where the host knows it (one of two kernels is
    chosen by it; without it, by the width of the page table)."""
    _cuda(q, row_req, page_table, kcache)
    n, qh, d = q.shape
    kvh = kcache.shape[2]
    if out is None:
        out = torch.empty(n, qh * d, dtype=torch.float16, device=q.device)
    if splits > 1 and scratch is None:
        need = native.lib().orinfer_attention_scratch_bytes(n, qh, d, splits)
        scratch = torch.empty(need // 4, dtype=torch.float32, device=q.device)
    check(native.lib().orinfer_attention(
        ptr(q), ptr(gate), ptr(row_req), ptr(row_pos), ptr(page_table), page_table.shape[1],
        ptr(kcache), ptr(vcache), ptr(kscale), ptr(vscale), ptr(out), n if rows is None else rows,
        qh, kvh, d, splits, ptr(scratch), max_kv_len or 0, stream()), "attention")
    count_launches(2 if splits > 1 else 1)
    return out


def attention_prefill(q: torch.Tensor, gate: Optional[torch.Tensor], chunks: torch.Tensor,
                      max_q_len: int, page_table: torch.Tensor, kcache: torch.Tensor,
                      vcache: torch.Tensor, kscale: torch.Tensor, vscale: torch.Tensor, *,
                      out: Optional[torch.Tensor] = None, total_rows: Optional[int] = None,
                      max_kv_len: Optional[int] = None) -> bool:
    """tcgen05 flash attention over prefill chunks.  ``chunks`` is int32 [C, 4] =
    (first row, rows, position of the first row, page-table row).  ``max_kv_len``: keys that any
    chunk reaches at most, where the host knows it (the launch is chosen by it; without it, by
    the width of the page table).  Returns False when the head size is not implemented by the
    tensor-core kernel (nothing was launched)."""
    _cuda(q, chunks, page_table, kcache)
    n, qh, d = q.shape
    assert chunks.dtype == torch.int32 and chunks.dim() == 2 and chunks.shape[1] == 4
    if out is None:
        raise native.KernelError("attention_prefill needs a preallocated output")
    rc = native.lib().orinfer_attention_prefill(
        ptr(q), ptr(gate), ptr(chunks), chunks.shape[0], max_q_len,
        n if total_rows is None else total_rows, ptr(page_table), page_table.shape[1],
        ptr(kcache), ptr(vcache), ptr(kscale), ptr(vscale), ptr(out), qh, kcache.shape[2], d,
        kcache.shape[0], max_kv_len or 0, stream())
    if rc == -4:
        return False
    check(rc, "attention_prefill")
    count_launches(1)
    return True


class SharedPrefix:
    """Plan of a batch of single rows whose contexts share prefixes, for :func:`attention_shared`.
    ``groups``: (first row, rows, keys) each; the page-table rows of a group's rows begin with the
    same pages as far as their first ``keys`` keys lie on them (whole pages, as ``fork_pages`` and
    the prefix cache share them).  Groups do not overlap; rows of no group share nothing.
    ``max_kv_len`` bounds the keys that any row sees while the plan is in use, so that one plan
    serves the steps of a decode loop; rows of unlike lengths are served better by a list with a bound
    for each.  It holds the call's workspace: one stream at a time.  A batch
    whose shared keys are cheaper read again by every row is left to the row kernels, unless
    ``force``."""

    def __init__(self, groups: Sequence[Tuple[int, int, int]], rows: int, *, qh: int, kvh: int,
                 head_dim: int, max_kv_len: Union[int, Sequence[int]], device, force: bool = False):
        bounds = None
        if isinstance(max_kv_len, (list, tuple)):
            bounds = [int(n) for n in max_kv_len]
            _need(len(bounds) == rows and min(bounds, default=0) >= 0, "max_kv_len: one for each row")
            max_kv_len = max(bounds, default=0)
        _need(rows >= 0 and max_kv_len >= 0, "rows and max_kv_len are not negative")
        _need(head_dim in (64, 128, 256), "heads of 64, 128 or 256 channels")
        rep = qh // kvh if kvh > 0 and qh % kvh == 0 else 0
        _need(rep in (1, 2, 4, 8) or (rep == 5 and head_dim == 128),
              f"{qh} query heads on {kvh} KV heads of {head_dim} channels")
        taken = [False] * rows
        for first, n, keys in groups:
            _need(0 <= first and n >= 0 and first + n <= rows, f"group outside the {rows} rows")
            _need(0 <= keys <= max_kv_len, f"{keys} shared keys of {max_kv_len}")
            _need(not any(taken[first:first + n]), "a row is in two groups")
            taken[first:first + n] = [True] * n
        self.rows, self.qh, self.kvh, self.head_dim = rows, qh, kvh, head_dim
        self.device = torch.device(device)
        groups = [(int(f), int(n), int(k)) for f, n, k in groups if n > 0 and k > 0]
        self.longest = max((k for _, _, k in groups), default=0)
        items, info, self.parts = self._split(groups, force)
        put = lambda v: torch.tensor(v, dtype=torch.int32, device=self.device)
        self.items = put(items) if items else None
        self.info = put(info if info else [[0] * 4])
        f32 = lambda n: torch.empty(n, dtype=torch.float32, device=self.device) if n else None
        # (behind the parts the word by which the kernels of a call hand on what lies before them)
        self.part_buffer = (torch.zeros(self.parts * qh * (head_dim + 2) + 1, dtype=torch.float32,
                                        device=self.device) if items else None)
        self.own_keys, self.splits = self._own_parts([i[0] for i in info[:rows]], bounds, max_kv_len)
        self.scratch = f32(rows * qh * self.splits * (head_dim + 2)) if self.splits > 1 else None
        self._args = (ptr(self.items), len(items), ptr(self.info), ptr(self.part_buffer),
                      self.parts, self.splits, ptr(self.scratch), self.own_keys)

    # The row kernels cut every row's own keys into as many parts.  Microseconds of 128 channels of a key
    # in a part, of a CTA, of a record of 128 channels for the merge and of its launch; and what a wave
    # behind the first counts beside a prefix, whose CTAs end one by one.  Over 720 batches of five
    # geometries (1 to 128 rows of 16 to 5000 own keys, with and without a prefix, and with one long row
    # among short ones) the number that this chooses takes 2 % more than the best of ten on average, 45 %
    # at worst (4 rows of 1000 behind 8192).  32 / 8 heads of 128: one row of 16500 keys beside eight of
    # 100 behind 16384 takes 174 us in one part and 61 in sixteen; without a prefix 64 rows of 1000 keys 38
    # in one part and 56 in six, 16 rows of 2000 (three parts are a wave) 21 in three and 26 in four.
    KEY_US, OWN_CTA_US, RECORD_US, MERGE_US, WAVE = 0.0135, 0.0056, 0.0015, 2.2, 0.4

    def _own_parts(self, shared, bounds, max_kv_len):
        """(own keys of the row that has the most, as far as that is known, parts of every row's)."""
        rows, wide = max(1, self.rows), self.head_dim / 128
        if bounds is not None:
            own = [max(0, n - s) for n, s in zip(bounds, shared)]
        else:
            # One number for all: a row behind a shorter prefix, or none, may have as many keys (a long
            # request) or be no longer than those behind the longest (or padding).  Taken between the two,
            # a long row among short ones takes 16 % more than with the best number of parts (without the
            # allowance 92 %), rows that all are short 13 % (with the whole of it 25 %).
            near = max(1, max_kv_len - max(shared, default=0))
            own = [near ** 0.4 * (max_kv_len - s) ** 0.6 for s in shared]
        longest = max(1, round(max(own, default=1)))
        if not self.parts:
            from ..tuning import tables
            if tables.attention_lookup(longest, rows, self.kvh) is not None:
                return longest, attention_splits(longest, rows, self.kvh)
        more = sum(own) / rows * (self.WAVE if self.parts else 1)
        wave = 148 * (2 if self.head_dim > 128 else 3 if self.head_dim > 64 else 4)

        def us(n):
            waves = -(-rows * self.kvh * n // wave)
            each = self.kvh * self.OWN_CTA_US + (n > 1) * self.qh * self.RECORD_US * wide
            return ((longest + (waves - 1) * more) / n * self.KEY_US * wide + n * rows * each
                    + (n > 1) * self.MERGE_US)
        return longest, min(range(1, min(32, max(1, longest // 16)) + 1), key=us)

    # Microseconds of a step of keys (64, or 32 with 256 channels), of a CTA besides its steps, of a megabyte
    # of parts to be written and read, and of a megabyte of keys and values that the row kernels would
    # read again.  Over 1440 batches of eight geometries (2 to 128 rows in one group or four behind 128 to
    # 16384 keys) what this chooses takes 0.5 % more than the better on average, 23 % at worst.  Up to 300
    # own keys, with the prefix shared and without, 32 / 8 heads of 128: 2 rows behind 2048 keys 11.5 and
    # 10.2 us, 8 rows 17.3 and 14.4, 32 rows 19.5 and 30.6, 64 rows 25.1 and 53.2, 64 behind 8192 38.4 and
    # 142; 16 / 8 of 64: 16 rows behind 2048 13.8 and 12.6, 64 behind 8192 19.8 and 84; 16 / 2 of 256: 16
    # rows 23.9 and 17.8, 64 behind 8192 48.8 and 125.
    STEP_US = {64: 0.62, 128: 0.94, 256: 0.81}
    CTA_US, PART_US, AGAIN_US = 4.9, 0.2, 0.167

    def _split(self, groups, force):
        """Which CTAs take which rows and keys: (items, (shared keys, first part, parts, 0) of every
        row, parts in all).  A unit is a tile of rows; the units' keys are cut so that the CTAs fill
        their waves and the longest of them ends soonest."""
        step = native.lib().orinfer_shared_step(self.head_dim)
        per = 128 // (self.qh // self.kvh)             # rows of a tile
        units, info = [], [[0, 0, 0, 0] for _ in range(self.rows)]
        for first, n, keys in groups:
            units += [(at, min(per, first + n - at), -(-keys // step), keys)
                      for at in range(first, first + n, per)]
        if not units:
            return [], info, 0
        columns = self.kvh * max(1, self.head_dim // 128)
        bytes_of = self.qh * self.head_dim * 4e-6      # a part of a row, in megabytes

        def cut(limit):
            """Parts of every unit where no CTA takes more than ``limit`` steps."""
            return [-(-u[2] // limit) for u in units]

        best = None
        waves = -(-len(units) * columns // 148)
        for room in ((waves + i) * 148 // columns for i in range(3)):
            lo, hi = 1, max(u[2] for u in units)       # the fewest steps that fit the waves
            while lo < hi:
                mid = (lo + hi) // 2
                lo, hi = (lo, mid) if sum(cut(mid)) <= room else (mid + 1, hi)
            for limit in {lo, lo * 5 // 4 + 1, lo * 8 // 5 + 1, 2 * lo + 1, 4 * lo + 1}:
                parts = cut(limit)
                mb = sum(p * u[1] for p, u in zip(parts, units)) * bytes_of
                longest = max(-(-u[2] // p) for p, u in zip(parts, units))
                took = -(-sum(parts) * columns // 148)
                us = took * (longest * self.STEP_US[self.head_dim] + self.CTA_US) + mb * self.PART_US
                if best is None or us < best[0]:
                    best = us, parts
        again = sum((n - 1) * keys for _, n, keys in groups) * \
            self.kvh * (2 * self.head_dim + 4 * (self.head_dim // 64)) * 1e-6
        if not force and again * self.AGAIN_US < best[0]:          # cheaper read again than shared
            return [], info, 0
        items, total = [], 0
        for (at, n, steps, keys), parts in zip(units, best[1]):
            for i in range(n):
                info[at + i] = [keys, total + i * parts, parts, 0]
            total += n * parts
            items += [[at, n, steps * p // parts, steps * (p + 1) // parts, keys, p, 0, 0]
                      for p in range(parts)]
        items.sort(key=lambda x: x[2] - x[3])          # the longest first
        return items, info, total


def attention_shared(q: torch.Tensor, gate: Optional[torch.Tensor], row_req: torch.Tensor,
                     row_pos: torch.Tensor, page_table: torch.Tensor, kcache: torch.Tensor,
                     vcache: torch.Tensor, kscale: torch.Tensor, vscale: torch.Tensor,
                     plan: SharedPrefix, *, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`attention` of a batch whose rows share prefixes (``plan``): a shared key is read once
    for all rows of its group.  A row sees keys 0..row_pos[r]; one at position -1 sees none and
    gives zeros (a request that has ended may leave its row so while the plan stays)."""
    n, d, kvh, i32, f16 = plan.rows, plan.head_dim, plan.kvh, torch.int32, torch.float16
    _need(q.shape == (n, plan.qh, d) and q.dtype == f16 and q.is_contiguous(),
          "q: contiguous FP16 [rows, heads, D], as the plan has them")
    _need(row_req.dtype == i32 and row_pos.dtype == i32 and page_table.dtype == i32
          and row_req.numel() >= n and row_pos.numel() >= n and row_req.is_contiguous()
          and row_pos.is_contiguous() and page_table.dim() == 2 and page_table.is_contiguous(),
          "row_req, row_pos: int32 [rows]; page_table: int32 [requests, pages]")
    slots, width = page_table.shape
    pages = kcache.shape[0]
    for t in (kcache, vcache):
        _need(t.shape == (pages, 128, kvh, d) and t.dtype == torch.int8 and t.is_contiguous(),
              "caches: contiguous int8 [pages, 128, kvh, D]")
    for t in (kscale, vscale):
        _need(t.shape == (pages, 128, kvh, d // 64) and t.dtype == f16 and t.is_contiguous(),
              "scales: contiguous FP16 [pages, 128, kvh, D / 64]")
    if gate is not None:
        _need(gate.dtype == f16 and gate.is_contiguous() and gate.numel() == n * plan.qh * d,
              "gate: contiguous FP16, as q")
    if out is None:
        out = torch.empty(n, plan.qh * d, dtype=f16, device=q.device)
    else:
        _need(out.dtype == f16 and out.is_contiguous() and out.numel() == n * plan.qh * d,
              "out: contiguous FP16 [rows, heads * D]")
    where = plan.info.device
    _need(where.type == "cuda", "the plan is not for a GPU")
    for t in (q, gate, row_req, row_pos, page_table, kcache, vcache, kscale, vscale, out):
        _need(t is None or t.device == where, "every tensor on the plan's GPU")
    _need(plan.longest <= width * 128, "more shared keys than the table has pages")
    check(native.lib().orinfer_attention_shared(
        ptr(q), ptr(gate), ptr(row_req), ptr(row_pos), ptr(page_table), slots, width, ptr(kcache),
        ptr(vcache), ptr(kscale), ptr(vscale), ptr(out), n, plan.qh, kvh, d, pages, *plan._args,
        stream()), "attention_shared")
    count_launches((plan.items is not None) + (2 if plan.splits > 1 else 1))
    return out


# ---------------------------------------------------------------- pages of the cache
class CachePages:
    """The tensors of a paged cache (each contiguous [pages, 128, ...], all on one device), as the
    page operators address them: ``KVPool.cache_pages()`` makes one for a model's cache.  It holds
    the tensors, and the calls' workspace: one stream at a time."""

    UNIT = 16384                                   # bytes that a CTA copies at a time

    def __init__(self, tensors: Sequence[torch.Tensor]):
        _need(len(tensors) > 0, "a cache has tensors")
        _cuda(*tensors)
        self.tensors = list(tensors)
        self.pages, self.device = tensors[0].shape[0], tensors[0].device
        sizes, units = [], []
        for i, t in enumerate(tensors):
            _need(t.dim() >= 2 and t.shape[0] == self.pages and t.shape[1] == 128
                  and t.is_contiguous() and t.device == self.device and t.numel() > 0,
                  "cache tensors: contiguous [pages, 128, ...] on one device")
            size = t.element_size() * (t.numel() // (self.pages * 128))
            step = max(16, min(128, self.UNIT // size // 16 * 16))
            sizes.append(size)
            units += [(i, at, min(step, 128 - at)) for at in range(0, 128, step)]
        put = lambda v, dt: torch.tensor(v, dtype=dt, device=self.device)
        self.bases = put([t.data_ptr() for t in tensors], torch.int64)
        self.token_bytes, self.units = put(sizes, torch.int32), put(units, torch.int32)
        self._args = (ptr(self.bases), ptr(self.token_bytes), ptr(self.units), len(units),
                      self.pages)
        self._words = [torch.empty(4 + 3 * (self.pages // 2 + 1), dtype=torch.int32,
                                   device=self.device)]

    def _work(self, words: int) -> int:
        """Address of as many words.  Smaller buffers stay too: a captured graph may hold them."""
        if self._words[-1].numel() < words:
            self._words.append(torch.empty(2 * words, dtype=torch.int32, device=self.device))
        return self._words[-1].data_ptr()


def _tables(ins, out, where):
    """The tensors that a page operator writes, all on GPU ``where``: ``out``, or new ones like its
    inputs (the table first)."""
    table, i32 = ins[0], torch.int32
    for t in ins:
        if t.dtype != i32 or not t.is_contiguous() or t.device != where or not t.is_cuda:
            raise native.KernelError("table, lens, refs: contiguous int32, on one GPU, the cache's")
    if table.dim() != 2 or table.numel() == 0:
        raise native.KernelError("table: [slots, pages of a slot]")
    if out is None:
        return [torch.empty_like(t) for t in ins]
    _need(len(out) == len(ins), "out: a tensor for each input")
    for t, o in zip(ins, out):
        _need(o.shape == t.shape and o.dtype == i32 and o.is_contiguous() and o.device == where,
              "out: tensors like the inputs, on their GPU")
    return out


def _slots(*lists, where):
    n = lists[0].numel()
    for t in lists:
        if (t.dtype != torch.int32 or t.dim() != 1 or t.numel() != n or not t.is_contiguous()
                or not t.is_cuda or t.device != where):
            raise native.KernelError("lists of slots or pages: int32 [n], on the others' GPU")
    return n


def copy_pages(cache: CachePages, source: torch.Tensor, target: torch.Tensor,
               tokens: Optional[torch.Tensor] = None) -> None:
    """Copies pages ``source`` to ``target`` in every tensor of the cache, or their first
    ``tokens`` tokens (int32 [n] each).  No target is a source, and none is named twice."""
    lists = (source, target) if tokens is None else (source, target, tokens)
    n = _slots(*lists, where=cache.device)
    if tokens is None:
        tokens = torch.full_like(source, 128)
    copies = torch.stack((source, target, tokens), dim=1)
    count = torch.full((1,), n, dtype=torch.int32, device=source.device)
    check(native.lib().orinfer_copy_pages(*cache._args, ptr(copies), ptr(count), n, stream()),
          "copy_pages")
    count_launches(1 if n else 0)


def fork_pages(cache: CachePages, table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor,
               parents: torch.Tensor, children: torch.Tensor, *, out=None):
    """Makes slot ``children[i]``, which is empty, a copy of slot ``parents[i]``: whole pages are
    shared, and a page that is not full is copied to a free one, the lowest first in the order of
    the pairs.  ``table`` int32 [slots, pages], ``lens`` tokens per slot, ``refs`` references per
    page (page 0 is nobody's).  Returns (table, lens, refs, status int32 [1]); ``out`` may be the
    inputs.  Status 1: not enough free pages, 2: a pair that cannot be (a slot that does not exist,
    a child that is not empty, named twice or a parent as well, a parent's page that nobody holds);
    nothing is changed then."""
    n = _slots(parents, children, where=cache.device)
    t, l, r = _tables((table, lens, refs), out, cache.device)
    slots, width = table.shape
    if lens.dim() != 1 or lens.numel() != slots or refs.dim() != 1 or refs.numel() != cache.pages:
        raise native.KernelError("lens: [slots], refs: [pages]")
    status = torch.empty(1, dtype=torch.int32, device=cache.device)
    check(native.lib().orinfer_fork_pages(
        *cache._args, table.data_ptr(), t.data_ptr(), lens.data_ptr(), l.data_ptr(),
        refs.data_ptr(), r.data_ptr(), parents.data_ptr(), children.data_ptr(), n, slots, width,
        cache._work(4 + 6 * n + 2 * slots), status.data_ptr(), stream()), "fork_pages")
    count_launches(2)
    return t, l, r, status


def free_pages(table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, slots: torch.Tensor, *,
               out=None):
    """Empties ``slots`` (int32 [n]; one named again is emptied once): every page of their rows
    loses a reference.  Returns (table, lens, refs); ``out`` may be the inputs.  A slot or page that
    does not exist, or a page that nobody holds, is left alone and reported by the status word."""
    n = _slots(slots, where=table.device)
    t, l, r = _tables((table, lens, refs), out, table.device)
    total, width = table.shape
    pages = refs.numel()
    if lens.dim() != 1 or lens.numel() != total or refs.dim() != 1 or pages == 0:
        raise native.KernelError("lens: [slots], refs: [pages]")
    check(native.lib().orinfer_free_pages(
        table.data_ptr(), t.data_ptr(), lens.data_ptr(), l.data_ptr(), refs.data_ptr(),
        r.data_ptr(), slots.data_ptr(), n, total, width, pages, stream()), "free_pages")
    count_launches(2 if t is table or l is lens else 1)
    return t, l, r


def compact_pages(cache: CachePages, table: torch.Tensor, refs: torch.Tensor, *, out=None):
    """Moves the pages that are held to the front: with L of them, the k-th one above page L goes to
    the k-th free page of 1..L.  Returns (table, refs, moved): ``moved`` int32 [pages] says where
    each page has gone.  ``out`` (table, refs) may be the inputs."""
    t, r = _tables((table, refs), out, cache.device)
    if refs.dim() != 1 or refs.numel() != cache.pages:
        raise native.KernelError("refs: [pages]")
    slots, width = table.shape
    moved = torch.empty_like(refs)
    check(native.lib().orinfer_compact_pages(
        *cache._args, table.data_ptr(), t.data_ptr(), refs.data_ptr(), r.data_ptr(),
        moved.data_ptr(), slots, width, cache._work(4 + 3 * (cache.pages // 2 + 1)), stream()),
        "compact_pages")
    count_launches(2)
    return t, r, moved


def argmax(logits: torch.Tensor, out: Optional[torch.Tensor] = None,
           scratch: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
           rows: Optional[int] = None) -> torch.Tensor:
    _cuda(logits)
    m, v = logits.shape
    assert logits.dtype == torch.float32 and logits.is_contiguous()
    parts = native.lib().orinfer_argmax_parts(v)
    if scratch is None:
        scratch = (torch.empty(m * parts, dtype=torch.float32, device=logits.device),
                   torch.empty(m * parts, dtype=torch.int32, device=logits.device))
    if out is None:
        out = torch.empty(m, dtype=torch.int32, device=logits.device)
    check(native.lib().orinfer_argmax(ptr(logits), m if rows is None else rows, v, ptr(scratch[0]),
                                      ptr(scratch[1]), ptr(out), stream()), "argmax")
    count_launches(2)
    return out


# ---------------------------------------------------------------------------- MoE
def router_topk(y: torch.Tensor, router_w: torch.Tensor, experts: int, top_k: int, *,
                renorm: bool = True, rows: Optional[int] = None, ids=None, probs=None,
                gate=None):
    """Router projection + softmax + top-k (ties to the lower expert id).  ``router_w`` has
    ``experts`` rows plus an optional shared-expert gate row.  Returns (ids int32 [M,k],
    probs fp32 [M,k], sigmoid shared gate fp32 [M] or None)."""
    _cuda(y, router_w)
    m, h = y.shape
    has_shared = router_w.shape[0] == experts + 1
    dev = y.device
    ids = torch.empty(m, top_k, dtype=torch.int32, device=dev) if ids is None else ids
    probs = torch.empty(m, top_k, dtype=torch.float32, device=dev) if probs is None else probs
    if has_shared and gate is None:
        gate = torch.empty(m, dtype=torch.float32, device=dev)
    check(native.lib().orinfer_router_topk(ptr(y), ptr(router_w), m if rows is None else rows, h,
                                           experts, int(has_shared), top_k, int(renorm), ptr(ids),
                                           ptr(probs), ptr(gate), stream()), "router_topk")
    count_launches(1)
    return ids, probs, gate


class MoeScratch:
    """Static buffers of one MoE layer evaluation for up to ``max_rows`` tokens."""

    def __init__(self, max_rows: int, top_k: int, experts: int, hidden: int, ffn: int, device):
        s = max_rows * top_k
        e = lambda *shape, dt: torch.empty(*shape, dtype=dt, device=device)
        self.max_tiles = (s + 127) // 128 + experts
        self.ids = e(max_rows, top_k, dt=torch.int32)
        self.probs = e(max_rows, top_k, dt=torch.float32)
        self.gate = e(max_rows, dt=torch.float32)
        self.counts = e(experts, dt=torch.int32)
        self.offsets = e(experts + 1, dt=torch.int32)
        self.tiles = torch.zeros(self.max_tiles, 4, dtype=torch.int32, device=device)
        self.meta = torch.zeros(4, dtype=torch.int32, device=device)
        self.slots = e(s, dt=torch.int32)
        self.q8 = e(s, hidden, dt=torch.int8)
        self.scale = e(s, dt=torch.float32)
        self.gate_up = e(s, 2 * ffn, dt=torch.float16)
        self.q8_mid = e(s, ffn, dt=torch.int8)
        self.scale_mid = e(s, dt=torch.float32)
        self.down = e(s, hidden, dt=torch.float16)


def moe_dispatch(ids: torch.Tensor, q8: Optional[torch.Tensor], scale: Optional[torch.Tensor],
                 experts: int, sc: MoeScratch, rows: int, base_expert: int = 0,
                 local_experts: Optional[int] = None) -> None:
    """Deterministic dispatch metadata + copy of the routed rows into expert-contiguous
    slots (``q8 = None``: numbering only).  With ``local_experts`` only rows routed to experts
    [base_expert, base_expert + local_experts) are dispatched; other slots become -1."""
    top_k = ids.shape[1]
    width = sc.q8.shape[1] if q8 is None else q8.shape[1]
    if local_experts is not None and local_experts != experts:
        check(native.lib().orinfer_moe_dispatch_ep(
            ptr(ids), rows, top_k, base_expert, local_experts, ptr(q8), ptr(scale), width,
            ptr(sc.counts), ptr(sc.offsets), ptr(sc.tiles), ptr(sc.meta), sc.max_tiles,
            ptr(sc.slots), ptr(sc.q8), ptr(sc.scale), stream()), "moe_dispatch_ep")
        count_launches(1 if q8 is None else 2)
        return
    check(native.lib().orinfer_moe_dispatch(
        ptr(ids), rows, top_k, experts, ptr(q8), ptr(scale), width, ptr(sc.counts),
        ptr(sc.offsets), ptr(sc.tiles), ptr(sc.meta), sc.max_tiles, ptr(sc.slots), ptr(sc.q8),
        ptr(sc.scale), stream()), "moe_dispatch")
    count_launches(1 if q8 is None else 2)


def qgemm_grouped(a: torch.Tensor, a_scale: torch.Tensor, codes: torch.Tensor,
                  w_scale: torch.Tensor, fmt: str, n: int, out: torch.Tensor, sc: MoeScratch,
                  total_rows: int, expected_rows: Optional[int] = None) -> torch.Tensor:
    """Grouped projection over the dispatched rows of ``sc``.  ``total_rows`` bounds them; where
    it is far above the rows that this bank will get (its share of the experts, receive buffers
    sized for the worst case) ``expected_rows`` says how many to expect.  The choice of kernels
    follows it, and that a row goes to an expert once."""
    experts = codes.shape[0]
    expected = total_rows if expected_rows is None else max(1, expected_rows)
    tallest = total_rows // sc.ids.shape[1]
    check(native.lib().orinfer_qgemm_grouped(
        FMT[fmt], ptr(a), ptr(a_scale), ptr(codes), ptr(w_scale), ptr(out), total_rows, n,
        a.shape[1], experts, ptr(sc.tiles), ptr(sc.meta), sc.max_tiles, stream(), expected,
        tallest), "qgemm_grouped")
    count_launches(native.lib().orinfer_qgemm_grouped_launches(FMT[fmt], total_rows, experts,
                                                               sc.max_tiles, expected, tallest))
    return out


def moe_combine(expert_out: torch.Tensor, slots: torch.Tensor, probs: torch.Tensor,
                shared_out: Optional[torch.Tensor], gate: Optional[torch.Tensor],
                out: torch.Tensor, rows: int) -> torch.Tensor:
    check(native.lib().orinfer_moe_combine(ptr(expert_out), ptr(slots), ptr(probs), rows,
                                           probs.shape[1], ptr(shared_out), ptr(gate), ptr(out),
                                           out.shape[1], stream()), "moe_combine")
    count_launches(1)
    return out


# ---------------------------------------------------------------- gated delta rule
def small_proj(x: torch.Tensor, w: torch.Tensor, rows: Optional[int] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """fp32 ``x[rows, H] @ w[N, H]^T`` for a narrow fp16 weight (the GDN a/b gates)."""
    _cuda(x, w)
    assert x.dtype == torch.float16 and w.dtype == torch.float16 and x.is_contiguous()
    rows = x.shape[0] if rows is None else rows
    if out is None:
        out = torch.empty(x.shape[0], w.shape[0], dtype=torch.float32, device=x.device)
    check(native.lib().orinfer_small_proj(ptr(x), ptr(w), ptr(out), rows, x.shape[1], w.shape[0],
                                          stream()), "small_proj")
    count_launches(1)
    return out


def gdn_conv(x: torch.Tensor, weight: torch.Tensor, hist: torch.Tensor, row_first: torch.Tensor,
             row_slot: torch.Tensor, row_pos: torch.Tensor, segs: torch.Tensor, n_segs: int,
             rows: int, hk: int, hv: int, head_dim: int,
             out: Optional[torch.Tensor] = None, update_history: bool = True) -> torch.Tensor:
    """Causal conv4 + SiLU + L2(q, k) over the q|k|v channels of ``x`` [rows, >= conv_dim];
    ``hist`` fp16 [slots, 3, conv_dim] is read, then advanced in place per segment (unless
    ``update_history`` is off: a verification pass commits its history later)."""
    _cuda(x, weight, hist, row_first, row_slot, row_pos, segs)
    conv_dim = (2 * hk + hv) * head_dim
    assert x.dtype == torch.float16 and x.stride(1) == 1 and hist.shape[-1] == conv_dim
    assert weight.shape == (conv_dim, 4) and weight.is_contiguous()
    if out is None:
        out = torch.empty(x.shape[0], conv_dim, dtype=torch.float16, device=x.device)
    check(native.lib().orinfer_gdn_conv(ptr(x), x.stride(0), ptr(weight), ptr(hist),
                                        ptr(row_first), ptr(row_slot), ptr(row_pos), ptr(segs),
                                        n_segs, rows,
                                        hk, hv, head_dim, ptr(out), stream(),
                                        int(update_history)), "gdn_conv")
    count_launches(2 if update_history else 1)
    return out


def gdn_scan(qkv: torch.Tensor, ab: torch.Tensor, a_log: torch.Tensor, dt_bias: torch.Tensor,
             segs: torch.Tensor, n_segs: int, row_slot: torch.Tensor, row_pos: torch.Tensor,
             hk: int, hv: int, head_dim: int, state: torch.Tensor,
             out: Optional[torch.Tensor] = None,
             factors: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gated-delta recurrence, row by row for short segments and in chunks of 32 rows for long
    ones; ``state`` fp32 [slots, HV, D, D] updated in place.  With ``factors`` (fp32 [rows, HV,
    2D+1]) the state is left untouched and every step's (decay, k, delta) is recorded for
    :func:`gdn_commit`.  The chunked kernel is launched where a segment may be long: no longer
    than the rows of ``qkv`` less one for every other segment, so ``qkv`` should hold the packet
    alone and every segment a row (results do not depend on it, the choice of kernel does)."""
    _cuda(qkv, ab, a_log, dt_bias, segs, state, row_slot, row_pos)
    assert ab.dtype == torch.float32 and state.dtype == torch.float32 and state.is_contiguous()
    assert a_log.dtype == torch.float32 and dt_bias.dtype == torch.float32
    if out is None:
        out = torch.empty(qkv.shape[0], hv, head_dim, dtype=torch.float32, device=qkv.device)
    longest = qkv.shape[0] - (n_segs - 1)
    check(native.lib().orinfer_gdn_scan(ptr(qkv), ptr(ab), ptr(a_log), ptr(dt_bias), ptr(segs),
                                        n_segs, ptr(row_slot), ptr(row_pos), hk, hv, head_dim,
                                        ptr(state), ptr(out), stream(), ptr(factors), longest),
          "gdn_scan")
    chunked = longest >= (40 if n_segs == 1 else 64) and head_dim == 128 and factors is None
    count_launches(2 if chunked and qkv.data_ptr() % 16 == 0 else 1)
    return out


def gdn_commit(x: torch.Tensor, factors: torch.Tensor, segs: torch.Tensor, n_segs: int,
               accepted: torch.Tensor, row_slot: torch.Tensor, row_pos: torch.Tensor, hk: int,
               hv: int, head_dim: int, hist: torch.Tensor, state: torch.Tensor) -> None:
    """Keeps the first ``accepted[s]`` rows of every segment of a verification pass: advances
    the convolution history by them and replays their recorded state updates."""
    _cuda(x, factors, segs, accepted, row_slot, row_pos, hist, state)
    assert accepted.dtype == torch.int32 and factors.dtype == torch.float32
    check(native.lib().orinfer_gdn_commit(ptr(x), x.stride(0), ptr(factors), ptr(segs), n_segs,
                                          ptr(accepted), ptr(row_slot), ptr(row_pos), hk, hv,
                                          head_dim, ptr(hist), ptr(state), stream()),
          "gdn_commit")
    count_launches(2)


def gdn_gated_norm(o: torch.Tensor, z: torch.Tensor, weight: torch.Tensor, eps: float, rows: int,
                   hv: int, head_dim: int, sigmoid_gate: bool = False,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``rmsnorm(o) * w * silu(z)`` per head; ``z`` may be a column view of the projection."""
    _cuda(o, z, weight)
    assert o.dtype == torch.float32 and z.dtype == torch.float16 and z.stride(1) == 1
    if out is None:
        out = torch.empty(o.shape[0], hv * head_dim, dtype=torch.float16, device=o.device)
    check(native.lib().orinfer_gdn_gated_norm(ptr(o), ptr(z), z.stride(0), ptr(weight), float(eps),
                                              int(sigmoid_gate), rows, hv, head_dim, ptr(out),
                                              stream()), "gdn_gated_norm")
    count_launches(1)
    return out


# ---------------------------------------------------------------- sampling
def sample_topk(logits: torch.Tensor, top_k: torch.Tensor, temperature: torch.Tensor,
                top_p: torch.Tensor, uniform: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Per-row top-k/top-p categorical draw on the device.  ``logits`` fp32 [rows, vocab];
    ``top_k`` int32, ``temperature`` / ``top_p`` / ``uniform`` fp64, all [rows].  Returns
    (tokens int32, flags int32); a set flag means the host law must serve that row."""
    _cuda(logits, top_k, temperature, top_p, uniform)
    assert logits.dtype == torch.float32 and logits.stride(1) == 1 and top_k.dtype == torch.int32
    assert temperature.dtype == torch.float64 and top_p.dtype == torch.float64
    assert uniform.dtype == torch.float64
    rows, vocab = logits.shape
    tok = torch.empty(rows, dtype=torch.int32, device=logits.device)
    flag = torch.zeros(rows, dtype=torch.int32, device=logits.device)
    check(native.lib().orinfer_sample_topk(ptr(logits), rows, vocab, logits.stride(0), ptr(top_k),
                                           ptr(temperature), ptr(top_p), ptr(uniform), ptr(tok),
                                           ptr(flag), stream()), "sample_topk")
    count_launches(1)
    return tok, flag


MASKED = -1e30      # a score that is never drawn: the arg-max and the sampler want finite ones


def process_logits(logits: torch.Tensor, *, history: Optional[torch.Tensor] = None,
                   history_len: Optional[torch.Tensor] = None,
                   repetition: Optional[torch.Tensor] = None,
                   presence: Optional[torch.Tensor] = None,
                   frequency: Optional[torch.Tensor] = None,
                   bias_start: Optional[torch.Tensor] = None,
                   bias_ids: Optional[torch.Tensor] = None,
                   bias_values: Optional[torch.Tensor] = None,
                   mask: Optional[torch.Tensor] = None, mask_rows: Optional[torch.Tensor] = None,
                   masked: float = MASKED, out: Optional[torch.Tensor] = None,
                   flags: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Penalties, biases and grammar masks on ``logits`` fp32 [rows, vocab], by the host law's
    arithmetic (64 bits), rounded once to FP32.

    ``history`` int32 [rows, n] holds ``history_len[r]`` tokens of row r (ids outside the vocabulary
    do not count); ``repetition``, ``presence``, ``frequency`` are fp64 [rows] (1, 0, 0 without
    them).  Row r's biases are ``bias_values`` (fp64) of tokens ``bias_ids`` at bias_start[r] ..
    bias_start[r + 1], the last one of a token counting.  ``mask`` int32 [m, (vocab + 31) / 32]: a
    set bit permits its token; row r is bound by mask ``mask_rows[r]``, by none below 0, by mask r
    without ``mask_rows``.  Tokens that are not permitted get ``masked``.  Returns (out, flags int32
    [rows]): 1 where nothing is permitted, 2 where a logit or a permitted token's score is not
    finite (the host law refuses those rows), the mask does not exist or the row has more than 32768
    biases, else 0.  ``out`` may be ``logits``."""
    i32, f64 = torch.int32, torch.float64
    _cuda(logits)
    where = logits.device
    for t in (history, history_len, repetition, presence, frequency, bias_start, bias_ids,
              bias_values, mask, mask_rows, out, flags):
        if t is not None and t.device != where:
            raise native.KernelError("every tensor on the GPU of the logits")
    if logits.dim() != 2 or logits.dtype != torch.float32 or logits.stride(1) != 1:
        raise native.KernelError("logits: fp32 [rows, vocab], rows in one piece")
    rows, vocab = logits.shape
    _need(vocab > 0, "logits: fp32 [rows, vocab], rows in one piece")
    hist_stride = cap = bias_total = mask_stride = masks = 0

    def of_rows(t, dtype, n=rows):
        return t is not None and t.dtype == dtype and t.shape == (n,) and t.is_contiguous()

    if history is not None:
        if history.dtype != i32 or history.dim() != 2:
            raise native.KernelError("history: int32 [rows, n]")
        (of, cap), (hist_stride, step) = history.shape, history.stride()
        if of != rows or (cap > 1 and step != 1) or not of_rows(history_len, i32):
            raise native.KernelError("history: int32 [rows, n], history_len: int32 [rows]")
    for t in (repetition, presence, frequency):
        if t is not None and (history is None or not of_rows(t, f64)):
            raise native.KernelError("repetition, presence, frequency: fp64 [rows], with a history")
    if bias_start is not None:
        _need(of_rows(bias_start, i32, rows + 1), "bias_start: int32 [rows + 1]")
        _need(bias_ids is not None and bias_values is not None, "bias_ids and bias_values")
        bias_total = bias_ids.numel()
        _need(of_rows(bias_ids, i32, bias_total) and of_rows(bias_values, f64, bias_total),
              "bias_ids: int32, bias_values: fp64, [entries]")
    if mask is not None:
        _need(mask.dtype == i32 and mask.dim() == 2 and mask.stride(1) == 1
              and mask.shape[1] >= (vocab + 31) // 32, "mask: int32 [m, (vocab + 31) / 32]")
        mask_stride, masks = mask.stride(0), mask.shape[0]
        _need(masks >= rows if mask_rows is None else of_rows(mask_rows, i32),
              "mask_rows: int32 [rows], or a mask per row")
    if out is None:
        out = torch.empty(rows, vocab, dtype=torch.float32, device=logits.device)
    else:
        _need(out.shape == logits.shape and out.dtype == torch.float32 and out.stride(1) == 1,
              "out: fp32 [rows, vocab]")
    if flags is None:
        flags = torch.empty(rows, dtype=i32, device=logits.device)
    else:
        _need(of_rows(flags, i32), "flags: int32 [rows]")
    check(native.lib().orinfer_process_logits(
        ptr(logits), logits.stride(0), ptr(history), hist_stride, cap, ptr(history_len),
        ptr(repetition), ptr(presence), ptr(frequency), ptr(bias_start), ptr(bias_ids),
        ptr(bias_values), bias_total, ptr(mask), mask_stride, ptr(mask_rows), masks, masked,
        ptr(out), out.stride(0), ptr(flags), rows, vocab, stream()), "process_logits")
    count_launches(1 if rows else 0)
    return out, flags
