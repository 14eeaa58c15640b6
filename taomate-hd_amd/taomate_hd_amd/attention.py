"""Segment attention: the functional entry to the HIP attention kernels.

``segment_attention`` computes ``softmax(q k^T * scale) v`` for a selection of
token-major query rows over an ordered table of slot segments (no mask), as
``torch.nn.functional.scaled_dot_product_attention(..., is_causal=False)``
does over the concatenated K/V in the reference
(src/taomate_hd/streaming/attention_hook.py:100-115).  ``backend="i8qk"`` runs
the SageAttention-style variant (smooth-K, per-128-block INT8 Q/K, bf16 P.V;
ref attention_hook.py:335-371, inference/sage_value_padding.py:79-97).

Segments may lie in slots held in 8 bits (``KVSlot8``).  A ``"bf16"`` call
whose segments all do, in one format, reads their codes in place
(``tmhd_attn_fwd_kv8``) where it has up to ``KV8_ROWS`` query rows or the batch
is small; for any other call they are expanded to bf16 first, which is exact,
and the call runs as over bf16 slots, whose kernel rounds the scaled Q to bf16.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass, replace
from typing import Any, Sequence

from . import _native
from .profiling import ComponentTimer, maybe_region
from .slots import KV_TILE, KVSlot, KVSlot8, SlotView, expand_views, round_up, vt_columns

BACKENDS = ("bf16", "i8qk")
# 8-bit segments are read in place by calls of up to KV8_ROWS query rows (more than any
# chunk's), and by batches of up to KV8_WORK (query row, token, channel) products.  The
# kernels that read codes multiply Q as it is and the scores by the scale in fp32; the
# bf16 kernel multiplies Q by the scale first and rounds it to bf16 (2^-8 of a score's
# products).  So a row's result does not change its accuracy with the rows beside it: off
# in the 2-norm by 0.0023 to 0.0024 in place and 0.0028 to 0.0030 expanded on N(0, 1) keys,
# and more apart at larger scores.  What that costs, in place / expanded, us, three
# segments, both sides in turn: 14 heads of 128 over 40,788 tokens, e4m3, 98/181 at 256
# rows, 285/338 at 1,024, 553/592 at 2,048, 1,301/1,153 at 4,836, 3,151/2,706 at 12,252,
# int8 1,387/1,156 at 4,836; over 11,232 tokens 136/131 at 1,536, 378/335 at 4,836; over
# 2,717 133/111 at 4,836; over 700 29/42 at 2,560 (3.2e9 products), 129/90 at 12,252
# (15e9); 4 heads over 2,800 19/45 at 2,048; 14 heads of 64 over 40,788 967/787 at 4,836.
# Views that expand_views wrote are attended at the bf16 kernel's time and rounding.
KV8_ROWS = 1 << 14
KV8_WORK = 5 << 29


class QKQuantWorkspace:
    """Grow-only INT8-QK operand storage, keyed by (device, stream).

    Work on one stream is ordered, so a call may reuse the buffers of the
    previous call on that stream without synchronising.  ``nbytes`` reports
    what it holds and ``release`` returns it to the allocator.
    """

    def __init__(self, torch: Any) -> None:
        self._torch = torch
        self._buffers: dict[tuple[Any, ...], dict[str, Any]] = {}

    @property
    def nbytes(self) -> int:
        return sum(int(t.numel()) * t.element_size() for store in self._buffers.values() for t in store.values())

    def release(self) -> None:
        self._buffers.clear()

    def _grow(self, store: dict[str, Any], name: str, numel: int, dtype: Any, device: Any) -> Any:
        buf = store.get(name)
        if buf is None or buf.numel() < numel:
            buf = self._torch.empty(max(numel, 1), dtype=dtype, device=device)
            store[name] = buf
        return buf

    def quant_struct(self, *, heads: int, head_dim: int, lq: int, tokens: Sequence[int], device: Any) -> tuple[Any, dict[str, Any]]:
        structs, views = self.quant_structs(heads=heads, head_dim=head_dim, calls=[(lq, tokens)], device=device,
                                            with_views=True)
        return structs[0], views[0]

    def quant_structs(self, *, heads: int, head_dim: int, calls: Sequence[tuple[int, Sequence[int]]], device: Any,
                      with_views: bool = False) -> tuple[Any, list[dict[str, Any]]]:
        """The operands of ``calls`` (query rows, segment tokens) side by side in
        this stream's buffers: an array of structs, and with ``with_views`` a
        dict of tensors per call."""
        torch = self._torch
        key = (str(device), _native.stream_ptr(torch, device))
        store = self._buffers.setdefault(key, {})
        # 256-byte aligned carve-out offsets inside the int8 and fp32 buffers
        plan, q_total, qs_total, k_total, ks_total = [], 0, 0, 0, 0
        for lq, tokens in calls:
            qcap = round_up(max(lq, 1), _native.QUERY_TILE)
            segs = []
            for t in tokens:
                cap = round_up(t, KV_TILE)
                nblk = round_up(cap, _native.QUANT_BLOCK) // _native.QUANT_BLOCK
                segs.append((cap, nblk, k_total, ks_total))
                k_total += round_up(heads * cap * head_dim, 256)
                ks_total += round_up(heads * nblk, 64)
            plan.append((qcap, q_total, qs_total, segs))
            q_total += heads * qcap * head_dim
            qs_total += round_up(heads * (qcap // _native.QUANT_BLOCK), 64)
        n = len(plan)
        width = heads * head_dim
        q_i8 = self._grow(store, "q_i8", q_total, torch.int8, device)
        q_scale = self._grow(store, "q_scale", qs_total, torch.float32, device)
        k_i8 = self._grow(store, "k_i8", k_total, torch.int8, device)
        k_scale = self._grow(store, "k_scale", ks_total, torch.float32, device)
        k_mean = self._grow(store, "k_mean", n * width, torch.bfloat16, device)
        q_at, qs_at, k_at, ks_at, mean_at = (_native.ptr(t) for t in (q_i8, q_scale, k_i8, k_scale, k_mean))
        structs = (_native.QKQuant * n)()
        views = []
        for i, (qcap, q_off, qs_off, segs) in enumerate(plan):
            qq = structs[i]
            qq.q_i8 = q_at + q_off
            qq.q_scale = qs_at + 4 * qs_off
            qq.q_head_stride = qcap * head_dim
            qq.q_scale_head_stride = qcap // _native.QUANT_BLOCK
            for j, (cap, nblk, k_off, s_off) in enumerate(segs):
                qq.k_i8[j] = k_at + k_off
                qq.k_scale[j] = ks_at + 4 * s_off
                qq.k_head_stride[j] = cap * head_dim
                qq.k_scale_head_stride[j] = nblk
            qq.k_mean = mean_at + 2 * i * width
            if with_views:
                views.append({
                    "q_i8": q_i8[q_off : q_off + heads * qcap * head_dim].view(heads, qcap, head_dim),
                    "q_scale": q_scale[qs_off : qs_off + heads * (qcap // _native.QUANT_BLOCK)].view(heads, -1),
                    "k_mean": k_mean[i * width : (i + 1) * width].view(heads, head_dim),
                    "k_i8": [k_i8[o : o + heads * c * head_dim].view(heads, c, head_dim) for c, _, o, _ in segs],
                    "k_scale": [k_scale[o : o + heads * b].view(heads, b) for _, b, _, o in segs],
                })
        return structs, views


_SPLIT_WORKSPACES: dict[tuple[Any, ...], Any] = {}


def split_workspace(torch: Any, device: Any, head_dim: int) -> Any:
    """Scratch for the key-range split of an attention call's last round.

    One uint8 buffer per (device, stream), grown to what the library asks for
    on that device; calls on one stream are ordered, so they share it.
    """
    need = int(_native.load().tmhd_attn_split_workspace_bytes(int(head_dim)))
    key = (str(device), _native.stream_ptr(torch, device))
    buf = _SPLIT_WORKSPACES.get(key)
    if buf is None or buf.numel() < need:
        buf = torch.empty(max(need, 1), dtype=torch.uint8, device=device)
        _SPLIT_WORKSPACES[key] = buf
    return buf


def split_workspace_bytes() -> int:
    """Bytes held by the split workspaces of every (device, stream) so far."""
    return sum(int(buf.numel()) for buf in _SPLIT_WORKSPACES.values())


def release_split_workspaces() -> None:
    """Return the split workspaces to the allocator (the next call regrows its own)."""
    _SPLIT_WORKSPACES.clear()


def _validate_tokens_major(torch: Any, tensor: Any, name: str) -> None:
    _native.require_device_tensor(torch, tensor, name)
    if tensor.dtype != torch.bfloat16 or tensor.ndim != 3 or tensor.stride(2) != 1:
        raise ValueError(f"{name} must be a [tokens, heads, dim] bf16 view with unit dim stride")


def _row_list(torch: Any, rows: Any, device: Any, limit: int, name: str, checked: bool) -> Any:
    """A row list as a contiguous int32 tensor on ``device`` with entries in
    [0, limit).  The range check reads the list's min / max back (one sync);
    callers whose lists are valid by construction pass ``checked``."""
    if not torch.is_tensor(rows) or rows.device != torch.device(device):
        raise ValueError(f"{name} must be a tensor on the GPU of the rows it indexes")
    if rows.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be an int32 or int64 tensor")
    rows = rows.reshape(-1)
    if not checked and rows.numel():
        # on the list as given: an int64 entry past 2^31 must not wrap into range
        lo, hi = (int(v) for v in torch.aminmax(rows))
        if lo < 0 or hi >= limit:
            raise ValueError(f"{name} entries must lie in [0, {limit})")
    return rows.to(torch.int32).contiguous()


def _key_sums(torch: Any, segments: Sequence[SlotView], stream: int, qq: Any, out: Any, base: int,
              new: dict[tuple[KVSlot, tuple[int, int, int]], Any]) -> None:
    """Where the exact fixed-point key sums of each segment (the smooth-K mean's
    terms) are or go, memoised on its slot per (row0, tokens, stream): a cached
    block's keys are summed once, not on every call.  The slot drops the memo
    whenever it is written.  Sums that this batch takes go to ``new``: the
    caller memoises them once their kernels are queued (a refused batch must
    not leave unfilled ones behind)."""
    for j, view in enumerate(segments):
        slot = view.slot
        key = (int(view.row0), int(view.tokens), int(stream))
        hit = slot.key_sums.get(key)
        if hit is None:
            hit = new.get((slot, key))
        if hit is None:
            hit = new[slot, key] = torch.empty((slot.heads, slot.head_dim), dtype=torch.int64, device=slot.device)
            out[base + j] = _native.ptr(hit)  # summed by this batch
        else:
            qq.k_sum[j] = _native.ptr(hit)


def _coalesce_segments(torch: Any, segments: list[SlotView], limit: int) -> list[SlotView]:
    """One launch takes at most ``limit`` segments; the reference has no such
    bound (it concatenates every part).  With more, the oldest segments are
    copied, in order, into one temporary slot: their keys stay the same keys,
    so the result is the attention over the same set (the INT8-QK key blocks
    then run over the merged rows, as they run over any segment)."""
    n_merge = len(segments) - limit + 1
    head, rest = segments[:n_merge], segments[n_merge:]
    keys, values = [], []
    for view in head:
        slot, r0, n = view.slot, int(view.row0), int(view.tokens)
        keys.append(slot.k[:, r0 : r0 + n, :].permute(1, 0, 2))
        cols = r0 + vt_columns(torch, n, slot.device)  # r0 is a multiple of 64: whole 16-token groups
        values.append(slot.vt.index_select(2, cols).permute(2, 0, 1))
    key, value = torch.cat(keys, 0).contiguous(), torch.cat(values, 0).contiguous()
    first = head[0].slot
    merged = KVSlot(torch, heads=first.heads, head_dim=first.head_dim, capacity=int(key.shape[0]), device=first.device)
    merged.pack(key, value)
    return [merged.view(), *rest]


def segment_attention(
    torch: Any,
    query: Any,
    segments: Sequence[SlotView],
    *,
    scale: float,
    backend: str = "bf16",
    q_rows: Any | None = None,
    q_row0: int = 0,
    lq: int | None = None,
    out: Any | None = None,
    o_rows: Any | None = None,
    o_row0: int = 0,
    workspace: QKQuantWorkspace | None = None,
    split: bool = True,
    return_quant: bool = False,
    timer: ComponentTimer | None = None,
    rows_checked: bool = False,
) -> Any:
    """Attention of the selected query rows over ``segments`` (no mask; bf16 slots are
    read in place, 8-bit ones by the rule at ``KV8_ROWS``).

    Query row ``i`` is ``query[q_rows[i]]`` (or ``query[q_row0 + i]``); its
    output goes to ``out[o_rows[i]]`` (or ``out[o_row0 + i]``).  Without
    ``out`` a new ``[lq, H, D]`` tensor is returned.  ``split`` lets the
    library run the items of a partial last round as key ranges (merged on
    the same stream); results agree with the unsplit run to fp32 rounding.
    Row lists are device tensors; their range is checked (one sync) unless
    ``rows_checked`` says the caller built them in range.
    """
    outs, views = segment_attention_batch(
        torch,
        [AttentionCall(query, segments, q_rows=q_rows, q_row0=q_row0, lq=lq, out=out, o_rows=o_rows, o_row0=o_row0,
                       rows_checked=rows_checked)],
        scale=scale, backend=backend, workspace=workspace, split=split, return_quant=return_quant, timer=timer,
    )
    return (outs[0], views[0]) if return_quant and backend == "i8qk" else outs[0]


@dataclass
class AttentionCall:
    """One call of ``segment_attention_batch``: the arguments of
    ``segment_attention`` that belong to a single call."""

    query: Any
    segments: Sequence[SlotView]
    q_rows: Any | None = None
    q_row0: int = 0
    lq: int | None = None
    out: Any | None = None
    o_rows: Any | None = None
    o_row0: int = 0
    rows_checked: bool = False


def _call_args(torch: Any, call: AttentionCall, args: Any, scale: float, keep: list[Any],
               new: Any | None = None) -> tuple[Any, list[SlotView]]:
    """Check one call and fill its C arguments (``AttnArgs``, or ``KV8Call`` for
    8-bit segments read in place); returns its output (``new``, if it fits a
    call without one) and segments."""
    query, out, q_rows, o_rows, lq = call.query, call.out, call.q_rows, call.o_rows, call.lq
    q_row0, o_row0 = int(call.q_row0), int(call.o_row0)
    _validate_tokens_major(torch, query, "query")
    rows_in, heads, head_dim = query.shape
    device = query.device
    if q_rows is not None:
        q_rows = _row_list(torch, q_rows, device, rows_in, "q_rows", call.rows_checked)
        keep.append(q_rows)
        n = int(q_rows.numel())
        if lq is not None and int(lq) != n:
            raise ValueError("lq differs from the query row list")
        lq = n
    elif lq is None:
        lq = rows_in - q_row0
    lq = int(lq)
    if out is None:
        out = new
        if out is None or out.shape != (lq, heads, head_dim):
            out = torch.empty((lq, heads, head_dim), dtype=torch.bfloat16, device=device)
        o_rows, o_row0 = None, 0
    else:
        _validate_tokens_major(torch, out, "out")
        if tuple(out.shape[1:]) != (heads, head_dim):
            raise ValueError("out heads/dim differ from query")
        if o_rows is not None:
            o_rows = _row_list(torch, o_rows, out.device, int(out.shape[0]), "o_rows", call.rows_checked)
            keep.append(o_rows)
            if int(o_rows.numel()) != lq:
                raise ValueError("output row list length differs from the query rows")
        elif not (0 <= o_row0 and o_row0 + lq <= int(out.shape[0])):
            raise ValueError(f"output rows [{o_row0}, {o_row0 + lq}) outside out ({int(out.shape[0])} rows)")
    if q_rows is None and not (0 <= q_row0 and q_row0 + lq <= rows_in):
        raise ValueError(f"query rows [{q_row0}, {q_row0 + lq}) outside query ({rows_in} rows)")
    segments = [s for s in call.segments if s.tokens > 0]
    if not segments:
        raise ValueError("attention needs at least one key/value token")
    for s in segments:
        slot = s.slot
        if slot.heads != heads or slot.head_dim != head_dim or slot.device != device:
            raise ValueError("segment heads/dim/device differ from the query")
    if len(segments) > _native.MAX_SEGMENTS:
        segments = _coalesce_segments(torch, segments, _native.MAX_SEGMENTS)
        keep.append(segments)
    args.q = query.data_ptr()
    args.q_token_stride, args.q_head_stride, _ = query.stride()
    args.q_rows = _native.ptr(q_rows) if q_rows is not None and lq else None
    args.q_row0 = q_row0
    args.lq = lq
    args.o = out.data_ptr()
    args.o_token_stride, args.o_head_stride, _ = out.stride()
    args.o_rows = _native.ptr(o_rows) if o_rows is not None and lq else None
    args.o_row0 = o_row0
    args.n_segments = len(segments)
    table = args.seg
    if isinstance(args, _native.KV8Call):
        for i, s in enumerate(segments):
            s.slot.fill_segment8(table, i, s.row0, s.tokens)
        return out, segments
    args.heads = heads
    args.head_dim = head_dim
    args.scale = scale
    for i, s in enumerate(segments):
        s.fill_segment(table[i])
    return out, segments


def _in_place_format(call: AttentionCall) -> str | None:
    """The format of the call's segments, if all are 8-bit ones of one format and no more than one launch takes."""
    fmt, count = None, 0
    for s in call.segments:
        if s.tokens > 0:
            if not isinstance(s.slot, KVSlot8) or fmt not in (None, s.slot.format):
                return None
            fmt, count = s.slot.format, count + 1
    return fmt if count <= _native.MAX_SEGMENTS else None


def _call_rows(call: AttentionCall) -> int:
    """A call's query rows (its arguments are checked later)."""
    if call.q_rows is not None:
        return int(call.q_rows.numel()) if hasattr(call.q_rows, "numel") else 0
    return int(call.query.shape[0] - call.q_row0 if call.lq is None else call.lq)


def _in_place_formats(calls: Sequence[AttentionCall]) -> list[str | None]:
    """For each ``"bf16"`` call the format of the segments that it reads in place, None where they are expanded."""
    rows = [_call_rows(call) for call in calls]
    work = sum(n * sum(s.tokens * s.slot.heads * s.slot.head_dim for s in call.segments) for n, call in zip(rows, calls))
    return [_in_place_format(call) if n <= KV8_ROWS or work <= KV8_WORK else None for n, call in zip(rows, calls)]


def _new_outputs(calls: Sequence[AttentionCall]) -> dict[int, Any]:
    """The outputs of calls that bring none, side by side in one allocation (1.7 us of host time each)."""
    at = [i for i, call in enumerate(calls) if call.out is None]
    rows = [_call_rows(calls[i]) for i in at]
    if len(at) < 2 or min(rows) < 0:
        return {}
    query = calls[at[0]].query
    return dict(zip(at, query.new_empty((sum(rows), *query.shape[1:])).split(rows)))


def _attend_in_place(torch: Any, calls: Sequence[AttentionCall], scale: float, timer: ComponentTimer | None) -> list[Any]:
    """Calls over 8-bit segments of one format, in one launch (per 16 calls and 24 segments)."""
    keep: list[Any] = []
    n = len(calls)
    args = (_native.KV8Call * n)()
    new = _new_outputs(calls)
    outs = [_call_args(torch, call, args[i], scale, keep, new.get(i))[0] for i, call in enumerate(calls)]
    query = calls[0].query
    device, shape = query.device, query.shape[1:]
    for call, out in zip(calls, outs):
        if call.query.shape[1:] != shape or call.query.device != device or out.device != device:
            raise ValueError("the queries and outputs of a batch must share heads, head_dim and one GPU")
    heads, head_dim = shape
    lib = _native.load()
    with _native.device_of(torch, query), maybe_region(timer, "attention"):
        need = lib.tmhd_attn_kv8_workspace_bytes(args, n, heads, head_dim)
        # from the caching allocator each time: ordered with its stream, and a captured graph's own
        ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        status = lib.tmhd_attn_fwd_kv8(args, n, heads, head_dim, scale, ws.data_ptr() if need else None, need,
                                       _native.stream_ptr(torch, device))
    _native.check(status, "tmhd_attn_fwd_kv8")
    return outs


def _attend_8bit(torch: Any, calls: list[AttentionCall], **options: Any) -> tuple[list[Any], list[dict[str, Any]]]:
    """``segment_attention_batch`` of calls some of whose segments are held in 8 bits."""
    scale, timer = float(options["scale"]), options["timer"]
    formats = _in_place_formats(calls) if options["backend"] == "bf16" else [None] * len(calls)
    kinds = set(formats)
    if len(kinds) == 1 and None not in kinds:
        return _attend_in_place(torch, calls, scale, timer), []
    outs: list[Any] = [None] * len(calls)
    rest = [i for i, f in enumerate(formats) if f is None]
    segments = [[s for s in calls[i].segments if s.tokens > 0] for i in rest]
    for i, segs in zip(rest, segments):
        _validate_tokens_major(torch, calls[i].query, "query")
        for s in segs:
            if (s.slot.heads, s.slot.head_dim, s.slot.device) != (*calls[i].query.shape[1:], calls[i].query.device):
                raise ValueError("segment heads/dim/device differ from the query")
    for fmt in sorted(kinds - {None}):
        at = [i for i, f in enumerate(formats) if f == fmt]
        for i, out in zip(at, _attend_in_place(torch, [calls[i] for i in at], scale, timer)):
            outs[i] = out
    with maybe_region(timer, "expand"):
        expanded = iter(expand_views(torch, [s for segs in segments for s in segs]))
    calls = [replace(calls[i], segments=[next(expanded) for _ in segs]) for i, segs in zip(rest, segments)]
    got, views = segment_attention_batch(torch, calls, **options) if calls else ([], [])
    for i, out in zip(rest, got):
        outs[i] = out
    return outs, views


def segment_attention_batch(
    torch: Any,
    calls: Sequence[AttentionCall],
    *,
    scale: float,
    backend: str = "bf16",
    workspace: QKQuantWorkspace | None = None,
    split: bool = True,
    return_quant: bool = False,
    timer: ComponentTimer | None = None,
) -> tuple[list[Any], list[dict[str, Any]]]:
    """Independent ``segment_attention`` calls in one kernel launch (see
    ``tmhd_attn_fwd_bf16_batch``): a hook call's condition, media and padding
    attention, or a packed sequence's documents, none of which alone fills the
    GPU's last round of workgroups.  The calls share heads, head_dim and the
    query and output strides; their output rows must not overlap.  Returns
    their outputs (those of a batch over 8-bit segments may lie in one
    allocation), and with ``return_quant`` the INT8-QK operand views."""
    if backend not in BACKENDS:
        raise ValueError(f"unknown attention backend {backend!r}")
    if not calls:
        return [], []
    if any(isinstance(s.slot, KVSlot8) for call in calls for s in call.segments if s.tokens > 0):
        return _attend_8bit(torch, list(calls), scale=scale, backend=backend, workspace=workspace, split=split,
                            return_quant=return_quant, timer=timer)
    keep: list[Any] = []  # row lists and merged slots, alive until the launches are queued
    args = (_native.AttnArgs * len(calls))()
    outs, segments = [], []
    for i, call in enumerate(calls):
        out, segs = _call_args(torch, call, args[i], float(scale), keep)
        outs.append(out)
        segments.append(segs)
    device, heads, head_dim = calls[0].query.device, args[0].heads, args[0].head_dim
    if any(call.query.device != device or out.device != device for call, out in zip(calls, outs)):
        raise ValueError("the queries and outputs of a batch must share one GPU")
    lib = _native.load()
    stream = _native.stream_ptr(torch, device)
    if split and any(a.lq for a in args):
        ws = split_workspace(torch, device, head_dim)
        args[0].split_workspace = _native.ptr(ws)
        args[0].split_workspace_bytes = int(ws.numel())
    if backend == "bf16":
        with maybe_region(timer, "attention"):
            status = lib.tmhd_attn_fwd_bf16_batch(args, len(calls), stream)
        _native.check(status, "tmhd_attn_fwd_bf16")
        return outs, []
    if workspace is None:
        workspace = QKQuantWorkspace(torch)
    quants, views = workspace.quant_structs(
        heads=heads, head_dim=head_dim, calls=[(a.lq, [s.tokens for s in segs]) for a, segs in zip(args, segments)],
        device=device, with_views=return_quant,
    )
    with maybe_region(timer, "qk_quant"):
        sums = (ctypes.c_void_p * (_native.MAX_SEGMENTS * len(calls)))()
        new_sums: dict[tuple[KVSlot, tuple[int, int, int]], Any] = {}
        for i, segs in enumerate(segments):
            _key_sums(torch, segs, stream, quants[i], sums, i * _native.MAX_SEGMENTS, new_sums)
        status = lib.tmhd_qk_smooth_quant_batch(args, quants, sums, len(calls), stream)
    _native.check(status, "tmhd_qk_smooth_quant")
    for (slot, key), value in new_sums.items():
        slot.key_sums[key] = value
    with maybe_region(timer, "attention"):
        status = lib.tmhd_attn_fwd_i8qk_batch(args, quants, len(calls), stream)
    _native.check(status, "tmhd_attn_fwd_i8qk")
    return outs, views
