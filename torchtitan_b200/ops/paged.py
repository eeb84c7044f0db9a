"""Paged key / value cache: the plan of a step, the write of its new rows, and attention over the pages.

A layer's cache is a pair of pools ``k_pages, v_pages [num_pages, Hkv, page_size, D]``; the pages of a sequence are listed
in its row (*slot*) of ``block_table [slots, columns]``.  A step feeds a flat stream of new rows: ``new[b]`` rows of the
sequence in slot ``slots[b]``, which has ``cached[b]`` tokens in its pages already.  ``page_plan`` extends the table rows
by the pages handed out and computes, on the device, where every row goes; ``write_kv`` stores the rows' keys and values;
``attention`` lets every row attend to its sequence's tokens up to and including itself.

Sequences that share a prefix (their tables begin with the same pages) may be passed as groups of neighbours: the prefix
is then attended to once for all rows of the group and merged with what follows it.

Lengths and tables live on the device and are checked there: an entry that is out of range is skipped (its row gets slot
-1) and 16 is set in ``torch.ops.tb200.status`` (32: a bounded wait inside an attention kernel ran out);
``torch.ops.tb200.take_status(48)`` reads and clears these two behind the current stream's work.  On CPU tensors the plain
forms of ``ops/reference.py`` run, which raise instead.
"""

from __future__ import annotations

from dataclasses import dataclass, field

import torch

from . import ext, reference as ref
from .functional import _count, _library_fallback, settings

__all__ = ["PagePlan", "page_plan", "write_kv", "attention", "supported"]

PAGE_SIZES = (16, 32, 64, 128, 256)
HEAD_DIMS = (64, 128, 256)
MAX_SEQS = 4096                  # of one step on CUDA


@dataclass(eq=False)
class PagePlan:
    """Where the rows of one step go; made once per step and used by every layer."""

    row_start: torch.Tensor      # [B + 1] int32: first row of each sequence in the flat stream
    positions: torch.Tensor      # [R] int64: position of each row in its sequence (0 behind the last sequence)
    slot_map: torch.Tensor       # [R] int64: page * page_size + offset of each row, -1 = nowhere
    cached: torch.Tensor
    slots: torch.Tensor
    block_table: torch.Tensor
    page_size: int
    num_pages: int
    total_rows: int
    heads: tuple[int, int] | None = None                                 # (query, key heads) of the attention work lists
    groups: int = 0
    max_rows: int = 0                                                    # of one sequence or group
    shared_rows: int = 0                                                 # of all groups that share a prefix
    work: dict[int, torch.Tensor] = field(default_factory=dict)          # by window


def supported(q: torch.Tensor, k_pages: torch.Tensor) -> bool:
    """Shapes of the attention kernels: bf16, head dimension 64, 128 or 256."""
    return q.is_cuda and q.dtype == torch.bfloat16 and k_pages.dtype == torch.bfloat16 and q.shape[-1] in HEAD_DIMS


def page_plan(cached: torch.Tensor, new: torch.Tensor, block_table: torch.Tensor, slots: torch.Tensor, pages: torch.Tensor,
              page_size: int, total_rows: int, *, num_pages: int, mapped: torch.Tensor | None = None,
              group_start: torch.Tensor | None = None, group_prefix: torch.Tensor | None = None, n_heads: int | None = None,
              n_kv_heads: int | None = None, windows: tuple[int, ...] = (0,), max_rows: int | None = None,
              shared_rows: int | None = None) -> PagePlan:
    """Plan of one step over ``B = len(slots)`` sequences (all index tensors int32 on one device).

    ``pages`` are the ids handed out, in the order of the sequences: sequence ``b`` takes as many as it needs for
    ``cached[b] + new[b]`` tokens beyond the ``mapped[b]`` columns of its table row that are filled already (default:
    those that hold its cached tokens).  ``total_rows`` is the length of the flat stream, at least ``sum(new)``.

    With ``n_heads`` and ``n_kv_heads`` the plan also holds what ``attention`` needs for layers of these heads, for each of
    ``windows`` (0 = no window).  ``group_start [groups + 1]`` and ``group_prefix [groups]`` declare that the sequences
    ``group_start[g] .. group_start[g + 1]`` share their first ``group_prefix[g]`` tokens: their table rows begin with the
    same pages.  Offsets that are not in order are flagged and nothing is shared.  ``max_rows``: an upper bound of the new
    rows of one sequence or group, if the caller knows one.  ``shared_rows``: the same of the rows of all groups with a prefix
    and two or more sequences with rows: attention needs ``2 shared_rows Hq (D + 2)`` floats of workspace for them, and a
    group beyond the bound is attended to without sharing.  Both cost speed only when they are wrong."""
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_plan: page_size must be one of {PAGE_SIZES}, got {page_size}")
    if (group_start is None) != (group_prefix is None) or (group_start is not None and group_start.numel() != group_prefix.numel() + 1):
        raise ValueError("page_plan: group_start [groups + 1] and group_prefix [groups] come together")
    if any(int(w or 0) < 0 for w in windows):
        raise ValueError(f"page_plan: windows {tuple(windows)} (0 = none)")
    args = (cached, new, block_table, slots, pages, mapped, int(page_size), int(total_rows), int(num_pages))
    if block_table.is_cuda:
        _count()
        row_start, positions, slot_map = ext.require().page_plan(*args)
    else:
        if group_start is not None:
            at = group_start.tolist()
            if sorted(at) != at or at[0] < 0 or at[-1] > cached.numel():
                raise ValueError(f"page_plan: the groups' offsets {at} are not in order")
        row_start, positions, slot_map = ref.page_plan(*args)
    plan = PagePlan(row_start, positions, slot_map, cached, slots, block_table, int(page_size), int(num_pages), int(total_rows))
    if n_heads is not None:
        if not n_kv_heads or n_heads % n_kv_heads:
            raise ValueError(f"page_plan: {n_heads} query heads on {n_kv_heads} key heads")
        plan.heads, plan.groups = (int(n_heads), int(n_kv_heads)), 0 if group_prefix is None else group_prefix.numel()
        plan.max_rows = int(total_rows) if max_rows is None else min(int(max_rows), int(total_rows))
        plan.shared_rows = 0 if not plan.groups else int(total_rows) if shared_rows is None else max(0, min(int(shared_rows), int(total_rows)))
        if block_table.is_cuda:
            for w in dict.fromkeys(int(w or 0) for w in windows):
                _count()
                plan.work[w] = ext.require().paged_work(cached, row_start, slots, group_start, group_prefix, block_table.shape[1],
                                                        int(page_size), int(total_rows), *plan.heads, w, plan.shared_rows)
    return plan


def _vectors(t: torch.Tensor) -> torch.Tensor:
    """``t`` itself when its last dimension is contiguous and every vector starts on 16 bytes, else a copy."""
    s0, s1, s2 = t.stride()
    n = 16 // t.element_size()
    if s2 == 1 and s0 > 0 and s1 > 0 and s0 % n == 0 and s1 % n == 0 and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def write_kv(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, slot_map: torch.Tensor) -> None:
    """Store ``k, v [R, Hkv, D]`` at their slots of the pools; rows with slot -1 are left out.  The slots of a call differ:
    of two rows for one slot, parts of either may be left."""
    if k_pages.is_cuda:
        _count()
        ext.require().paged_write(_vectors(k), _vectors(v), k_pages, v_pages, slot_map)
    else:
        ref.paged_write(k, v, k_pages, v_pages, slot_map)


def attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, plan: PagePlan, scale: float, *, window: int = 0,
              sinks: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``q [R, Hq, D]`` -> ``[R, Hq, D]``: row ``r`` at position ``p`` of its sequence attends to the tokens
    ``max(0, p - window + 1) .. p`` (``window = 0``: all up to ``p``).  ``sinks [Hq]``: one logit per head in the softmax
    denominator.  A row that sees no key, or only scores of minus infinity, is zero; a NaN among its scores makes it NaN.  Values
    that are not finite reach the rows that see them, in their own columns, and no others (rows that have a NaN are computed
    again, key by key, which takes longer).  Probabilities are rounded to the values' bf16 before the product, scores, sums
    and partial outputs are fp32.  Rows behind the last sequence are zero, or left as they are when ``out`` is given.  For inference: no gradient flows back.  Not batch-invariant on CUDA (the other sequences' lengths
    decide where a sequence's keys are cut into partial sums), so batch-invariant mode refuses it."""
    R, hq, D = q.shape
    n_pages, hkv, ps, dk = k_pages.shape
    if not 1.2e-38 <= scale <= 2.3e38:               # times log2(e) a normal fp32 number: masked scores stay minus infinity
        raise ValueError(f"paged attention: the scale must be positive and finite in 32 bits, got {scale}")
    if window < 0:
        raise ValueError(f"paged attention: window {window} (0 = none)")
    if R != plan.total_rows:
        raise ValueError(f"paged attention: {R} query rows, the plan has {plan.total_rows}")
    if v_pages.shape != k_pages.shape or n_pages != plan.num_pages or ps != plan.page_size:
        raise ValueError(f"paged attention: pools {tuple(k_pages.shape)} / {tuple(v_pages.shape)} do not fit a plan of "
                         f"{plan.num_pages} pages of {plan.page_size}")
    if hq % hkv or D != dk:
        raise ValueError(f"paged attention: queries {tuple(q.shape)} against pools {tuple(k_pages.shape)}")
    if not supported(q, k_pages):
        if q.is_cuda:
            _library_fallback(f"paged attention on {q.dtype} with head dimension {q.shape[-1]}")
        o = ref.paged_attention(q, k_pages, v_pages, plan.block_table, plan.slots, plan.cached, plan.row_start, float(scale),
                                int(window), sinks)
        if out is None:
            return o
        n = int(plan.row_start[-1])
        out[:n] = o[:n]
        return out
    if settings.strict_native:
        raise RuntimeError("paged attention cuts a sequence's keys by the lengths of all sequences of the step, which is not "
                           "batch-invariant (debug.batch_invariant is on)")
    work = plan.work.get(int(window))
    if plan.heads != (hq, hkv) or work is None:
        raise ValueError(f"paged attention: {hq} / {hkv} heads with window {window}, the plan was made for {plan.heads} and "
                         f"windows {tuple(plan.work)}")
    _count(3 if D <= 128 and plan.max_rows * (hq // hkv) > 16 else 2)
    if sinks is not None and (sinks.dtype != torch.float32 or not sinks.is_contiguous()):
        sinks = sinks.float().contiguous()
    dst = q.new_empty((R, hq, D)) if out is None else out
    ext.require().paged_attention(_vectors(q), k_pages, v_pages, plan.block_table, plan.slots, plan.cached, plan.row_start, work, plan.groups,
                                  plan.max_rows, plan.shared_rows, float(scale), int(window), sinks, dst, out is None)
    return dst
