"""Grouped-query attention with a fused QKV projection.

The projection weight ``wqkv`` stacks ``[q heads | k heads | v heads]``; it is
saved to checkpoints as ``qkv_linear.wq/wk/wv`` (parity with the key layout of
torchtitan/models/common/attention.py:722-867).  RoPE is applied in place on the
packed projection output, q/k/v are strided views of it, and the pre-norm is
folded into the projection's autograd function.

Masking.  ``AttentionContext`` carries what the inner kernel needs: document ids
derived from ``positions`` (a document starts where ``positions == 0``), an
optional sliding window, and for context parallelism the global token indices of
this rank's queries.  (Reference: mask mods in attention.py:429-565, CP
placements in decoder_sharding.py:263-302.)
"""

from __future__ import annotations

import math
from dataclasses import dataclass, field

import torch
import torch.nn as nn

from torchtitan_b200.ops import functional as OF
from torchtitan_b200.parallel import tp_ops

from .layers import Linear, RMSNorm, RoPE, TPContext
from .module import InitSpec, Module, set_init

__all__ = ["GQAttention", "AttentionContext", "KVCache", "BatchedKVCache", "PagedKVCache", "cached_attention",
           "fused_qk_norm_rope", "build_attention_context"]


@dataclass
class AttentionContext:
    doc_ids: torch.Tensor | None = None  # [T_local] int32, None = single document
    q_pos: torch.Tensor | None = None  # global token index of local rows (CP)
    cp: object | None = None  # parallel.context_parallel.CPContext
    max_doc_len: int | None = None
    kv_first: torch.Tensor | None = None  # [T_local] int32: index of the first token of each token's document
    rope_positions: torch.Tensor | None = None  # [3, T_local] multimodal rotary positions (overrides ``positions``)
    kv_cache: "KVCache | BatchedKVCache | PagedKVCache | None" = None  # incremental decoding: keys / values of earlier tokens, per attention layer


class KVCache:
    """Keys and values of the tokens seen so far, one pair of buffers per attention layer (incremental decoding
    with the training model itself; the reference's generator keeps its cache inside vLLM,
    torchtitan/experiments/rl).  Buffers grow in chunks; ``update`` appends the new rows and returns views of
    everything cached."""

    def __init__(self, chunk: int = 256):
        self.chunk = chunk
        self._k: dict[int, torch.Tensor] = {}
        self._v: dict[int, torch.Tensor] = {}
        self._len: dict[int, int] = {}

    def length(self, layer) -> int:
        return self._len.get(id(layer), 0)

    def state(self, layer) -> dict:
        """Free-form per-layer state for layers that are not attention (a recurrent layer's state matrix and the
        tail of its convolution inputs)."""
        if not hasattr(self, "_state"):
            self._state = {}
        return self._state.setdefault(id(layer), {})

    def update(self, layer, k: torch.Tensor, v: torch.Tensor):
        key = id(layer)
        n0, n = self._len.get(key, 0), k.shape[0]
        if key not in self._k or self._k[key].shape[0] < n0 + n:
            cap = (n0 + n + self.chunk - 1) // self.chunk * self.chunk
            nk = k.new_empty((cap,) + tuple(k.shape[1:]))
            nv = v.new_empty((cap,) + tuple(v.shape[1:]))
            if n0:
                nk[:n0], nv[:n0] = self._k[key][:n0], self._v[key][:n0]
            self._k[key], self._v[key] = nk, nv
        self._k[key][n0:n0 + n] = k
        self._v[key][n0:n0 + n] = v
        self._len[key] = n0 + n
        return self._k[key][:n0 + n], self._v[key][:n0 + n]


class BatchedKVCache:
    """Several sequences decoded in one forward pass: the flat token stream holds ``rows[i]`` consecutive rows of
    sequence ``i`` (its whole prompt at prefill, one row while decoding), each attending to its own ``caches[i]``.
    The projections and feed-forward layers run once over all rows; only the attention core is per sequence."""

    def __init__(self, caches: "list[KVCache]", rows: list[int]):
        assert len(caches) == len(rows)
        self.caches, self.rows = caches, rows


class PagedKVCache:
    """Keys and values of many sequences in pages of one pool per attention layer (``ops.paged``).

    Every sequence has a *slot* (a row of the block table on the device); which pages it owns is known on the host as
    well, where pages are handed out and taken back.  ``add`` admits a sequence, ``begin_step`` plans one forward pass
    over some rows of some sequences (one H2D copy of their lengths and new page ids, the tables are built on the device),
    ``attend`` is what a layer calls, ``end_step`` advances the lengths, ``release`` ends a sequence.

    Sequences whose prompts have the same whole pages (all but the last token at most) share those pages: the later ones start
    behind them, and attention reads them once for all rows of the group.  The whole pages have to be equal in number, too:
    a prompt that only begins with another's pages computes all of its own.  Whole requests are reserved at ``add`` (prompt
    and the tokens to come), so a sequence in flight never runs out of pages."""

    def __init__(self, heads: tuple[int, int], windows: tuple[int, ...], *, tokens: int, max_seqs: int, max_length: int,
                 page_size: int = 64, device, share_prefixes: bool = True):
        from torchtitan_b200.ops.paged import MAX_SEQS, PAGE_SIZES

        if page_size not in PAGE_SIZES:
            raise ValueError(f"page size {page_size} (have {PAGE_SIZES})")
        if max_seqs > MAX_SEQS:
            raise ValueError(f"a paged cache for {max_seqs} sequences: a step takes at most {MAX_SEQS}")
        if tokens <= 0 or max_seqs <= 0 or max_length <= 0:
            raise ValueError("a paged cache needs tokens, sequences and a maximum length")
        self.heads, self.windows, self.page_size, self.device = heads, windows, page_size, torch.device(device)
        self.num_pages = -(-tokens // page_size)
        self.max_length, self.share_prefixes = max_length, share_prefixes
        cols = min(-(-max_length // page_size), self.num_pages)
        self.block_table = torch.full((max_seqs, cols), -1, dtype=torch.int32, device=self.device)
        self.pools: dict[int, tuple[torch.Tensor, torch.Tensor]] = {}
        self.plan = None
        self.reset()

    @classmethod
    def for_model(cls, model, **kw) -> "PagedKVCache":
        """A cache for a decoder whose attention layers are all grouped-query layers with the same head counts."""
        from .mla import MLAttention

        layers = [m for m in model.modules() if isinstance(m, GQAttention)]
        heads = {(m.n_heads, m.n_kv_heads) for m in layers}
        if any(isinstance(m, MLAttention) for m in model.modules()) or len(heads) != 1:
            raise ValueError("the paged cache covers decoders whose attention layers are grouped-query layers of one shape "
                             f"(found {sorted(heads)}); use the contiguous cache")
        recurrent = any(type(b.attention).__name__ == "GatedDeltaNet" for b in model.modules() if hasattr(b, "attention"))
        kw["share_prefixes"] = kw.get("share_prefixes", True) and not recurrent     # a recurrent state is not in the pages
        return cls(heads.pop(), tuple(sorted({int(m.window or 0) for m in layers})), **kw)

    # -- sequences ---------------------------------------------------------
    def reset(self) -> None:
        self._free = list(range(self.num_pages - 1, -1, -1))
        self._slots = list(range(self.block_table.shape[0] - 1, -1, -1))
        self._refs = [0] * self.num_pages
        self._pages: dict[int, list[int]] = {}       # slot -> pages, prefix first
        self._length: dict[int, int] = {}            # slot -> tokens in the pages
        self._mapped: dict[int, int] = {}            # slot -> columns of its table row that are filled
        self._group: dict[int, tuple] = {}           # slot -> (group number, prefix tokens)
        self._index: dict[tuple, tuple[int, int]] = {}   # leading tokens -> (group number, a live slot that holds them)
        self._states: dict[int, KVCache] = {}
        self._groups_made = 0
        self._step: tuple[list[int], list[int]] | None = None

    def _prefix_key(self, prompt) -> tuple:
        return tuple(prompt[:(len(prompt) - 1) // self.page_size * self.page_size]) if self.share_prefixes else ()

    def shared_tokens(self, prompt) -> int:
        """Leading tokens of ``prompt`` that ``add`` would take from a sequence in flight: its whole pages or nothing."""
        key = self._prefix_key(prompt)
        return len(key) if key in self._index else 0

    def pages_needed(self, prompt, new_tokens: int) -> int:
        """Pages that ``add`` would take from the pool."""
        total = -(-min(len(prompt) + new_tokens, self.max_length) // self.page_size)
        return total - self.shared_tokens(prompt) // self.page_size

    def can_add(self, prompt, new_tokens: int) -> bool:
        return bool(self._slots) and self.pages_needed(prompt, new_tokens) <= len(self._free)

    def add(self, prompt, new_tokens: int) -> tuple[int, int]:
        """Admit a sequence of ``prompt`` and up to ``new_tokens`` more; returns ``(slot, tokens already cached)``."""
        if len(prompt) > self.max_length or not prompt:
            raise ValueError(f"a prompt of {len(prompt)} tokens in a cache for up to {self.max_length}")
        if not self.can_add(prompt, new_tokens):
            raise RuntimeError(f"the paged cache is full: {len(self._free)} pages and {len(self._slots)} sequences left")
        need = self.pages_needed(prompt, new_tokens)
        key = self._prefix_key(prompt)
        slot = self._slots.pop()
        pages, cached = [], 0
        if key in self._index:
            group, other = self._index[key]
            cached = len(key)
            pages = self._pages[other][:cached // self.page_size]
            self._group[slot] = (group, cached)
        elif key:
            self._groups_made += 1
            self._index[key] = (self._groups_made, slot)
            self._group[slot] = (self._groups_made, len(key))
        pages = pages + [self._free.pop() for _ in range(need)]
        for i in pages:
            self._refs[i] += 1
        self._pages[slot], self._length[slot], self._mapped[slot] = pages, cached, 0
        self._states[slot] = KVCache()
        return slot, cached

    def release(self, slot: int) -> None:
        for i in self._pages.pop(slot):
            self._refs[i] -= 1
            if self._refs[i] == 0:
                self._free.append(i)
        del self._length[slot], self._mapped[slot], self._states[slot]
        group = self._group.pop(slot, None)
        for key, (g, holder) in list(self._index.items()):
            if holder == slot:                       # hand the entry to another member, if there is one
                other = next((s for s, m in self._group.items() if m == group), None)
                if other is None:
                    del self._index[key]
                else:
                    self._index[key] = (g, other)
        self._slots.append(slot)

    def forget_prefixes(self) -> None:
        """New sequences do not join those in flight any more (the weights changed)."""
        self._index.clear()

    def group_of(self, slot: int) -> int:
        """Sort key that brings the members of a group together."""
        return self._group.get(slot, (0, 0))[0]

    # -- one forward pass --------------------------------------------------
    def begin_step(self, slots: list[int], rows: list[int]) -> None:
        """The flat token stream will hold ``rows[i]`` consecutive rows of ``slots[i]``; members of a group are neighbours."""
        from torchtitan_b200.ops import paged

        ps = self.page_size
        cached, mapped, pages = [], [], []
        for s, n in zip(slots, rows):
            c, m = self._length[s], self._mapped[s]
            end = -(-(c + n) // ps)
            if c + n > self.max_length or end > len(self._pages[s]):
                raise RuntimeError(f"slot {s}: {c} + {n} tokens are more than were reserved")
            cached.append(c)
            mapped.append(m)
            pages += self._pages[s][m:end]
            self._mapped[s] = max(m, end)
        start, prefix, shared_rows, longest = self._prefix_groups(slots, rows, cached)
        B, NG = len(slots), len(start)
        flat = torch.tensor(cached + rows + slots + mapped + pages + start + [B] * (NG > 0) + prefix, dtype=torch.int32)
        if self.device.type == "cuda":
            flat = flat.pin_memory().to(self.device, non_blocking=True)
        c, r, s, m, pg, st, pr = flat.split([B, B, B, B, len(pages), NG + (NG > 0), NG])
        groups = dict(group_start=st, group_prefix=pr, shared_rows=shared_rows) if NG else {}
        self.plan = paged.page_plan(c, r, self.block_table, s, pg, ps, sum(rows), num_pages=self.num_pages, mapped=m,
                                    n_heads=self.heads[0], n_kv_heads=self.heads[1], windows=self.windows, max_rows=longest,
                                    **groups)
        self._step = (list(slots), list(rows))

    def _prefix_groups(self, slots: list[int], rows: list[int], cached: list[int]) -> tuple[list[int], list[int], int, int]:
        """``(first sequences, prefixes, rows that share, most rows of one group or sequence)`` of a step.  Only neighbours
        that have a common prefix in their pages already are a group with one; everything between two of them is one
        group without a prefix, and a step in which nothing is shared has no groups."""
        start, prefix, shared_rows, longest, i = [], [], 0, max(rows, default=0), 0
        while i < len(slots):
            g, j = self._group.get(slots[i]), i + 1
            while j < len(slots) and g is not None and self._group.get(slots[j]) == g:
                j += 1
            live = [k for k in range(i, j) if rows[k] > 0]
            if g is not None and len(live) > 1 and min(cached[k] for k in live) > 0:
                start.append(i)
                prefix.append(g[1])
                shared_rows += sum(rows[i:j])
                longest = max(longest, sum(rows[i:j]))
            elif not prefix or prefix[-1]:
                start.append(i)
                prefix.append(0)
            i = j
        return (start, prefix, shared_rows, longest) if shared_rows else ([], [], 0, longest)

    def end_step(self) -> None:
        for s, n in zip(*self._step):
            self._length[s] += n
        self._step = None

    @property
    def caches(self) -> "list[KVCache]":             # free-form per-layer state of the step's sequences (recurrent layers)
        return [self._states[s] for s in self._step[0]]

    @property
    def rows(self) -> list[int]:
        return self._step[1]

    def attend(self, layer, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, *, window: int = 0,
               sinks: torch.Tensor | None = None) -> torch.Tensor:
        from torchtitan_b200.ops import paged

        pool = self.pools.get(id(layer))
        if pool is None:
            shape = (self.num_pages, k.shape[1], self.page_size, k.shape[2])
            pool = self.pools[id(layer)] = (k.new_zeros(shape), k.new_zeros(shape))
        paged.write_kv(k.detach(), v.detach(), *pool, self.plan.slot_map)
        return paged.attention(q.detach(), *pool, self.plan, scale, window=window, sinks=sinks)


def cached_attention(layer, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kv_cache, scale: float, *, window: int = 0,
                     sinks: torch.Tensor | None = None) -> torch.Tensor:
    """Append the new keys / values to ``layer``'s cache and attend the new queries to everything cached (causal
    among the new rows).  ``kv_cache``: one ``KVCache`` (all rows belong to one sequence), a ``BatchedKVCache``
    (consecutive row blocks of several sequences) or a ``PagedKVCache`` (the same in one launch over all pages).  Query / key and value head dimensions may differ (latent
    attention); shapes the flash kernels do not cover run the PyTorch block attention."""
    from torchtitan_b200.ops import flash as FL

    def attend(cache, q_, k_, v_):
        kc, vc = cache.update(layer, k_.detach(), v_.detach())
        o_, lse = FL.block_fwd(q_.contiguous(), kc, vc, scale, causal=True, causal_offset=kc.shape[0] - q_.shape[0],
                               window=window)
        if sinks is not None:
            o_ = (o_.float() * torch.sigmoid(lse - sinks.float()[:, None]).t()[..., None]).to(q_.dtype)
        return o_

    if isinstance(kv_cache, PagedKVCache):
        return kv_cache.attend(layer, q, k, v, scale, window=window, sinks=sinks)
    if not isinstance(kv_cache, BatchedKVCache):
        return attend(kv_cache, q, k, v)
    parts, r0 = [], 0
    for cache, n in zip(kv_cache.caches, kv_cache.rows):
        parts.append(attend(cache, q[r0:r0 + n], k[r0:r0 + n], v[r0:r0 + n]))
        r0 += n
    assert r0 == q.shape[0], f"BatchedKVCache rows cover {r0} of {q.shape[0]} tokens"
    return torch.cat(parts)


def build_attention_context(positions: torch.Tensor, *, assume_single_document: bool = False,
                            cp=None, q_pos: torch.Tensor | None = None) -> AttentionContext:
    """Derive document ids from ``positions`` (no host sync)."""
    if assume_single_document:
        return AttentionContext(None, q_pos, cp)
    starts = (positions == 0).to(torch.int32)
    doc_ids = torch.cumsum(starts, dim=0, dtype=torch.int32)
    # a document starts where positions == 0, so token i's document starts at (global index of i) - positions[i];
    # under context parallelism the rows are sharded and ``q_pos`` holds their global indices
    index = q_pos if (cp is not None and q_pos is not None) else torch.arange(positions.shape[0], device=positions.device)
    kv_first = (index - positions).to(torch.int32)
    return AttentionContext(doc_ids, q_pos, cp, kv_first=kv_first)


def fused_qk_norm_rope(qkv: torch.Tensor, hq: int, hkv: int, q_norm, k_norm, rope: RoPE | None, positions: torch.Tensor,
                       q_scale: float = 1.0):
    """``(q, k, v)`` of a packed projection output ``[T, Hq + 2 Hkv, D]`` from the one-pass norm + rotation, or None when
    ``kernels.qk_norm_rope`` does not ask for it or the layer has no per-head norms or shapes that it does not cover."""
    if OF.settings.qk_norm_rope != "fused" or q_norm is None or q_norm.eps != k_norm.eps:
        return None
    gain = getattr(q_norm, "gain_center", 0.0)
    plain = all(type(n) is RMSNorm or hasattr(n, "gain_center") for n in (q_norm, k_norm))
    D = qkv.shape[2]
    rot = rope.cache.shape[1] if rope is not None else 0
    if not plain or gain != getattr(k_norm, "gain_center", 0.0) or D % 8 or D > 256 or rot > D or (
            rot % (8 if rope is not None and rope.interleaved else 16)):
        return None
    return OF.qk_norm_rope(qkv, hq, hkv, q_norm.weight, k_norm.weight, None if rope is None else rope.cache, positions,
                           rope is not None and rope.interleaved, eps=q_norm.eps, gain_center=gain, q_scale=q_scale,
                           axes=None if rope is None else rope.axes_for(positions))


class GQAttention(Module):
    @dataclass(kw_only=True, slots=True)
    class Config(Module.Config):
        dim: int = 0
        n_heads: int = 0
        n_kv_heads: int | None = None
        head_dim: int | None = None
        wqkv: Linear.Config = field(default_factory=Linear.Config)
        wo: Linear.Config = field(default_factory=Linear.Config)
        qk_norm: RMSNorm.Config | None = None
        rope: RoPE.Config = field(default_factory=RoPE.Config)
        sliding_window: int | None = None
        use_sinks: bool = False
        softmax_scale: float | None = None

    def __init__(self, config: "GQAttention.Config", **_):
        super().__init__(config)
        c = config
        self.n_heads = c.n_heads
        self.n_kv_heads = c.n_kv_heads or c.n_heads
        self.head_dim = c.head_dim or c.dim // c.n_heads
        hd = self.head_dim
        c.wqkv.in_features = c.dim
        c.wqkv.out_features = (self.n_heads + 2 * self.n_kv_heads) * hd
        c.wqkv.row_blocks = [self.n_heads * hd, self.n_kv_heads * hd, self.n_kv_heads * hd]
        c.wo.in_features, c.wo.out_features = self.n_heads * hd, c.dim
        self.wqkv = c.wqkv.build()
        self.wo = c.wo.build()
        self.q_norm = self.k_norm = None
        if c.qk_norm is not None:
            c.qk_norm.dim = hd
            self.q_norm = c.qk_norm.build()
            self.k_norm = c.qk_norm.build()
        c.rope.dim = c.rope.dim or hd
        self.rope = c.rope.build()
        self.scale = c.softmax_scale if c.softmax_scale is not None else 1.0 / math.sqrt(hd)
        self.window = c.sliding_window
        self.sinks = None
        if c.use_sinks:
            self.sinks = nn.Parameter(torch.empty(self.n_heads))
            set_init(self.sinks, InitSpec(kind="trunc_normal", std=0.02))
        self.tp: TPContext | None = None

    # -- parallel ----------------------------------------------------------
    def shard_(self, tp: TPContext) -> None:
        if self.n_kv_heads % tp.size:
            raise ValueError(f"n_kv_heads={self.n_kv_heads} must divide by tp={tp.size}")
        self.wqkv.shard_("colwise", tp)
        self.wo.shard_("rowwise", tp)
        if self.sinks is not None:
            n = self.n_heads // tp.size
            s = nn.Parameter(torch.empty(n, device=self.sinks.device, dtype=self.sinks.dtype))
            s._tp_slices = (0, [(tp.rank * n, (tp.rank + 1) * n)], (self.n_heads,))
            set_init(s, self.sinks._init_spec)
            self.sinks = s
        self.n_heads //= tp.size
        self.n_kv_heads //= tp.size
        self.tp = tp

    def checkpoint_slices(self):
        hd = self.head_dim
        q, kv = self.n_heads * hd, self.n_kv_heads * hd
        out = {
            "wqkv.weight": [
                ("qkv_linear.wq.weight", 0, q),
                ("qkv_linear.wk.weight", q, q + kv),
                ("qkv_linear.wv.weight", q + kv, q + 2 * kv),
            ]
        }
        if self.wqkv.bias is not None:
            out["wqkv.bias"] = [
                ("qkv_linear.wq.bias", 0, q),
                ("qkv_linear.wk.bias", q, q + kv),
                ("qkv_linear.wv.bias", q + kv, q + 2 * kv),
            ]
        return out

    # -- forward -----------------------------------------------------------
    def forward(self, x: torch.Tensor, positions: torch.Tensor, ctx: AttentionContext | None = None,
                norm: RMSNorm | None = None) -> torch.Tensor:
        tp = self.tp
        hd, hq, hkv = self.head_dim, self.n_heads, self.n_kv_heads
        fused = False
        if tp is not None:
            if norm is not None:
                x = norm(x)
            fused = tp.fused_ok(x, self.wqkv, self.wo) and tp.fused.supported(x.shape[0] * tp.size, x.shape[1], hq * hd)
            if fused:
                from torchtitan_b200.parallel import tp_fused

                qkv = tp_fused.all_gather_linear(x, self.wqkv.weight, tp.fused)
            else:
                x = tp_ops.all_gather_rows(x, tp) if tp.sequence_parallel else tp_ops.copy_to_tp(x, tp)
                qkv = self.wqkv(x)
        elif type(norm) is RMSNorm and type(self.wqkv) is Linear and norm.weight is not None and self.wqkv.bias is None:
            qkv = OF.norm_linear(x, norm.weight, self.wqkv.weight, norm.eps)
        else:
            qkv = self.wqkv(norm(x) if norm is not None else x)
        T = qkv.shape[0]
        if ctx is not None and ctx.rope_positions is not None:
            positions = ctx.rope_positions          # multimodal: [3, T] temporal / height / width
        if self.q_norm is None:
            qkv = self.rope.apply_packed_(qkv, positions, hq + hkv, hd)
        qkv = qkv.view(T, hq + 2 * hkv, hd)
        fused_qk = fused_qk_norm_rope(qkv, hq, hkv, self.q_norm, self.k_norm, self.rope, positions)
        if fused_qk is not None:
            q, k, v = fused_qk
        elif self.q_norm is not None:
            # QK-norm normalises each head vector before RoPE (Qwen3).
            qn = self.q_norm(qkv[:, :hq])
            kn = self.k_norm(qkv[:, hq:hq + hkv])
            q = self.rope(qn, positions)
            k = self.rope(kn, positions)
            v = qkv[:, hq + hkv:]
        else:
            q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        ctx = ctx or AttentionContext()
        if ctx.kv_cache is not None:
            # incremental decoding (no autograd): the new queries attend to everything cached plus themselves
            o = cached_attention(self, q, k, v, ctx.kv_cache, self.scale, window=int(self.window or 0), sinks=self.sinks)
        elif ctx.cp is not None:
            from torchtitan_b200.parallel.context_parallel import cp_attention

            o = cp_attention(q, k, v, ctx, scale=self.scale, window=self.window, sinks=self.sinks)
        elif self.q_norm is None and self.window is None and self.sinks is None:
            o = OF.attention_packed(qkv, hq, hkv, self.scale, doc_ids=ctx.doc_ids, kv_first=ctx.kv_first)
        else:
            o = OF.attention(q, k, v, scale=self.scale, causal=True, doc_ids=ctx.doc_ids, window=self.window,
                             sinks=self.sinks, kv_first=ctx.kv_first)
        if fused:
            from torchtitan_b200.parallel import tp_fused

            return tp_fused.linear_reduce_scatter(o.reshape(T, hq * hd), self.wo.weight, tp.fused)
        y = self.wo(o.reshape(T, hq * hd))
        if tp is not None:
            return tp_ops.reduce_scatter_rows(y, tp) if tp.sequence_parallel else tp_ops.all_reduce(y, tp)
        return y
