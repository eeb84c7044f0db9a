"""Paged key / value cache: step plans, page writes and attention over pages against plain 64-bit forms.

Tolerance of attention.  With ``A = sum_j p_j |v_j|`` (p normalised): the probabilities are rounded to bf16 before they meet
the values (half a step, 2^-8 of each: at most 2^-8 A in the sum), the result is rounded once (2^-8 |o|); scores are fp32
sums of at most 256 products and of the probabilities' exponent, whose error moves a probability by less than 2^-12 for the
scores of these tests (|s| < 64: 256 * 2^-24 * 64 = 2^-10 in the worst case of one-sided rounding, a sixteenth of that in
any order a kernel sums in).  Together 2^-8 |o| + (2^-8 + 2^-12) A."""

import math

import pytest
import torch

from torchtitan_b200.ops import ext, paged, reference as ref

DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]


def _i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


class _Step:
    """A step over groups of sequences: ``groups = [(prefix tokens, [(cached behind the prefix, new rows), ...]), ...]``.
    Page contents that no sequence owns are NaN, so that nothing outside a sequence can go unnoticed."""

    def __init__(self, groups, *, hq, hkv, D, ps, device, pad=0, seed=0, extra_cols=0, interleaved_pools=False, dtype=torch.bfloat16):
        g = torch.Generator().manual_seed(seed)
        self.hq, self.hkv, self.D, self.ps = hq, hkv, D, ps
        self.cached, self.new, start, prefix, own = [], [], [0], [], []
        for p, members in groups:
            for c, n in members:
                self.cached.append(p + c)
                self.new.append(n)
                own.append(len(start) - 1)
            start.append(len(self.cached))
            prefix.append(p)
        B = len(self.cached)
        total = [c + n for c, n in zip(self.cached, self.new)]
        W = max([1] + [-(-t // ps) for t in total]) + extra_cols
        S = B + 3
        slots = torch.randperm(S, generator=g)[:B].tolist()
        n_pages = sum(-(-t // ps) for t in total) + 4
        order = torch.randperm(n_pages, generator=g).tolist()
        table = torch.full((S, W), -7, dtype=torch.int32)
        self.pages_of = []
        for b in range(B):
            first = start[own[b]]
            common = prefix[own[b]] // ps if b != first else 0
            mine = self.pages_of[first][:common] if common else []
            while len(mine) < -(-total[b] // ps):
                mine = mine + [order.pop()]
            self.pages_of.append(mine)
            table[slots[b], :len(mine)] = torch.tensor(mine, dtype=torch.int32)
        R = sum(self.new) + pad
        kv = torch.full((2, n_pages, hkv, ps, D), float("nan"))
        for b in range(B):
            for j in range(-(-total[b] // ps)):
                n = min(ps, total[b] - j * ps)
                fresh = torch.isnan(kv[:, self.pages_of[b][j], :, :n, :1])
                kv[:, self.pages_of[b][j], :, :n] = torch.where(fresh, torch.randn(2, hkv, n, D, generator=g), kv[:, self.pages_of[b][j], :, :n])
        kv = kv.to(dtype)
        if interleaved_pools:                      # keys and values of a page side by side: strided pools
            pool = kv.transpose(0, 1).contiguous().to(device)
            self.kp, self.vp = pool[:, 0], pool[:, 1]
        else:
            self.kp, self.vp = kv[0].contiguous().to(device), kv[1].contiguous().to(device)
        self.q = torch.randn(R, hq, D, generator=g).to(dtype).to(device)
        self.sink = torch.randn(hq, generator=g).to(device)
        self.table, self.slots, self.n_pages, self.R, self.device = table.to(device), slots, n_pages, R, device
        self.start, self.prefix = start, prefix
        self.scale = 1 / math.sqrt(D)

    def plan(self, windows=(0,), grouped=True, **kw):
        d = self.device
        held = _i32([len(p) for p in self.pages_of], d)
        g = dict(group_start=_i32(self.start, d), group_prefix=_i32(self.prefix, d)) if grouped else {}
        return paged.page_plan(_i32(self.cached, d), _i32(self.new, d), self.table, _i32(self.slots, d), _i32([], d), self.ps, self.R,
                               num_pages=self.n_pages, mapped=held, n_heads=self.hq, n_kv_heads=self.hkv, windows=windows, **g, **kw)

    def oracle(self, window=0, sinks=None):
        """(o, sum_j p_j |v_j|) in 64 bits."""
        out = torch.zeros(self.q.shape, dtype=torch.float64)
        size = torch.zeros_like(out)
        kp, vp, q, r = self.kp.cpu().double(), self.vp.cpu().double(), self.q.cpu().double(), 0
        G = self.hq // self.hkv
        for b in range(len(self.new)):
            for i in range(self.new[b]):
                pos = self.cached[b] + i
                lo = max(0, pos - window + 1) if window else 0
                j = torch.arange(lo, pos + 1)
                page = torch.tensor(self.pages_of[b])[j // self.ps]
                k, v = kp[page, :, j % self.ps], vp[page, :, j % self.ps]
                s = torch.einsum("hgd,jhd->hgj", q[r].view(self.hkv, G, self.D), k) * self.scale
                if sinks is not None:
                    s = torch.cat([s, sinks.cpu().double().view(self.hkv, G, 1)], -1)
                p = torch.softmax(s, -1)[..., :len(j)]
                out[r] = torch.einsum("hgj,jhd->hgd", p, v).reshape(self.hq, self.D)
                size[r] = torch.einsum("hgj,jhd->hgd", p, v.abs()).reshape(self.hq, self.D)
                r += 1
        return out, size

    def check(self, got, window=0, sinks=None):
        want, size = self.oracle(window, sinks)
        n = sum(self.new)
        err = (got[:n].cpu().double() - want[:n]).abs()
        tol = 2 ** -8 * want[:n].abs() + (2 ** -8 + 2 ** -12) * size[:n]
        assert (err <= tol).all(), (float((err - tol).max()), float(err.max()))


# ------------------------------------------------------------------------------------------------------------------ plans
def _plan_oracle(cached, new, table, slots, pages, mapped, ps, R):
    """Token by token."""
    table = table.clone()
    it = iter(pages)
    starts, pos, slot = [0], [], []
    for c, n, s, m in zip(cached, new, slots, mapped):
        for col in range(m, -(-(c + n) // ps)):
            table[s, col] = next(it)
        for j in range(c, c + n):
            pos.append(j)
            slot.append(int(table[s, j // ps]) * ps + j % ps)
        starts.append(starts[-1] + n)
    pad = R - len(pos)
    return table, starts, pos + [0] * pad, slot + [-1] * pad


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("B,ps,top,most,pad", [(1, 16, 1, 1, 0), (1, 64, 500, 1, 3), (7, 16, 100, 40, 0), (300, 32, 2000, 3, 1), (64, 256, 90, 700, 5)])
def test_plan(device, B, ps, top, most, pad):
    g = torch.Generator().manual_seed(B)
    cached = torch.randint(0, top, (B,), generator=g).tolist()
    new = torch.randint(0, most + 1, (B,), generator=g).tolist()
    new[0] = max(new[0], 1)
    cached[0] = cached[0] // ps * ps                                   # a length that ends with its page
    W = max(-(-(c + n) // ps) for c, n in zip(cached, new)) + 1
    slots = torch.randperm(B + 4, generator=g)[:B].tolist()
    held = [-(-c // ps) for c in cached]
    mapped = list(held)
    mapped[-1] = 0                                                     # a new sequence whose prefix pages come along
    n_pages = sum(held) + sum(-(-(c + n) // ps) - m for c, n, m in zip(cached, new, mapped)) + 2
    order = torch.randperm(n_pages, generator=g).tolist()
    table = torch.full((B + 4, W), -9, dtype=torch.int32)
    for s, h in zip(slots[:-1], held[:-1]):
        table[s, :h] = torch.tensor([order.pop() for _ in range(h)], dtype=torch.int32)
    need = sum(max(0, -(-(c + n) // ps) - m) for c, n, m in zip(cached, new, mapped))
    pages = [order.pop() for _ in range(need)]
    R = sum(new) + pad
    want = _plan_oracle(cached, new, table, slots, pages, mapped, ps, R)
    t = table.to(device)
    p = paged.page_plan(_i32(cached, device), _i32(new, device), t, _i32(slots, device), _i32(pages, device), ps, R,
                        num_pages=n_pages, mapped=_i32(mapped, device))
    assert torch.equal(t.cpu(), want[0])
    assert p.row_start.tolist() == want[1] and p.positions.tolist() == want[2] and p.slot_map.tolist() == want[3]
    if device == "cuda":
        assert ext.require().status(True) == 0


@pytest.mark.parametrize("device", DEVICES)
def test_plan_without_sequences_or_rows(device):
    table = torch.full((2, 3), 5, dtype=torch.int32, device=device)
    e = _i32([], device)
    p = paged.page_plan(e, e, table, e, e, 16, 4, num_pages=9)
    assert p.row_start.tolist() == [0] and p.slot_map.tolist() == [-1] * 4 and p.positions.tolist() == [0] * 4
    p = paged.page_plan(_i32([20], device), _i32([0], device), table, _i32([1], device), e, 16, 0, num_pages=9)
    assert p.row_start.tolist() == [0, 0] and p.slot_map.numel() == 0
    assert (table == 5).all()


def test_plan_refusals_on_the_cpu():
    table = torch.zeros(2, 3, dtype=torch.int32)
    call = lambda c, n, s, pages, R=8, **kw: paged.page_plan(_i32(c, "cpu"), _i32(n, "cpu"), table, _i32(s, "cpu"), _i32(pages, "cpu"),
                                                             kw.get("ps", 16), R, num_pages=4)
    with pytest.raises(ValueError, match="page_size"):
        call([0], [1], [0], [0], ps=24)
    with pytest.raises(ValueError, match="block table"):
        call([0], [1], [2], [0])
    with pytest.raises(ValueError, match="block table"):
        call([47], [2], [0], [0])
    with pytest.raises(ValueError, match="too few pages"):
        call([0], [1], [0], [])
    with pytest.raises(ValueError, match="outside the pool"):
        call([0], [1], [0], [4])
    with pytest.raises(ValueError, match="same slot"):
        call([0, 0], [1, 1], [0, 0], [0, 1])
    with pytest.raises(ValueError, match="total_rows"):
        call([0], [9], [0], [0])


@pytest.mark.gpu
@pytest.mark.parametrize("cached,new,slots,pages,R,ps", [
    ([0], [1], [2], [0], 8, 16), ([0], [1], [-1], [0], 8, 16), ([47], [2], [0], [0], 8, 16), ([0], [1], [0], [], 8, 16),
    ([0], [1], [0], [4], 8, 16), ([0], [1], [0], [-2], 8, 16), ([0, 0], [1, 1], [0, 0], [0, 1], 8, 16), ([0], [9], [0], [0], 8, 16),
    ([-3], [1], [0], [0], 8, 16), ([2 ** 31 - 1], [1], [0], [0], 8, 16), ([0], [2 ** 31 - 1], [0], [0], 8, 16), ([0], [-1], [0], [0], 8, 16)])
def test_bad_device_data_sets_the_status_and_stays_inside(cached, new, slots, pages, R, ps):
    """What the CPU form refuses is flagged on the device: bad rows get slot -1 (or are left out), nothing outside the table is
    written, and attention and writes on such a plan return."""
    ops = ext.require()
    ops.status(True)
    guard = torch.full((6, 3), -5, dtype=torch.int32, device="cuda")
    table = guard[2:4]
    p = paged.page_plan(_i32(cached, "cuda"), _i32(new, "cuda"), table, _i32(slots, "cuda"), _i32(pages, "cuda"), ps, R, num_pages=4,
                        n_heads=8, n_kv_heads=2)
    assert ops.status(True) & 16
    assert (guard[:2] == -5).all() and (guard[4:] == -5).all()
    assert ((p.slot_map >= -1) & (p.slot_map < 4 * ps)).all() and int(p.row_start[-1]) <= R
    kp, vp = (torch.zeros(4, 2, ps, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    x = torch.ones(R, 2, 64, device="cuda", dtype=torch.bfloat16)
    paged.write_kv(x, x, kp, vp, p.slot_map)
    paged.attention(torch.ones(R, 8, 64, device="cuda", dtype=torch.bfloat16), kp, vp, p, 0.1)
    torch.cuda.synchronize()
    ops.status(True)


# ----------------------------------------------------------------------------------------------------------------- writes
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T,hkv,D,ps,dtype", [(1, 1, 64, 16, torch.bfloat16), (37, 3, 128, 32, torch.float32), (500, 8, 256, 64, torch.bfloat16),
                                              (5, 2, 8, 16, torch.bfloat16)])
def test_write(device, T, hkv, D, ps, dtype):
    g = torch.Generator().manual_seed(T)
    n_pages = T // ps + 5
    pool = torch.randn(n_pages, 2, hkv, ps, D, generator=g).to(dtype).to(device)
    kp, vp = pool[:, 0], pool[:, 1]                                    # strided pools
    packed = torch.randn(T, 4 * hkv, D, generator=g).to(dtype).to(device)
    k, v = packed[:, hkv:2 * hkv], packed[:, 3 * hkv:]                 # strided rows
    slot = torch.randperm(n_pages * ps, generator=g)[:T]
    slot[T // 2] = -1 if T > 1 else slot[0]
    want_k, want_v = kp.clone(), vp.clone()
    for t, s in enumerate(slot.tolist()):
        if s >= 0:
            want_k[s // ps, :, s % ps], want_v[s // ps, :, s % ps] = k[t], v[t]
    paged.write_kv(k, v, kp, vp, slot.to(device))
    assert torch.equal(kp, want_k) and torch.equal(vp, want_v)
    before = pool.clone()
    paged.write_kv(k[:0], v[:0], kp, vp, slot[:0].to(device))          # no rows
    assert torch.equal(pool, before)
    odd = torch.zeros(k.numel() + 1, dtype=dtype, device=device)[1:].view(T, hkv, D)       # vectors not on 16 bytes
    odd.copy_(v)
    paged.write_kv(odd, odd, kp, vp, slot.to(device))
    live = slot.to(device) >= 0
    assert torch.equal(kp.transpose(1, 2).reshape(-1, hkv, D)[slot.to(device)[live]], v[live])


@pytest.mark.gpu
def test_write_past_32_bit_offsets_and_out_of_range_slots():
    n_pages, ps = 20000, 64
    kp = torch.zeros(n_pages, 8, ps, 256, device="cuda", dtype=torch.bfloat16)             # 2.6e9 elements
    x = torch.randn(3, 8, 256, device="cuda").to(torch.bfloat16)
    slots = torch.tensor([n_pages * ps - 1, 0, 17000 * ps + 5], device="cuda")
    paged.write_kv(x, x, kp, kp, slots)
    flat = kp.transpose(1, 2)
    for i, s in enumerate(slots.tolist()):
        assert torch.equal(flat[s // ps, s % ps], x[i])
    ops = ext.require()
    assert ops.status(True) == 0
    paged.write_kv(x, x, kp, kp, torch.tensor([n_pages * ps, -4, 2 ** 40], device="cuda"))
    assert ops.status(True) & 16


def test_write_refusals():
    kp = torch.zeros(2, 2, 16, 64)
    with pytest.raises((RuntimeError, IndexError, ValueError)):
        paged.write_kv(torch.zeros(3, 1, 64), torch.zeros(3, 1, 32), kp, kp, torch.zeros(3, dtype=torch.int64))


# -------------------------------------------------------------------------------------------------------------- attention
_SHAPES = [
    # groups, hq, hkv, D, ps, window
    ([(0, [(0, 1)])], 4, 4, 64, 16, 0),                                            # one token, nothing cached
    ([(0, [(5, 1), (64, 1), (63, 1), (0, 1), (200, 1)])], 8, 2, 128, 16, 0),       # a group without a prefix
    ([(0, [(300, 1)]), (0, [(17, 1)]), (0, [(0, 3)]), (0, [(31, 0)]), (0, [(33, 2)])], 8, 1, 128, 32, 0),
    ([(0, [(1000, 1)])], 28, 4, 128, 64, 0),                                       # seven query heads per key head
    ([(0, [(130, 20)]), (0, [(0, 70)])], 16, 4, 128, 64, 0),                       # many rows a sequence
    ([(128, [(0, 1), (7, 1), (70, 1)]), (0, [(9, 1)]), (64, [(1, 2), (0, 1)])], 8, 2, 128, 64, 0),
    ([(256, [(i, 1) for i in range(20)])], 32, 4, 128, 16, 0),                     # many rows behind one prefix
    ([(192, [(3, 1), (50, 2), (0, 1)]), (0, [(400, 3)])], 8, 2, 64, 64, 100),      # a window that ends inside the prefix
    ([(0, [(90, 5)]), (0, [(500, 1)])], 64, 8, 64, 16, 33),
    ([(64, [(20, 1), (3, 1)]), (0, [(40, 4)])], 16, 4, 256, 32, 0),
    ([(0, [(77, 1)])], 40, 1, 64, 256, 7),
    ([(512, [(10, 9), (0, 30), (100, 1)])], 8, 2, 128, 128, 0),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shape", range(len(_SHAPES)))
@pytest.mark.parametrize("sinks", [False, True])
def test_attention(device, shape, sinks):
    groups, hq, hkv, D, ps, window = _SHAPES[shape]
    s = _Step(groups, hq=hq, hkv=hkv, D=D, ps=ps, device=device, pad=2 if shape % 2 else 0, seed=shape, extra_cols=shape % 3,
              interleaved_pools=shape % 2 == 0)
    sink = s.sink if sinks else None
    for grouped in (True, False):
        got = paged.attention(s.q, s.kp, s.vp, s.plan((window,), grouped), s.scale, window=window, sinks=sink)
        s.check(got, window, sink)
        assert not got[sum(s.new):].any()                                           # rows behind the last sequence
    if device == "cuda":
        assert ext.require().status(True) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("groups,hq,hkv,D,ps,window", [
    ([(0, [(20000, 1)])], 8, 2, 128, 64, 0),                                        # one long sequence: its axis is split
    ([(0, [(c, 1)]) for c in (3000, 1, 77, 2048, 640, 12, 4000)], 32, 8, 128, 64, 0),
    ([(2048, [(c, 1) for c in range(0, 320, 8)]), (1024, [(5, 1)] * 3), (0, [(999, 1)])], 16, 4, 128, 64, 0),
    ([(4096, [(c, 2) for c in range(33)])], 16, 2, 64, 32, 0),
    ([(3000 // 16 * 16, [(c, 1) for c in range(12)])], 16, 2, 256, 16, 500),
    ([(0, [(1000, 500)])], 8, 2, 128, 64, 0),                                       # a chunk of a prompt
    ([(0, [(6000, 1), (100, 1)])], 32, 1, 64, 128, 1024),
    ([(0, [(1000, 300)])] + [(0, [(c, 1)]) for c in (5, 3000, 64, 700)], 16, 4, 128, 32, 0),     # a prompt beside single tokens
])
def test_attention_long(groups, hq, hkv, D, ps, window):
    s = _Step(groups, hq=hq, hkv=hkv, D=D, ps=ps, device="cuda", seed=3)
    got = paged.attention(s.q, s.kp, s.vp, s.plan((window,)), s.scale, window=window)
    s.check(got, window)
    again = paged.attention(s.q, s.kp, s.vp, s.plan((window,)), s.scale, window=window)
    assert torch.equal(got, again)                                                  # the order of the sums is fixed


@pytest.mark.gpu
def test_a_wrong_bound_on_the_rows_costs_speed_only():
    s = _Step([(128, [(c, 2) for c in range(9)]), (0, [(300, 40), (5, 1)])], hq=8, hkv=2, D=128, ps=32, device="cuda")
    for claim in (1, 5, 1000):
        s.check(paged.attention(s.q, s.kp, s.vp, s.plan(max_rows=claim), s.scale))


@pytest.mark.gpu
def test_attention_writes_into_out_and_leaves_the_padding_alone():
    s = _Step([(64, [(5, 1), (9, 1)]), (0, [(30, 2)])], hq=8, hkv=2, D=128, ps=16, device="cuda", pad=3)
    out = torch.full(s.q.shape, 7.0, dtype=s.q.dtype, device="cuda")
    got = paged.attention(s.q, s.kp, s.vp, s.plan(), s.scale, out=out)
    assert got is out and (out[-3:] == 7).all()
    s.check(out)
    want = out.clone()
    wide = torch.zeros(s.R, 20, 128, dtype=s.q.dtype, device="cuda")                # queries as a slice of a packed projection
    wide[:, :8] = s.q
    assert torch.equal(paged.attention(wide[:, :8], s.kp, s.vp, s.plan(), s.scale, out=out)[:-3], want[:-3])
    odd = torch.zeros(s.q.numel() + 1, dtype=s.q.dtype, device="cuda")[1:].view(s.q.shape)
    odd.copy_(s.q)
    assert torch.equal(paged.attention(odd, s.kp, s.vp, s.plan(), s.scale, out=out)[:-3], want[:-3])


@pytest.mark.gpu
def test_attention_with_extreme_scores_and_infinite_keys_outside():
    """Scores of +-3e4 (one key takes everything), equal scores, and a sequence whose neighbour's pages hold infinities."""
    s = _Step([(0, [(100, 1)]), (0, [(50, 1)])], hq=4, hkv=2, D=64, ps=16, device="cuda")
    s.kp[s.pages_of[0][0], 0, 3] = 300.0
    s.q[0] = 1.0
    s.q[1] = 0.0                                                                    # all scores equal
    want, size = s.oracle()
    got = paged.attention(s.q, s.kp, s.vp, s.plan(), s.scale)
    assert ((got.cpu().double() - want).abs() <= 2 ** -8 * want.abs() + (2 ** -8 + 2 ** -12) * size).all()
    s.kp[s.pages_of[0][1]] = float("inf")
    other = paged.attention(s.q, s.kp, s.vp, s.plan(), s.scale)
    assert torch.equal(other[1], got[1])


@pytest.mark.gpu
@pytest.mark.parametrize("groups,window", [
    ([(0, [(70, 1), (9, 1)])], 0),                                                  # one piece a sequence
    ([(0, [(9000, 1), (20, 1)])], 0),                                               # parts of a long axis
    ([(1024, [(40, 1), (700, 1), (3, 1)]), (0, [(11, 1)])], 0),                     # two sources
    ([(4096, [(c, 1) for c in range(40)])], 0),                                     # many rows behind a prefix
    ([(0, [(2000, 40), (5, 20)])], 0),                                              # rows of a prompt
    ([(4096, [(c, 1) for c in range(40)])], 300),
])
@pytest.mark.parametrize("sinks", [False, True])
def test_a_nan_in_sight_stays_a_nan(groups, window, sinks):
    """A query of NaN, and a key of NaN that one row sees: those outputs are NaN, whichever way their keys are cut, and the
    others are what they were.  A sink of minus infinity is no sink."""
    s = _Step(groups, hq=8, hkv=2, D=128, ps=32, device="cuda", seed=7)
    sink = s.sink if sinks else None
    plan = s.plan((window,))
    want, size = s.oracle(window, sink)

    def check(touched):                                                             # [R, Hq]: outputs that have to be NaN
        got = paged.attention(s.q, s.kp, s.vp, plan, s.scale, window=window, sinks=sink).cpu().double()
        assert got[touched].isnan().all()
        err, tol = (got - want).abs()[~touched], (2 ** -8 * want.abs() + (2 ** -8 + 2 ** -12) * size)[~touched]
        assert (err <= tol).all()

    touched = torch.zeros(s.R, s.hq, dtype=torch.bool)
    check(touched)
    if sinks:
        s.check(paged.attention(s.q, s.kp, s.vp, plan, s.scale, window=window, sinks=torch.full_like(s.sink, -math.inf)), window)
    keep = s.q[1].clone()
    s.q[1] = math.nan
    touched[1] = True
    check(touched)
    s.q[1] = keep
    last = s.cached[0] + s.new[0] - 1                                               # only the last row of sequence 0 sees its last token
    s.kp[s.pages_of[0][last // s.ps], 1, last % s.ps] = math.nan
    touched[1] = False
    touched[s.new[0] - 1, 4:] = True
    check(touched)


@pytest.mark.gpu
def test_attention_past_32_bit_offsets():
    ps, D, hkv = 64, 128, 8
    n_pages = 36000                                                                  # 2.4e9 elements a pool
    kp, vp = (torch.zeros(n_pages, hkv, ps, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    ids = [35999, 3, 35998]
    g = torch.Generator("cuda").manual_seed(0)
    for i in ids:
        kp[i] = torch.randn(hkv, ps, D, device="cuda", generator=g).to(kp.dtype)
        vp[i] = torch.randn(hkv, ps, D, device="cuda", generator=g).to(kp.dtype)
    q = torch.randn(1, 8, D, device="cuda", generator=g).to(kp.dtype)
    table = _i32([ids], "cuda")
    plan = lambda t, n: paged.page_plan(_i32([149], "cuda"), _i32([1], "cuda"), t, _i32([0], "cuda"), _i32([], "cuda"), ps, 1,
                                        num_pages=n, mapped=_i32([3], "cuda"), n_heads=8, n_kv_heads=hkv)
    a = paged.attention(q, kp, vp, plan(table, n_pages), 0.1)
    b = paged.attention(q, kp[ids].contiguous(), vp[ids].contiguous(), plan(_i32([[0, 1, 2]], "cuda"), 3), 0.1)
    assert torch.equal(a, b)


@pytest.mark.parametrize("device", DEVICES)
def test_attention_refusals(device):
    s = _Step([(0, [(5, 1)])], hq=4, hkv=2, D=64, ps=16, device=device)
    plan = s.plan()
    with pytest.raises(ValueError, match="query rows"):
        paged.attention(s.q.repeat(2, 1, 1), s.kp, s.vp, plan, 1.0)
    with pytest.raises(ValueError, match="pools"):
        paged.attention(s.q, s.kp[:-1], s.vp[:-1], plan, 1.0)
    with pytest.raises(ValueError, match="pools"):
        paged.attention(s.q, s.kp, s.vp[..., :32], plan, 1.0)
    with pytest.raises(ValueError, match="scale"):
        paged.attention(s.q, s.kp, s.vp, plan, 0.0)
    with pytest.raises(ValueError, match="queries"):
        paged.attention(s.q[:, :3], s.kp, s.vp, plan, 1.0)


@pytest.mark.gpu
def test_other_types_take_the_counted_plain_form():
    from torchtitan_b200.ops import functional as OF

    s = _Step([(0, [(20, 1)])], hq=4, hkv=2, D=64, ps=16, device="cuda", dtype=torch.float32)
    n0 = OF.settings.library_fallbacks
    got = paged.attention(s.q, s.kp, s.vp, s.plan(), s.scale)
    assert OF.settings.library_fallbacks == n0 + 1
    want, size = s.oracle()
    assert ((got.cpu().double() - want).abs() <= 2 ** -12 * (size + want.abs())).all()


@pytest.mark.gpu
def test_a_captured_step_replays_on_other_lengths_and_pages():
    """Plan, write and attention in one graph: the lengths and tables are device data, so a replay follows them."""
    dev, ps, hq, hkv, D, B, W, n_pages = "cuda", 16, 8, 2, 128, 3, 20, 70
    kp, vp = (torch.zeros(n_pages, hkv, ps, D, device=dev, dtype=torch.bfloat16) for _ in range(2))
    cached, new, slots = _i32([0, 0, 0], dev), _i32([1, 1, 1], dev), _i32([0, 1, 2], dev)
    table = torch.arange(B * W, device=dev, dtype=torch.int32).view(B, W).contiguous()
    mapped = _i32([W] * B, dev)
    none = _i32([], dev)
    q = torch.zeros(4, hq, D, device=dev, dtype=torch.bfloat16)
    k, v = (torch.zeros(4, hkv, D, device=dev, dtype=torch.bfloat16) for _ in range(2))

    def step():
        p = paged.page_plan(cached, new, table, slots, none, ps, 4, num_pages=n_pages, mapped=mapped, n_heads=hq, n_kv_heads=hkv)
        paged.write_kv(k, v, kp, vp, p.slot_map)
        return paged.attention(q, kp, vp, p, 0.1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):                                 # two graphs of the same step, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = step()
        graphs.append((g, o))
    rnd = torch.Generator(dev).manual_seed(1)
    for i, lens in enumerate([(5, 100, 0), (300, 1, 64), (17, 200, 31), (3, 4, 5)]):
        for t in (q, k, v, kp, vp):
            t.copy_(torch.randn(t.shape, device=dev, generator=rnd).to(t.dtype))
        cached.copy_(_i32(lens, dev))
        new.copy_(_i32([1, 2, 1] if i % 2 else [1, 1, 1], dev))
        g, o = graphs[i % 2]
        g.replay()
        got = o.clone()
        assert torch.equal(got, step())


@pytest.mark.gpu
def test_a_side_stream_gives_the_same_result():
    s = _Step([(64, [(5, 1), (9, 1)]), (0, [(700, 2)])], hq=8, hkv=2, D=128, ps=16, device="cuda")
    want = paged.attention(s.q, s.kp, s.vp, s.plan(), s.scale)
    outs, streams = [], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for st in streams:                                  # two calls at once
        with torch.cuda.stream(st):
            outs.append(paged.attention(s.q, s.kp, s.vp, s.plan(), s.scale))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.gpu
def test_the_largest_number_of_sequences_and_one_more():
    B, ps, hq, hkv, D = 4096, 16, 4, 2, 64
    g = torch.Generator("cuda").manual_seed(0)
    kp, vp = (torch.randn(B + 1, hkv, ps, D, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
    q = torch.randn(B, hq, D, device="cuda", generator=g).to(torch.bfloat16)
    ar = torch.arange(B, dtype=torch.int32, device="cuda")
    lens = ar % ps
    table = ar.flip(0).view(B, 1).contiguous()
    plan = paged.page_plan(lens, torch.ones_like(ar), table, ar, _i32([], "cuda"), ps, B, num_pages=B + 1, mapped=torch.ones_like(ar),
                           group_start=torch.arange(B + 1, dtype=torch.int32, device="cuda"), group_prefix=torch.zeros_like(ar),
                           n_heads=hq, n_kv_heads=hkv)
    got = paged.attention(q, kp, vp, plan, 0.125)
    assert ext.require().status(True) == 0
    page = table[:, 0].long()
    k, v = kp[page].double(), vp[page].double()                                     # [B, hkv, ps, D]
    s = torch.einsum("bhgd,bhjd->bhgj", q.double().view(B, hkv, 2, D), k) * 0.125
    s = s.masked_fill(torch.arange(ps, device="cuda") > lens[:, None, None, None], float("-inf"))
    p = torch.softmax(s, -1)
    want = torch.einsum("bhgj,bhjd->bhgd", p, v).reshape(B, hq, D)
    size = torch.einsum("bhgj,bhjd->bhgd", p, v.abs()).reshape(B, hq, D)
    assert ((got.double() - want).abs() <= 2 ** -8 * want.abs() + (2 ** -8 + 2 ** -12) * size).all()
    more = torch.zeros(B + 1, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="4096"):
        paged.page_plan(more, more, table, more, _i32([], "cuda"), ps, 0, num_pages=B)


@pytest.mark.gpu
def test_a_group_whose_first_member_has_no_tokens_yet():
    """The first step of a group: the member that computes the prefix has it among its new rows, the others start behind it."""
    s = _Step([(64, [(0, 1), (3, 2), (0, 1)])], hq=8, hkv=2, D=128, ps=32, device="cuda")
    want = paged.attention(s.q, s.kp, s.vp, s.plan(grouped=False), s.scale)
    for prefix in (0, 1, 33, 63, 64, 1000, -5):                                     # clipped to the shortest member
        s.prefix = [prefix]
        s.check(paged.attention(s.q, s.kp, s.vp, s.plan(), s.scale))
    assert torch.equal(want, paged.attention(s.q, s.kp, s.vp, s.plan(grouped=False), s.scale))


@pytest.mark.gpu
def test_pages_with_heads_inside_slots_and_an_expanded_query():
    """Pools laid out [page, slot, head, D] are a permuted view; queries with a stride of zero are copied."""
    s = _Step([(0, [(90, 1), (17, 1)])], hq=8, hkv=2, D=64, ps=16, device="cuda")
    want = paged.attention(s.q, s.kp, s.vp, s.plan(), s.scale)
    kp, vp = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (s.kp, s.vp))
    assert torch.equal(paged.attention(s.q, kp, vp, s.plan(), s.scale), want)
    one = s.q[:1].expand(2, -1, -1)
    assert torch.equal(paged.attention(one, s.kp, s.vp, s.plan(), s.scale), paged.attention(one.contiguous(), s.kp, s.vp, s.plan(), s.scale))


@pytest.mark.gpu
def test_no_sequences_at_all():
    e = _i32([], "cuda")
    table = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    plan = paged.page_plan(e, e, table, e, e, 16, 3, num_pages=4, n_heads=4, n_kv_heads=2)
    kp = torch.zeros(4, 2, 16, 64, device="cuda", dtype=torch.bfloat16)
    assert not paged.attention(torch.ones(3, 4, 64, device="cuda", dtype=torch.bfloat16), kp, kp, plan, 1.0).any()
    plan = paged.page_plan(e, e, table, e, e, 16, 0, num_pages=4, n_heads=4, n_kv_heads=2)
    assert paged.attention(torch.ones(0, 4, 64, device="cuda", dtype=torch.bfloat16), kp, kp, plan, 1.0).shape == (0, 4, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("start", [[0, 3, 1, 4], [0, 4, 0, 4], [2, 0, 2, 4], [0, 2, 9, 9], [-1, 2, 2, 4], [4, 3, 2, 0]])
def test_groups_out_of_order_are_flagged_and_share_nothing(start):
    """Offsets that fall or leave the step: a sequence would belong to two groups.  Results are those without groups."""
    s = _Step([(64, [(5, 1), (9, 1)]), (64, [(30, 2), (3, 1)])], hq=8, hkv=2, D=128, ps=16, device="cuda", pad=1)
    want = paged.attention(s.q, s.kp, s.vp, s.plan(grouped=False), s.scale)
    ops = ext.require()
    assert ops.status(True) == 0
    s.start, s.prefix = start, [64, 64, 64]
    got = paged.attention(s.q, s.kp, s.vp, s.plan(), s.scale)
    assert ops.status(True) & 16
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [
    dict(groups=[(64, [(5, 1), (9, 3)]), (0, [(30, 2)]), (128, [(3, 1), (0, 2), (70, 1)]), (0, [(7, 1)]), (64, [(1, 4), (2, 1)])], hq=8, hkv=2, D=128, ps=32),
    dict(groups=[(0, [(300, 40)]), (256, [(c, 2) for c in range(20)]), (128, [(c, 9) for c in range(5)])], hq=16, hkv=2, D=64, ps=64),
    dict(groups=[(64, [(c, 1) for c in range(4)])] * 3, hq=16, hkv=4, D=256, ps=16),
])
@pytest.mark.parametrize("window", [0, 50])
def test_a_bound_on_the_shared_rows(shape, window):
    """Groups up to the bound share; those beyond it are attended to without sharing: the same results, whatever is claimed."""
    s = _Step(device="cuda", pad=2, seed=11, **shape)
    rows = [sum(s.new[a:b]) for a, b in zip(s.start, s.start[1:])]
    sizes = [n for n, p in zip(rows, s.prefix) if p]
    for claim in (None, s.R, sum(sizes), sum(sizes) - 1, sizes[0], sizes[0] - 1, 1, 0, -3, 10 ** 6):
        plan = s.plan((window,), shared_rows=claim)
        assert plan.shared_rows == (s.R if claim is None else max(0, min(claim, s.R)))
        got = paged.attention(s.q, s.kp, s.vp, plan, s.scale, window=window, sinks=s.sink)
        s.check(got, window, s.sink)
        assert not got[sum(s.new):].any()
    assert ext.require().status(True) == 0


@pytest.mark.gpu
def test_a_long_prompt_without_sharing_takes_little_workspace():
    """4096 rows of 32 heads of 128: partial sums of the rows would be 136 MB."""
    s = _Step([(0, [(0, 1)])], hq=32, hkv=8, D=128, ps=256, device="cuda")
    q = torch.zeros(4096, 32, 128, device="cuda", dtype=torch.bfloat16)
    kp, vp = (torch.zeros(32, 8, 256, 128, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    table = torch.arange(32, device="cuda", dtype=torch.int32).view(2, 16).contiguous()
    i32 = lambda x: _i32(x, "cuda")
    plan = paged.page_plan(i32([0, 64]), i32([4094, 2]), table, i32([0, 1]), i32([]), 256, 4096, num_pages=32, mapped=i32([16, 16]),
                           group_start=i32([0, 2]), group_prefix=i32([0]), n_heads=32, n_kv_heads=8, shared_rows=0)
    out = torch.empty_like(q)
    paged.attention(q, kp, vp, plan, s.scale, out=out)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    paged.attention(q, kp, vp, plan, s.scale, out=out)
    # parts: 296 CTAs x 2 x 16 rows and 148 CTAs x 2 x 128 rows of 130 floats
    assert torch.cuda.max_memory_allocated() - before <= (296 * 32 + 148 * 256) * 130 * 4 + (1 << 20)
    assert ext.require().status(True) == 0


def test_the_plain_forms_raise_on_what_the_kernels_flag():
    """Entries that were in the table before the step, slots and group offsets: nothing is read from the pool's other end."""
    for entry in (-1, 4, 2 ** 31 - 1):
        table = torch.tensor([[0, entry, 2]], dtype=torch.int32)
        plan = lambda c, n, **kw: paged.page_plan(_i32([c], "cpu"), _i32([n], "cpu"), table, _i32([0], "cpu"), _i32([], "cpu"), 16, 4,
                                                  num_pages=4, mapped=_i32([kw.pop("mapped", 3)], "cpu"), **kw)
        with pytest.raises(ValueError, match="outside the pool"):
            plan(20, 2)                                                 # a row of the step lies in that page
        plan(20, 0)
        p = plan(40, 4, n_heads=2, n_kv_heads=1)                        # a page of the past only
        q, kp = torch.zeros(4, 2, 64), torch.zeros(4, 1, 16, 64)
        with pytest.raises(ValueError, match="pool"):
            paged.attention(q, kp, kp, p, 1.0)
        with pytest.raises(ValueError, match="mapped"):
            plan(0, 1, mapped=-1)
        for start in ([0, 2], [1, 0], [-1, 1]):
            with pytest.raises(ValueError, match="order"):
                plan(40, 4, n_heads=2, n_kv_heads=1, group_start=_i32(start, "cpu"), group_prefix=_i32([16], "cpu"))
    kp = torch.zeros(4, 1, 16, 64)
    for slot in (-2, 64, 2 ** 40):
        with pytest.raises(ValueError, match="slot"):
            paged.write_kv(torch.ones(2, 1, 64), torch.ones(2, 1, 64), kp, kp, torch.tensor([5, slot]))
    assert not kp.any()


@pytest.mark.gpu
def test_the_plain_form_on_the_gpu_looks_at_the_pages_first():
    """fp32 pools take the plain form: a page outside the pool is an error on the host, before anything is indexed with it."""
    i32 = lambda x: _i32(x, "cuda")
    for table in ([[0, 9, 1]], [[0, -1, 1]]):
        plan = paged.page_plan(i32([40]), i32([1]), i32(table), i32([0]), i32([]), 16, 1, num_pages=4, mapped=i32([3]), n_heads=2, n_kv_heads=1)
        kp = torch.zeros(4, 1, 16, 64, device="cuda")
        with pytest.raises(ValueError, match="pool"):
            paged.attention(torch.zeros(1, 2, 64, device="cuda"), kp, kp, plan, 1.0)
    assert ext.require().status(True) == 0


@pytest.mark.parametrize("device", DEVICES)
def test_refusals_of_scales_and_windows(device):
    """A scale that is zero or infinite in 32 bits turns masked scores into NaN."""
    s = _Step([(0, [(5, 1)])], hq=4, hkv=2, D=64, ps=16, device=device)
    plan = s.plan((0, 3))
    for scale in (0.0, -1.0, 1e-46, 1e-40, 1e39, math.inf, math.nan):
        with pytest.raises(ValueError, match="scale"):
            paged.attention(s.q, s.kp, s.vp, plan, scale)
    for scale in (1e-37, 1e38):
        assert not paged.attention(s.q, torch.zeros_like(s.kp), s.vp.nan_to_num(), plan, scale).isnan().any()
    with pytest.raises(ValueError, match="window"):
        paged.attention(s.q, s.kp, s.vp, plan, 1.0, window=-1)
    with pytest.raises(ValueError, match="window"):
        s.plan((0, -2))


@pytest.mark.parametrize("device", DEVICES)
def test_group_arguments_come_together(device):
    s = _Step([(0, [(5, 1)])], hq=4, hkv=2, D=64, ps=16, device=device)
    call = lambda **kw: paged.page_plan(_i32(s.cached, device), _i32(s.new, device), s.table, _i32(s.slots, device), _i32([], device), s.ps, s.R,
                                        num_pages=s.n_pages, mapped=_i32([1], device), n_heads=4, n_kv_heads=2, **kw)
    for start, prefix in ((None, [0]), ([0, 1], None), ([0], [0]), ([0, 1], [0, 0]), ([], [])):
        with pytest.raises(ValueError, match="together"):
            call(group_start=None if start is None else _i32(start, device), group_prefix=None if prefix is None else _i32(prefix, device))
    assert call(group_start=_i32([0], device), group_prefix=_i32([], device)).groups == 0


@pytest.mark.gpu
def test_a_negative_count_of_mapped_columns_is_flagged():
    """The plain form raises; the kernel takes it for none."""
    ops = ext.require()
    ops.status(True)
    table = torch.full((1, 3), -5, dtype=torch.int32, device="cuda")
    p = paged.page_plan(_i32([0], "cuda"), _i32([1], "cuda"), table, _i32([0], "cuda"), _i32([2], "cuda"), 16, 1, num_pages=4, mapped=_i32([-3], "cuda"))
    assert ops.status(True) & 16
    assert table.tolist() == [[2, -5, -5]] and p.slot_map.tolist() == [32]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("groups,hq,hkv,D,ps,window", [
    ([(0, [(0, 5), (20, 1)])], 4, 2, 64, 16, 0),                                     # rows of a prompt in one unit
    ([(0, [(37, 3), (0, 2)]), (64, [(9, 2), (70, 1), (0, 1)])], 8, 2, 128, 32, 20),   # windows, a prefix that ends outside them
    ([(0, [(30, 6)])], 4, 1, 256, 16, 8),
    ([(0, [(100, 70), (3, 33)])], 16, 4, 128, 64, 0),                                # units of many rows
    ([(0, [(0, 90)]), (128, [(c, 9) for c in range(0, 70, 5)])], 8, 1, 64, 32, 100),
    ([(256, [(c, 3) for c in range(0, 150, 7)])], 14, 2, 128, 64, 64),
])
def test_values_that_a_row_does_not_see_do_not_reach_it(device, groups, hq, hkv, D, ps, window):
    """Infinite and NaN values in keys of the step: a row that sees them gets what IEEE sums give in those columns, its other
    columns and all other rows are what they were."""
    s = _Step(groups, hq=hq, hkv=hkv, D=D, ps=ps, device=device, seed=5)
    plan = s.plan((window,))
    want, size = s.oracle(window)
    rows, r0 = [], 0                                                                # (sequence, first row, position of each row)
    for b, n in enumerate(s.new):
        rows += [(b, s.cached[b] + i) for i in range(n)]
    g = torch.Generator().manual_seed(1)
    page_of = lambda b, pos: (s.pages_of[b][pos // ps], pos % ps)
    planted = {}                                                                    # (page, slot, head, column) -> value
    for _ in range(12):
        b, pos = rows[int(torch.randint(0, len(rows), (1,), generator=g))]
        pos = max(0, pos - int(torch.randint(0, window or 6, (1,), generator=g)))
        where = (*page_of(b, pos), int(torch.randint(0, hkv, (1,), generator=g)), int(torch.randint(0, D, (1,), generator=g)))
        planted[where] = [math.inf, -math.inf, math.nan][len(planted) % 3]
    for (page, slot, h, c), v in planted.items():
        s.vp[page, h, slot, c] = v
    G = hq // hkv
    hit = torch.zeros(s.R, hq, D, dtype=torch.float64)
    by_key = {}
    for (page, slot, h, c), v in planted.items():
        by_key.setdefault((page, slot), []).append((h, c, v))
    for r, (b, pos) in enumerate(rows):
        for j in range(max(0, pos - window + 1) if window else 0, pos + 1):
            for h, c, v in by_key.get(page_of(b, j), ()):
                hit[r, h * G:(h + 1) * G, c] += v                                   # inf - inf is NaN
    for _ in range(2):
        got = paged.attention(s.q, s.kp, s.vp, plan, s.scale, window=window).cpu().double()
        clean = hit == 0
        assert torch.equal(got[~clean].nan_to_num(7.0, 8.0, 9.0), hit[~clean].nan_to_num(7.0, 8.0, 9.0))
        err = (got - want).abs()[clean]
        assert (err <= (2 ** -8 * want.abs() + (2 ** -8 + 2 ** -12) * size)[clean]).all()
    assert clean.any() and not clean.all()
