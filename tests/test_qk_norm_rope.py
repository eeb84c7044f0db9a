"""Per-head query / key norms with the rotation in the same pass, against the formula in 64 bits.

Tolerances.  An output is rounded once, by at most half a step (``finfo.eps / 2`` of its value).  Before that, fp32: the
mean of squares is a sum of D terms over a tree of at most 8 + 5 additions, the rsqrt is good to 2 ulp, and the value goes
through at most 8 more roundings, each relative to a term no larger than the head's largest one, so 32 units of 2^-24 of the
largest absolute value of the head (for the backward: of ``r (|g| + |xh| mean|g xh|)``) bound what comes before the rounding.
Weight gradients sum T * H products per element with at most that many additions in a row."""

import pytest
import torch

from torchtitan_b200.ops import ext, functional as OF, reference as ref

F32 = 2.0 ** -24
DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _oracle(x, hq, hkv, qw, kw, table, pos, axes, interleaved, eps, gain, q_scale):
    """Double precision, differentiable: pairs as complex numbers."""
    out = []
    for xs, w, sc in ((x[:, :hq], qw, q_scale), (x[:, hq:hq + hkv], kw, 1.0)):
        n = xs / torch.sqrt(xs.square().mean(-1, keepdim=True) + eps) * sc
        if w is not None:
            n = n * (w + gain)
        if table is not None:
            half = table.shape[1] // 2
            f = torch.arange(half, device=x.device)
            at = pos[None].expand(half, -1).t() if axes is None else pos[axes.long()].t()
            turn = torch.complex(table.double()[at, f], table.double()[at, half + f])[:, None]
            i0, i1 = (2 * f, 2 * f + 1) if interleaved else (f, half + f)
            z = torch.complex(n[..., i0], n[..., i1]) * turn
            n = n.index_copy(-1, i0, z.real).index_copy(-1, i1, z.imag)
        out.append(n)
    return out


def _case(T, hq, hkv, D, rot, dtype, device, *, axes=1, weights=True, seed=0, ctx=512):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)
    x = rn(T, hq + 2 * hkv, D).to(dtype)
    qw, kw = ((1 + 0.3 * rn(D)).to(dtype), (1 + 0.3 * rn(D)).to(dtype)) if weights else (None, None)
    table = ref.rope_table(rot, ctx, 10000.0) if rot else None
    pos = torch.randint(0, ctx, (T,) if axes == 1 else (axes, T), generator=g) if rot else None
    ax = torch.randint(0, axes, (rot // 2,), generator=g).int() if rot and axes > 1 else None
    grads = [rn(T, h, D).to(dtype) for h in (hq, hkv, hkv)]
    move = lambda t: None if t is None else t.to(device)
    return [move(t) for t in (x, qw, kw, table, pos, ax)], [move(t) for t in grads]


def _check(ts, grads, hq, hkv, dtype, interleaved, eps=1e-6, gain=0.0, q_scale=1.0):
    x, qw, kw, table, pos, ax = ts
    leaves = [t.detach().clone().requires_grad_(True) if t is not None else None for t in (x, qw, kw)]
    q, k, v = OF.qk_norm_rope(leaves[0], hq, hkv, leaves[1], leaves[2], table, pos, interleaved, eps=eps, gain_center=gain,
                              q_scale=q_scale, axes=ax)
    assert q.dtype == k.dtype == dtype and torch.equal(v, x[:, hq + hkv:])
    wide = [t.detach().double().requires_grad_(True) if t is not None else None for t in (x, qw, kw)]
    want = _oracle(wide[0], hq, hkv, wide[1], wide[2], table, pos, ax, interleaved, eps, gain, q_scale)
    h = _half_step(dtype)
    for a, b in ((q, want[0]), (k, want[1])):
        tol = h * b.abs() + 32 * F32 * b.abs().amax(-1, keepdim=True)
        assert ((a.double() - b).abs() <= tol).all(), float(((a.double() - b).abs() - tol).max())
    have = [t for t in leaves if t is not None]
    got = torch.autograd.grad((q, k, v), have, grads)
    gw = torch.autograd.grad((want[0], want[1], wide[0][:, hq + hkv:]), [t for t in wide if t is not None],
                             [g.double() for g in grads])
    # size of the terms of dx and dw
    for i, (h0, h1, w, sc) in enumerate(((0, hq, wide[1], q_scale), (hq, hq + hkv, wide[2], 1.0))):
        xs = wide[0][:, h0:h1].detach()
        r = 1 / torch.sqrt(xs.square().mean(-1, keepdim=True) + eps)
        xh = xs * r
        big = grads[i].double().norm(dim=-1, keepdim=True)          # a rotation keeps the norm of a pair, so of the head
        gain_max = sc if w is None else float((w + gain).abs().max()) * sc
        size = r * big * gain_max * (1 + xh.abs().amax(-1, keepdim=True) ** 2)
        b = gw[0][:, h0:h1]
        tol = h * b.abs() + 32 * F32 * size
        assert ((got[0][:, h0:h1].double() - b).abs() <= tol).all()
        if w is not None:
            terms = (grads[i].double().abs().amax(-1, keepdim=True) * 2 * xh.abs() * abs(sc)).sum((0, 1))
            tol = h * gw[1 + i].abs() + (xs.shape[0] * xs.shape[1] + 32) * F32 * terms
            assert ((got[1 + i].double() - gw[1 + i]).abs() <= tol).all()
    assert torch.equal(got[0][:, hq + hkv:], grads[2])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T,hq,hkv,D,rot,interleaved,axes", [
    (1, 4, 1, 128, 128, False, 1), (7, 32, 8, 128, 128, False, 1), (33, 5, 3, 64, 64, True, 1), (19, 16, 4, 256, 64, False, 3),
    (5, 2, 2, 16, 16, False, 1), (65, 3, 1, 80, 32, False, 3), (12, 6, 2, 96, 96, True, 2), (9, 1, 1, 8, 8, True, 1),
    (14, 4, 2, 128, 0, False, 1), (300, 9, 1, 120, 48, False, 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_forward_and_gradients(device, T, hq, hkv, D, rot, interleaved, axes, dtype):
    ts, grads = _case(T, hq, hkv, D, rot, dtype, device, axes=axes, weights=T != 33)
    _check(ts, grads, hq, hkv, dtype, interleaved, gain=1.0 if D == 256 else 0.0, q_scale=1.5 if hkv == 1 else 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("T,hq,hkv,D,rot", [(4096, 32, 8, 128, 128), (2500, 16, 4, 256, 64), (6001, 4, 4, 64, 64)])
def test_long_streams(T, hq, hkv, D, rot):
    ts, grads = _case(T, hq, hkv, D, rot, torch.bfloat16, "cuda")
    _check(ts, grads, hq, hkv, torch.bfloat16, False)


def test_gradient_against_differences():
    """The operator's fp32 gradient against central differences of the 64-bit formula along random directions."""
    for device in ["cpu"] + (["cuda"] if torch.cuda.is_available() else []):
        ts, grads = _case(6, 4, 2, 32, 16, torch.float32, device, axes=3)
        x, qw, kw, table, pos, ax = ts
        leaves = [t.clone().requires_grad_(True) for t in (x, qw, kw)]
        out = OF.qk_norm_rope(*leaves[:1], 4, 2, *leaves[1:], table, pos, False, axes=ax, gain_center=0.5)
        got = torch.autograd.grad(out, leaves, grads)

        def f(x_, qw_, kw_):
            q, k = _oracle(x_, 4, 2, qw_, kw_, table, pos, ax, False, 1e-6, 0.5, 1.0)
            return sum((a * g.double()).sum() for a, g in zip((q, k, x_[:, 6:]), grads))

        g = torch.Generator().manual_seed(5)
        base = [t.double() for t in (x, qw, kw)]
        for i in range(3):
            u = torch.randn(base[i].shape, generator=g, dtype=torch.float64).to(device)
            lo, hi = list(base), list(base)
            lo[i], hi[i] = base[i] - 1e-5 * u, base[i] + 1e-5 * u
            diff = float(f(*hi) - f(*lo)) / 2e-5
            # fp32 gradient: 64 units of 2^-24 of the summed terms; differences: third derivatives times 1e-10
            assert abs(float((got[i].double() * u).sum()) - diff) <= 64 * F32 * float((got[i].double() * u).abs().sum()) + 1e-6


@pytest.mark.parametrize("device", DEVICES)
def test_strided_misaligned_and_empty_inputs(device):
    ts, _ = _case(11, 4, 2, 64, 64, torch.bfloat16, device)
    x, qw, kw, table, pos, _ = ts
    want = OF.qk_norm_rope(x, 4, 2, qw, kw, table, pos, False)
    wide = torch.zeros(11, 9, 64, dtype=x.dtype, device=device)
    wide[:, :8] = x
    odd = torch.zeros(x.numel() + 3, dtype=x.dtype, device=device)[3:].view(x.shape)       # rows not on 16 bytes
    odd.copy_(x)
    swapped = x.transpose(0, 1).contiguous().transpose(0, 1)                               # heads outermost
    for y in (wide[:, :8], odd, swapped):
        for a, b in zip(OF.qk_norm_rope(y, 4, 2, qw, kw, table, pos, False), want):
            assert torch.equal(a, b)
    leaf = x.clone().requires_grad_(True)
    q, k, v = OF.qk_norm_rope(leaf, 4, 2, qw, kw, table, pos, False)
    dq = torch.randn(64, 4, 11, device=device).to(x.dtype).permute(2, 1, 0)                 # any strides
    (g1,) = torch.autograd.grad(q, leaf, dq, retain_graph=True)                             # k and v unused: zero gradients
    (g2,) = torch.autograd.grad(q, leaf, dq.contiguous())
    assert torch.equal(g1, g2) and not g1[:, 4:].any()
    q, k, v = OF.qk_norm_rope(x[:0], 4, 2, qw, kw, table, pos[:0], False)
    assert q.shape == (0, 4, 64) and k.shape == (0, 2, 64)
    zero = torch.zeros(2, 8, 64, dtype=x.dtype, device=device).requires_grad_(True)        # a zero vector stays finite
    q, k, v = OF.qk_norm_rope(zero, 4, 2, qw, kw, table, pos[:2], False)
    (g,) = torch.autograd.grad(q.float().sum(), zero)
    assert not q.any() and torch.isfinite(g.float()).all()


def test_refusals():
    ts, _ = _case(3, 4, 2, 64, 64, torch.float32, "cpu")
    x, qw, kw, table, pos, _ = ts
    with pytest.raises(ValueError, match="expected"):
        OF.qk_norm_rope(x, 4, 1, qw, kw, table, pos, False)
    with pytest.raises(ValueError, match="positions"):
        OF.qk_norm_rope(x, 4, 2, qw, kw, table, pos[:2], False)
    with pytest.raises(ValueError, match="rotary width"):
        OF.qk_norm_rope(x[..., :32], 4, 2, qw[:32], kw[:32], table, pos, False)
    with pytest.raises(ValueError, match="rotary width"):
        OF.qk_norm_rope(x, 4, 2, qw, kw, table[:, :24].contiguous(), pos, False)


@pytest.mark.gpu
def test_refusals_and_bad_positions_on_the_gpu():
    ts, _ = _case(3, 4, 2, 64, 64, torch.float32, "cuda")
    x, qw, kw, table, pos, _ = ts
    for bad in (dict(x=x.half()), dict(qw=qw.bfloat16()), dict(table=table.double()), dict(pos=pos.cpu()), dict(x=x[..., :60])):
        a = dict(x=x, qw=qw, kw=kw, table=table, pos=pos, **{})
        a.update(bad)
        with pytest.raises((RuntimeError, ValueError)):
            OF.qk_norm_rope(a["x"], 4, 2, a["qw"], a["kw"], a["table"], a["pos"], False)
    ops = ext.require()
    ops.status(True)
    q, _, _ = OF.qk_norm_rope(x, 4, 2, qw, kw, table, torch.tensor([0, 100000, -3], device="cuda"), False)
    assert torch.isfinite(q).all() and ops.status(True) & 1
    axes = torch.full((32,), 7, dtype=torch.int32, device="cuda")                # an axis that does not exist
    OF.qk_norm_rope(x, 4, 2, qw, kw, table, pos[None].repeat(3, 1), False, axes=axes)
    assert ops.status(True) & 1


@pytest.mark.gpu
def test_captured_forward_and_backward_replay_on_new_inputs():
    ts, grads = _case(40, 8, 2, 128, 128, torch.bfloat16, "cuda")
    x, qw, kw, table, pos, _ = ts

    def step(x_):
        leaf = x_.detach().requires_grad_(True)
        w = [t.detach().requires_grad_(True) for t in (qw, kw)]
        out = OF.qk_norm_rope(leaf, 8, 2, *w, table, pos, False)
        return [t.detach() for t in out[:2]] + list(torch.autograd.grad(out, [leaf, *w], grads))

    static = x.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(static)
    for seed in (1, 2):
        fresh = torch.randn(x.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).to(x.dtype)
        static.copy_(fresh)
        graph.replay()
        for a, b in zip(got, step(fresh)):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("T,rot,weights,dtype", [(300, 128, (True, True), torch.bfloat16), (1, 64, (True, False), torch.bfloat16),
                                                 (70, 0, (False, True), torch.float32), (70, 32, (False, False), torch.float32)])
def test_the_python_and_the_cpp_node_agree(T, rot, weights, dtype, monkeypatch):
    """Gradients into ``main_grad`` and counted launches go through the node in Python, everything else through the one in C++:
    the same kernels, so the same bits, with any of the three outputs left out, under a checkpoint and next to ``main_grad``."""
    (x, qw, kw, table, pos, ax), grads = _case(T, 8, 2, 128, rot, dtype, "cuda")
    qw, kw = (w if on else None for w, on in zip((qw, kw), weights))

    def grads_of(used, counted, saved=False, main=False):
        monkeypatch.setattr(OF.settings, "count_launches", counted)
        leaves = [t.detach().clone().requires_grad_(True) if t is not None else None for t in (x, qw, kw)]
        held = [t for t in leaves if t is not None]
        for w in held[1:]:
            if main:
                w.main_grad = torch.empty_like(w.detach())
        fn = lambda a, b, c: OF.qk_norm_rope(a, 8, 2, b, c, table, pos, False, axes=ax)
        outs = torch.utils.checkpoint.checkpoint(fn, *leaves, use_reentrant=False) if saved else fn(*leaves)
        torch.autograd.backward([outs[i] for i in used], [grads[i] for i in used])
        return [outs[i].detach() for i in used] + [t.main_grad if getattr(t, "main_grad", None) is not None else t.grad for t in held]

    for used in ((0, 1, 2), (0,), (1,), (2,), (1, 2)):
        want = grads_of(used, True)
        for got in (grads_of(used, False), grads_of(used, False, saved=True), grads_of(used, False, main=True)):
            assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True))


@pytest.mark.gpu
def test_only_a_weight_needs_its_gradient():
    (x, qw, kw, table, pos, ax), grads = _case(40, 4, 2, 64, 64, torch.bfloat16, "cuda")
    full = [t.detach().clone().requires_grad_(True) for t in (x, qw, kw)]
    only = qw.detach().clone().requires_grad_(True)
    q, k, _ = OF.qk_norm_rope(full[0], 4, 2, full[1], full[2], table, pos, False)
    torch.autograd.backward([q, k], grads[:2])
    q, k, v = OF.qk_norm_rope(x, 4, 2, only, kw, table, pos, False)
    torch.autograd.backward([q, k], grads[:2])
    assert torch.equal(only.grad, full[1].grad) and x.grad is None and kw.grad is None


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T,hq,hkv,D,rot", [
    (1, 3, 1, 128, 128), (33, 5, 3, 64, 64),                                     # few tokens: a head a lane
    (2600, 12, 4, 128, 128), (4800, 3, 1, 64, 32), (2400, 5, 3, 256, 64)])       # several heads a lane
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_without_eps_heads_that_do_not_fill_a_warp_keep_their_weight_gradients(device, T, hq, hkv, D, rot, dtype):
    """A warp works on a power of two of heads; those past the last one are zeros, whose rsqrt is infinite at ``eps = 0``."""
    if device == "cpu" and T > 100:
        T = 100
    ts, grads = _case(T, hq, hkv, D, rot, dtype, device)
    _check(ts, grads, hq, hkv, dtype, False, eps=0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hq,hkv,D,rot", [(32, 8, 128, 128), (5, 3, 64, 32), (16, 4, 256, 64)])
def test_a_token_does_not_depend_on_the_others(dtype, hq, hkv, D, rot):
    """Batch-invariant mode allows the operator: few tokens (a head a lane) and many (several) give a token the same bits."""
    ts, grads = _case(5000, hq, hkv, D, rot, dtype, "cuda")
    x, qw, kw, table, pos, _ = ts

    def run(sl):
        leaf = x[sl].detach().clone().requires_grad_(True)
        out = OF.qk_norm_rope(leaf, hq, hkv, qw, kw, table, pos[sl].contiguous(), False)
        return [t.detach() for t in out] + list(torch.autograd.grad(out, leaf, [g[sl] for g in grads]))

    whole = run(slice(0, 5000))
    for sl in (slice(0, 1), slice(37, 50), slice(4000, 5000)):
        assert all(torch.equal(a, b[sl]) for a, b in zip(run(sl), whole))
