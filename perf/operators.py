"""Work on which the operators of a generated token's attention step (and its training twin) are timed.

Four operators: the per-head query / key norms with the rotation in the same pass (``qkn``), the step plan of the paged
key / value cache (``plan``), the scatter of new keys and values into pages (``write``) and attention over the pages with
shared prefixes (``attn``).  ``run`` is either their plain form in elementary torch operations or the call of the
framework's operator, by ``own``.
"""

import math

import torch

own = False

DEV = "cuda"
_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one decode step of a small batch: a single launch, latency
        _qkn("qkn_decode", T=48, hq=32, hkv=8, D=128, rot=128),
        # training forward + backward of a layer with 32 query and 4 key heads at the headline sequence length
        _qkn("qkn_train", T=8192, hq=32, hkv=4, D=128, rot=128, grad=True),
        # vision-language training: three position axes, a quarter of a 256-wide head rotates, gains centred at one
        _qkn("qkn_train_axes", T=4097, hq=16, hkv=4, D=256, rot=64, axes=3, gain=1.0, grad=True),
        # fp32 debugging runs: adjacent pairs, norms without gains, an odd token count
        _qkn("qkn_train_fp32", T=1023, hq=16, hkv=8, D=64, rot=64, dtype="fp32", interleaved=True, weights=False, grad=True),
        # page tables of a handful of requests that decode
        _plan("plan_decode", B=9, ps=16, max_cached=2000, max_new=1),
        # a full engine step: hundreds of requests, some of them with whole prompts, page tables of long contexts
        _plan("plan_mixed", B=500, ps=16, max_cached=30000, max_new=200),
        # the new rows of a decode step
        _write("write_decode", T=64, hkv=8, D=128, ps=64),
        # the rows of newly admitted prompts
        _write("write_prompt", T=16001, hkv=8, D=128, ps=64),
        # a single request far into its context: the axis has to be split
        _attn("attn_one_long", groups=[(1, 0)], lens=(100000, 100000), hq=32, hkv=8, D=128, ps=64),
        # a decode step over requests of very different lengths
        _attn("attn_decode_ragged", groups=[(1, 0)] * 61, lens=(30, 8000), hq=32, hkv=8, D=128, ps=64),
        # sampled groups: several prompts, each with many completions of different lengths behind it
        _attn("attn_shared_prefix", groups=[(16, 8192)] * 4 + [(1, 0)] * 3, lens=(1, 1000), hq=32, hkv=4, D=128, ps=64),
        # a few rows a request (the last rows of cached prompts), sliding window, sinks, 64-wide heads, small pages
        _attn("attn_rows_window", groups=[(1, 0)] * 24, lens=(0, 3000), hq=64, hkv=8, D=64, ps=16, max_new=9, window=128, sinks=True),
    ]


def _qkn(name, *, T, hq, hkv, D, rot, dtype="bf16", axes=1, interleaved=False, weights=True, gain=0.0, q_scale=1.0, grad=False):
    return dict(name=name, op="qkn", T=T, hq=hq, hkv=hkv, D=D, rot=rot, dtype=dtype, axes=axes, interleaved=interleaved,
                weights=weights, gain=gain, q_scale=q_scale, grad=grad, ctx=32768)


def _plan(name, *, B, ps, max_cached, max_new, pad=0, shared=False):
    return dict(name=name, op="plan", B=B, ps=ps, max_cached=max_cached, max_new=max_new, pad=pad, shared=shared)


def _write(name, *, T, hkv, D, ps, dtype="bf16"):
    return dict(name=name, op="write", T=T, hkv=hkv, D=D, ps=ps, dtype=dtype)


def _attn(name, *, groups, lens, hq, hkv, D, ps, max_new=1, window=0, sinks=False):
    """``groups``: (sequences, tokens of their common prefix); ``lens``: range of the cached tokens behind the prefix."""
    return dict(name=name, op="attn", groups=" ".join(f"{n}x{p}" for n, p in groups), lo=lens[0], hi=lens[1], hq=hq, hkv=hkv, D=D, ps=ps,
                max_new=max_new, window=window, sinks=sinks)


def _groups(case):
    return [tuple(int(x) for x in g.split("x")) for g in case["groups"].split()]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    kind = rng.choice(["qkn", "qkn", "plan", "write", "attn", "attn", "attn"])
    if kind == "qkn":
        hkv = rng.choice([1, 2, 4, 8])
        D = rng.choice([16, 64, 80, 96, 128, 256])
        rot = rng.choice([r for r in (16, 32, 64, 80, 96, 128, 256) if r <= D])
        hq = hkv * rng.choice([1, 2, 4, 5, 8])
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        grad = rng.random() < 0.6
        top = (8192 * 36 * 128) // ((hq + hkv) * D * (2 if dtype == "fp32" else 1))
        return _qkn(None, T=_log(rng, 1, min(top, 30000)), hq=hq, hkv=hkv, D=D, rot=rot, dtype=dtype,
                    axes=rng.choice([1, 1, 3]), interleaved=rng.random() < 0.3, weights=rng.random() < 0.8,
                    gain=rng.choice([0.0, 1.0]), q_scale=rng.choice([1.0, 1.5]), grad=grad)
    if kind == "plan":
        return _plan(None, B=_log(rng, 1, 500), ps=rng.choice([16, 32, 64, 128]), max_cached=_log(rng, 50, 30000),
                     max_new=_log(rng, 1, 200), pad=rng.choice([0, 0, 7]), shared=rng.random() < 0.5)
    if kind == "write":
        return _write(None, T=_log(rng, 1, 16000), hkv=rng.choice([1, 2, 4, 8]), D=rng.choice([64, 128, 256]),
                      ps=rng.choice([16, 32, 64, 128]), dtype=rng.choice(["bf16", "bf16", "fp32"]))
    hq, hkv, D = rng.choice([(32, 8, 128), (32, 4, 128), (16, 8, 128), (28, 4, 128), (64, 8, 64), (16, 4, 256), (8, 1, 128), (4, 4, 64)])
    shape = rng.choice(["one", "ragged", "ragged", "shared", "rows"])
    window = rng.choice([0, 0, 0, 128, 1000])
    sinks = rng.random() < 0.25
    ps = rng.choice([16, 32, 64, 128])
    if shape == "one":
        n = _log(rng, 1, 100000)
        return _attn(None, groups=[(1, 0)], lens=(n, n), hq=hq, hkv=hkv, D=D, ps=ps, window=window, sinks=sinks,
                     max_new=rng.choice([1, 1, 4]))
    if shape == "ragged":
        return _attn(None, groups=[(1, 0)] * _log(rng, 2, 64), lens=(0, _log(rng, 10, 6000)), hq=hq, hkv=hkv, D=D, ps=ps,
                     window=window, sinks=sinks)
    if shape == "rows":
        return _attn(None, groups=[(1, 0)] * _log(rng, 1, 16), lens=(0, _log(rng, 1, 3000)), hq=hq, hkv=hkv, D=D, ps=ps,
                     window=window, sinks=sinks, max_new=_log(rng, 2, 100))
    groups = []
    for _ in range(rng.randint(1, 4)):
        groups.append((_log(rng, 1, 16), ps * _log(rng, 1, 8000 // ps)))
    return _attn(None, groups=groups, lens=(0, _log(rng, 1, 800)), hq=hq, hkv=hkv, D=D, ps=ps, window=window, sinks=sinks,
                 max_new=rng.choice([1, 1, 3]))


# ----------------------------------------------------------------------------------------------------------- the inputs
def _axis_map(rot, axes):
    """Which position axis each of the rot / 2 frequencies follows: interleaved thirds, the rest on the first axis."""
    f = torch.arange(rot // 2, dtype=torch.int32)
    if axes == 1:
        return None
    third = (rot // 2) // 3
    out = torch.zeros_like(f)
    for a in (1, 2):
        out[(f % 3 == a) & (f < 3 * third)] = a
    return out


def _new_rows(case, n):
    """New rows of each of ``n`` sequences: their sum, the length of the token stream, belongs to the case."""
    rng = torch.Generator().manual_seed(1000 * n + case["max_new"])
    return torch.randint(1, case["max_new"] + 1, (n,), generator=rng).tolist()


def _plan_inputs(case, g, cpu):
    """Request lengths of a step, the table as the step before left it, and the pages to hand out."""
    B, ps = case["B"], case["ps"]
    cached = torch.randint(0, case["max_cached"] + 1, (B,), generator=cpu)
    new = torch.tensor(_new_rows(case, B))
    if B > 3:
        new[0] = 0                                   # one that waits this step out
        cached[1] = 0                                # a request that was just admitted
    new = new[torch.randperm(B, generator=cpu)]
    W = -(-(case["max_cached"] + case["max_new"]) // ps)
    S = B + 5
    held = (cached + ps - 1) // ps
    mapped = held.clone()
    if case["shared"]:
        mapped[0] = 0                                # newly admitted with a cached prefix: its pages come with the call
    end = (cached + new + ps - 1) // ps
    n_pages = int(held.sum() + (end - mapped).sum()) + 3
    perm = torch.randperm(n_pages, generator=cpu).to(torch.int32)
    table = torch.full((S, W), -1, dtype=torch.int32)
    slots = torch.randperm(S, generator=cpu)[:B].to(torch.int32)
    at = 0
    for b in range(B):
        n = int(mapped[b])
        table[slots[b], :n] = perm[at:at + n]
        at += n
    i32 = dict(dtype=torch.int32, device=DEV)
    return dict(cached=cached.to(**i32), new=new.to(**i32), mapped=mapped.to(**i32), slots=slots.to(DEV), table=table.to(DEV),
                pages=perm[at:at + int((end - mapped).sum())].to(DEV), ps=ps, n_pages=n_pages,
                rows=int(new.sum()) + case["pad"])


def _attn_inputs(case, g, cpu):
    ps, D, hkv = case["ps"], case["D"], case["hkv"]
    new = _new_rows(case, sum(n for n, _ in _groups(case)))
    new = [new[i] for i in torch.randperm(len(new), generator=cpu).tolist()]
    cached, owner, start, prefix = [], [], [0], []
    for gi, (n, p) in enumerate(_groups(case)):
        for _ in range(n):
            cached.append(p + int(torch.randint(case["lo"], case["hi"] + 1, (1,), generator=cpu)))
            owner.append(gi)
        start.append(len(cached))
        prefix.append(p)
    B = len(cached)
    total = [c + n for c, n in zip(cached, new)]
    W = max(-(-t // ps) for t in total)
    firsts = [start[o] for o in owner]
    common = [prefix[owner[b]] // ps if b != firsts[b] else 0 for b in range(B)]     # pages a member takes from the first
    n_pages = sum(-(-t // ps) - k for t, k in zip(total, common)) + 2
    perm = torch.randperm(n_pages, generator=cpu).to(torch.int32)
    table = torch.full((B, W), -1, dtype=torch.int32)
    at = 0
    for b in range(B):
        k, n = common[b], -(-total[b] // ps)
        table[b, :k] = table[firsts[b], :k]
        table[b, k:n] = perm[at:at + n - k]
        at += n - k
    R = sum(new)
    kp = torch.randn(n_pages, hkv, ps, D, device=DEV, generator=g).to(torch.bfloat16)
    vp = torch.randn(n_pages, hkv, ps, D, device=DEV, generator=g).to(torch.bfloat16)
    q = torch.randn(R, case["hq"], D, device=DEV, generator=g).to(torch.bfloat16)
    sinks = torch.randn(case["hq"], device=DEV, generator=g) if case["sinks"] else None
    return dict(q=q, kp=kp, vp=vp, table=table.to(DEV), sinks=sinks, cached=cached, new=new, start=start, prefix=prefix, ps=ps)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed + 17)
    s = dict(case=case, op=case["op"])
    if case["op"] == "qkn":
        dt, T, hq, hkv, D, rot = _DT[case["dtype"]], case["T"], case["hq"], case["hkv"], case["D"], case["rot"]
        rn = lambda *shape: torch.randn(*shape, device=DEV, generator=g)
        s["qkv"] = rn(T, hq + 2 * hkv, D).to(dt).requires_grad_(case["grad"])
        mid = 1.0 - case["gain"]
        w = [(mid + 0.2 * rn(D)).to(dt).requires_grad_(case["grad"]) for _ in range(2)] if case["weights"] else [None, None]
        s["qw"], s["kw"] = w
        inv = 1.0 / (1e6 ** (torch.arange(0, rot, 2, dtype=torch.float64) / rot))
        ang = torch.outer(torch.arange(case["ctx"], dtype=torch.float64), inv)
        s["table"] = torch.cat([ang.cos(), ang.sin()], 1).float().to(DEV)
        if case["axes"] == 1:
            first = torch.randint(0, case["ctx"] - T, (1,), generator=cpu) if T < case["ctx"] else torch.zeros(1, dtype=torch.int64)
            s["pos"] = (torch.arange(T) + first).to(DEV)
        else:
            s["pos"] = torch.randint(0, case["ctx"], (case["axes"], T), generator=cpu).to(DEV)
        m = _axis_map(rot, case["axes"])
        s["axes"] = None if m is None else m.to(DEV)
        if case["grad"]:
            s["dout"] = [rn(T, h, D).to(dt) for h in (hq, hkv, hkv)]
    elif case["op"] == "plan":
        s.update(_plan_inputs(case, g, cpu))
    elif case["op"] == "write":
        dt, T, ps = _DT[case["dtype"]], case["T"], case["ps"]
        n_pages = -(-T // ps) + 3 + min(T, 64)
        shape = (n_pages, case["hkv"], ps, case["D"])
        s["kp"], s["vp"] = (torch.zeros(shape, device=DEV, dtype=dt) for _ in range(2))
        # new keys are a fresh tensor, values are the tail heads of a packed projection output
        s["k"] = torch.randn(T, case["hkv"], case["D"], device=DEV, generator=g).to(dt)
        s["v"] = torch.randn(T, 3 * case["hkv"], case["D"], device=DEV, generator=g).to(dt)[:, 2 * case["hkv"]:]
        if T <= 64:                                  # decode: every row goes to a page of its own
            page = torch.randperm(n_pages, generator=cpu)[:T]
            s["slot"] = (page * ps + torch.randint(0, ps, (T,), generator=cpu)).to(DEV)
        else:                                        # prompts: consecutive rows fill pages handed out in random order
            page = torch.randperm(n_pages, generator=cpu)
            r = torch.arange(T)
            s["slot"] = (page[r // ps] * ps + r % ps).to(DEV)
    else:
        s.update(_attn_inputs(case, g, cpu))
        s["scale"] = 1.0 / math.sqrt(case["D"])
        if own:
            # the plan of the step: made once, used by every layer
            from torchtitan_b200.ops import paged

            i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
            B = len(s["cached"])
            held = i32([-(-(c + n) // s["ps"]) for c, n in zip(s["cached"], s["new"])])
            s["plan"] = paged.page_plan(
                i32(s["cached"]), i32(s["new"]), s["table"], torch.arange(B, dtype=torch.int32, device=DEV),
                torch.empty(0, dtype=torch.int32, device=DEV), s["ps"], sum(s["new"]), num_pages=s["kp"].shape[0], mapped=held,
                group_start=i32(s["start"]), group_prefix=i32(s["prefix"]), n_heads=case["hq"], n_kv_heads=case["hkv"],
                windows=(case["window"],), max_rows=max(max(s["new"]), max(
                    sum(s["new"][a:b]) for a, b in zip(s["start"], s["start"][1:]))))
    return s


# ---------------------------------------------------------------------------------------------------------- the passes
def _qkn_plain_one(x, w, cos, sin, case, scale):
    rot, half = case["rot"], case["rot"] // 2
    n = x.float()
    n = n * torch.rsqrt((n * n).mean(-1, keepdim=True) + 1e-6) * scale
    if w is not None:
        n = n * (w.float() + case["gain"])
    r, rest = n[..., :rot], n[..., rot:]
    if case["interleaved"]:
        a, b = r[..., 0::2], r[..., 1::2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = r[..., :half], r[..., half:]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y, rest], -1).to(x.dtype)


def _qkn_run(s):
    case = s["case"]
    hq, hkv = case["hq"], case["hkv"]
    if own:
        from torchtitan_b200.ops import functional as OF

        q, k, v = OF.qk_norm_rope(s["qkv"], hq, hkv, s["qw"], s["kw"], s["table"], s["pos"], case["interleaved"], eps=1e-6,
                                  gain_center=case["gain"], q_scale=case["q_scale"], axes=s["axes"])
    else:
        half = case["rot"] // 2
        if s["axes"] is None:
            cs = s["table"][s["pos"]]
        else:
            f = torch.arange(half, device=DEV)
            at = s["pos"][s["axes"].long()].t()
            cs = torch.cat([s["table"][at, f], s["table"][at, f + half]], 1)
        cos, sin = cs[:, None, :half], cs[:, None, half:]
        q = _qkn_plain_one(s["qkv"][:, :hq], s["qw"], cos, sin, case, case["q_scale"])
        k = _qkn_plain_one(s["qkv"][:, hq:hq + hkv], s["kw"], cos, sin, case, 1.0)
        v = s["qkv"][:, hq + hkv:]
    if not case["grad"]:
        return {"q": q, "k": k}
    leaves = [s["qkv"]] + ([s["qw"], s["kw"]] if case["weights"] else [])
    grads = torch.autograd.grad((q, k, v), leaves, s["dout"])
    out = {"q": q.detach(), "k": k.detach(), "dqkv": grads[0]}
    if case["weights"]:
        out["dqw"], out["dkw"] = grads[1], grads[2]
    return out


def _plan_run(s):
    ps, R = s["ps"], s["rows"]
    if own:
        from torchtitan_b200.ops import paged

        p = paged.page_plan(s["cached"], s["new"], s["table"], s["slots"], s["pages"], ps, R, num_pages=s["n_pages"],
                            mapped=s["mapped"])
        return {"table": s["table"], "row_start": p.row_start, "positions": p.positions, "slot_map": p.slot_map}
    cached, new, mapped, table, slots = s["cached"].long(), s["new"].long(), s["mapped"].long(), s["table"], s["slots"].long()
    W = table.shape[1]
    need = (cached + new + ps - 1) // ps - mapped
    off = need.cumsum(0) - need
    row_start = torch.cat([new.new_zeros(1), new.cumsum(0)])
    rows = table[slots].long()
    col = torch.arange(W, device=DEV)[None]
    mine = (col >= mapped[:, None]) & (col < (mapped + need)[:, None])
    at = (off[:, None] + col - mapped[:, None]).clamp(0, max(s["pages"].numel() - 1, 0))
    if s["pages"].numel():
        rows = torch.where(mine, s["pages"].long()[at], rows)
    table[slots] = rows.to(torch.int32)
    r = torch.arange(R, device=DEV)
    seq = torch.searchsorted(row_start[1:], r, right=True)
    live = seq < new.numel()
    seq = seq.clamp(max=new.numel() - 1)
    pos = torch.where(live, cached[seq] + r - row_start[seq], torch.zeros_like(r))
    slot = torch.where(live, rows[seq, pos // ps] * ps + pos % ps, torch.full_like(r, -1))
    return {"table": table, "row_start": row_start.to(torch.int32), "positions": pos, "slot_map": slot}


def _write_run(s):
    if own:
        from torchtitan_b200.ops import paged

        paged.write_kv(s["k"], s["v"], s["kp"], s["vp"], s["slot"])
    else:
        ps = s["case"]["ps"]
        page, off = s["slot"] // ps, s["slot"] % ps
        s["kp"][page, :, off] = s["k"]
        s["vp"][page, :, off] = s["v"]
    return {"k_pages": s["kp"], "v_pages": s["vp"]}


def _attn_run(s):
    case = s["case"]
    if own:
        from torchtitan_b200.ops import paged

        return paged.attention(s["q"], s["kp"], s["vp"], s["plan"], s["scale"], window=case["window"], sinks=s["sinks"])
    hq, hkv, D, ps = case["hq"], case["hkv"], case["D"], s["ps"]
    outs, r0 = [], 0
    for b, (c, n) in enumerate(zip(s["cached"], s["new"])):
        L = c + n
        pages = s["table"][b, :-(-L // ps)].long()
        k = s["kp"][pages].transpose(0, 1).reshape(hkv, -1, D)[:, :L].float()
        v = s["vp"][pages].transpose(0, 1).reshape(hkv, -1, D)[:, :L].float()
        q = s["q"][r0:r0 + n].float().view(n, hkv, hq // hkv, D).permute(1, 2, 0, 3).reshape(hkv, -1, D)    # [hkv, G n, D]
        sc = torch.matmul(q, k.transpose(1, 2)).view(hkv, hq // hkv, n, L) * s["scale"]
        i, j = torch.arange(n, device=DEV)[:, None] + c, torch.arange(L, device=DEV)[None]
        see = j <= i
        if case["window"]:
            see &= j > i - case["window"]
        sc = torch.where(see, sc, torch.full_like(sc, float("-inf")))
        m = sc.amax(-1, keepdim=True)
        if s["sinks"] is not None:
            sink = s["sinks"].view(hkv, -1, 1, 1)
            m = torch.maximum(m, sink)
        p = torch.exp(sc - m)
        den = p.sum(-1, keepdim=True)
        if s["sinks"] is not None:
            den = den + torch.exp(sink - m)
        o = torch.matmul(p.view(hkv, -1, L), v).view(hkv, hq // hkv, n, D) / den
        outs.append(o.permute(2, 0, 1, 3).reshape(n, hq, D).to(torch.bfloat16))
        r0 += n
    return torch.cat(outs)


def run(state):
    return {"qkn": _qkn_run, "plan": _plan_run, "write": _write_run, "attn": _attn_run}[state["op"]](state)


# ------------------------------------------------------------------------------------------------------------- the work
def work(case):
    if case["op"] == "qkn":
        e = 2 if case["dtype"] == "bf16" else 4
        T, hq, hkv, D = case["T"], case["hq"], case["hkv"], case["D"]
        b = 2 * T * (hq + hkv) * D * e + 8 * T * case["axes"] + 4 * min(T * case["axes"], case["ctx"]) * case["rot"]
        f = 8 * T * (hq + hkv) * D
        if case["grad"]:
            b += T * D * e * (2 * (hq + hkv) + hkv + hq + 2 * hkv)
            f += 16 * T * (hq + hkv) * D
        return {"bytes": b, "flops": f}
    if case["op"] == "plan":
        rows = case["B"] * (1 + case["max_new"]) // 2 + case["pad"]
        pages = case["B"] * (1 + case["max_new"] // (2 * case["ps"]))
        return {"bytes": case["B"] * 20 + pages * 8 + rows * 20, "flops": 10 * rows}
    if case["op"] == "write":
        e = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": 4 * case["T"] * case["hkv"] * case["D"] * e + 8 * case["T"], "flops": 0}
    hq, hkv, D, w = case["hq"], case["hkv"], case["D"], case["window"]
    rows_per, tail = (1 + case["max_new"]) / 2, (case["lo"] + case["hi"]) / 2
    keys = flops = rows = 0.0
    for n, p in _groups(case):
        seen = tail + rows_per
        own_keys, shared = seen, p
        if w:
            own_keys = min(seen, w + rows_per)
            shared = min(p, max(0.0, w + rows_per - own_keys))
        keys += n * own_keys + shared
        rows += n * rows_per
        flops += n * rows_per * 4 * hq * D * (min(seen + p, w) if w else seen + p)
    return {"bytes": int(keys * hkv * D * 4 + rows * hq * D * 4), "flops": int(flops)}


# ------------------------------------------------------------------------------------- the definitions in 64 bits, again
def exact(case, seed):
    if case["op"] == "plan":
        return None                                  # whole numbers only
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    with torch.no_grad():
        return {"qkn": _exact_qkn, "write": _exact_write, "attn": _exact_attn}[case["op"]](s)


def _exact_write(s):
    ps, out = s["case"]["ps"], {}
    for name, new, pages in (("k_pages", s["k"], s["kp"]), ("v_pages", s["v"], s["vp"])):
        by_slot = pages.double().transpose(1, 2).flatten(0, 1)                  # [slots, heads, D]
        by_slot = by_slot.index_copy(0, s["slot"], new.double())
        out[name] = by_slot.unflatten(0, (-1, ps)).transpose(1, 2)
    return out


def _exact_qkn(s):
    case = s["case"]
    T, hq, hkv, D, rot = case["T"], case["hq"], case["hkv"], case["D"], case["rot"]
    half = rot // 2
    x = s["qkv"].detach().double()
    pos = s["pos"].view(-1, T)
    row = torch.zeros(half, dtype=torch.int64, device=DEV) if s["axes"] is None else s["axes"].long()
    freq = torch.arange(half, device=DEV)
    # the rotation as complex numbers: pair f of token t turns by cos + i sin
    turn = torch.complex(s["table"].double()[pos[row].t(), freq], s["table"].double()[pos[row].t(), half + freq])[:, None]
    i0, i1 = (2 * freq, 2 * freq + 1) if case["interleaved"] else (freq, half + freq)

    def rotate(y, t):
        z = torch.complex(y[..., i0], y[..., i1]) * t
        y = y.clone()
        y[..., i0], y[..., i1] = z.real, z.imag
        return y

    out, dx, dws = {}, torch.zeros_like(x), []
    for name, h0, h1, w, sc in (("q", 0, hq, s["qw"], case["q_scale"]), ("k", hq, hq + hkv, s["kw"], 1.0)):
        xs = x[:, h0:h1]
        gain = torch.ones(D, dtype=torch.float64, device=DEV) if w is None else w.detach().double() + case["gain"]
        r = 1.0 / torch.sqrt(xs.square().sum(-1, keepdim=True) / D + 1e-6)
        out[name] = rotate(xs * r * gain * sc, turn)
        if case["grad"]:
            dn = rotate(s["dout"][0 if name == "q" else 1].double(), turn.conj())
            gl = dn * gain * sc
            dx[:, h0:h1] = gl * r - xs * r.pow(3) * ((gl * xs).sum(-1, keepdim=True) / D)
            dws.append((dn * xs * r * sc).sum((0, 1)))
    if case["grad"]:
        dx[:, hq + hkv:] = s["dout"][2].double()
        out["dqkv"] = dx
        if case["weights"]:
            out["dqw"], out["dkw"] = dws
    return out


def _exact_attn(s):
    case = s["case"]
    hq, hkv, D, ps = case["hq"], case["hkv"], case["D"], s["ps"]
    G = hq // hkv
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    r = 0
    for b in range(len(s["cached"])):
        for i in range(s["new"][b]):
            last = s["cached"][b] + i
            first = max(0, last - case["window"] + 1) if case["window"] else 0
            j = torch.arange(first, last + 1, device=DEV)
            page, off = s["table"][b].long()[j // ps], j % ps
            k, v = s["kp"][page, :, off].double(), s["vp"][page, :, off].double()                      # [keys, hkv, D]
            z = torch.einsum("hgd,jhd->hgj", s["q"][r].double().view(hkv, G, D), k) * s["scale"]
            if s["sinks"] is not None:
                z = torch.cat([z, s["sinks"].double().view(hkv, G, 1)], -1)
            p = torch.softmax(z, -1)[..., :j.numel()]
            out[r] = torch.einsum("hgj,jhd->hgd", p, v).reshape(hq, D)
            r += 1
    return out
