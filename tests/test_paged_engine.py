"""The operators of the paged cache and of the one-pass query / key norms as the models and the generation engine use them."""

import asyncio

import pytest
import torch

from torchtitan_b200.experiments.rl import CachedGenerator, GenerationEngine, SamplingConfig
from torchtitan_b200.models import get_model_spec
from torchtitan_b200.models.common.attention import AttentionContext, PagedKVCache
from torchtitan_b200.ops import functional as OF


def _model(name, flavor, layers=2, seed=0):
    spec = get_model_spec(name, flavor.split(":")[0])
    if flavor.endswith(":hd64"):                      # the debug model with heads of the kernels' smallest width
        from torchtitan_b200.models.gpt_oss import build_gpt_oss_config

        spec.model = build_gpt_oss_config(dim=256, n_layers=4, n_heads=8, n_kv_heads=2, head_dim=64, moe_hidden_dim=256,
                                          num_experts=8, top_k=4, vocab_size=2048)
    spec.model.layers = spec.model.layers[:layers]
    spec.model.n_layers = len(spec.model.layers)
    model = spec.model.build()
    model.init_states(seed=seed)
    return model


def _run(coro):
    return asyncio.run(asyncio.wait_for(coro, timeout=120))


def _paged(**kw):
    kw = {"threaded": False, "kv_cache": "paged", "kv_page_size": 16, "kv_cache_tokens": 1024, **kw}
    return GenerationEngine.Config(**kw)


async def _generate(eng, prompts, sampling):
    outs = await asyncio.gather(*(eng.generate(p, request_id=f"r{i}", sampling_config=sampling) for i, p in enumerate(prompts)))
    await eng.close()
    return outs


def _all_pages_back(cache):
    return sorted(cache._free) == list(range(cache.num_pages)) and not any(cache._refs) and not cache._pages and not cache._index


@pytest.fixture
def fused():
    OF.settings.qk_norm_rope = "fused"
    yield
    OF.settings.qk_norm_rope = "separate"


@pytest.mark.parametrize("name,flavor,layers", [("llama3", "debugmodel", 2), ("qwen3", "debugmodel", 2), ("gpt_oss", "debugmodel", 2),
                                                ("muse_glimmer", "debugmodel", 4), ("qwen3_5", "debugmodel", 4)])
def test_paged_engine_matches_single_sequence_decoding(name, flavor, layers):
    """Prompts of one token up to several pages, two with the same leading pages; greedy tokens and log-probabilities equal
    those of the one-sequence generator."""
    model = _model(name, flavor, layers)
    base = [(7 * i) % 200 + 1 for i in range(37)]
    prompts = [base, [9], base[:32] + [3, 4], base[:33], [5, 6, 7] * 11]
    want = [CachedGenerator(model, temperature=0.0).generate(torch.tensor(p), 5) for p in prompts]
    eng = GenerationEngine(_paged(max_num_seqs=4), model=model)
    outs = _run(_generate(eng, prompts, SamplingConfig(temperature=0.0, max_tokens=5)))
    for got, w in zip(outs, want):
        assert got.token_ids == w.response.tolist()
        assert torch.allclose(torch.tensor(got.token_logprobs), w.logprobs, atol=1e-4)
    assert _all_pages_back(eng._paged)


def test_samples_of_one_prompt_compute_its_pages_once():
    model = _model("llama3", "debugmodel")
    rows = []
    forward = model.forward

    def spy(tokens, positions, ctx=None, **kw):
        rows.append(tokens.numel())
        return forward(tokens, positions, ctx, **kw)

    model.forward = spy
    prompt = [(3 * i) % 100 + 1 for i in range(40)]
    outs = {}
    for share in (True, False):
        rows.clear()
        eng = GenerationEngine(_paged(share_prefixes=share), model=model)
        outs[share] = _run(_generate(eng, [prompt] * 6, SamplingConfig(temperature=0.0, max_tokens=4)))
        assert rows[0] == (40 + 5 * 8 if share else 6 * 40) and rows[1:] == [6] * 3      # 32 of the 40 tokens lie in whole pages
        assert _all_pages_back(eng._paged)
    for a, b in zip(outs[True], outs[False]):
        assert a.token_ids == b.token_ids
        assert torch.allclose(torch.tensor(a.token_logprobs), torch.tensor(b.token_logprobs), atol=1e-4)


def test_a_small_pool_makes_requests_wait_and_weights_end_the_sharing():
    model = _model("llama3", "debugmodel")
    prompt = list(range(1, 36))
    greedy = SamplingConfig(temperature=0.0, max_tokens=9)
    want = CachedGenerator(model, temperature=0.0).generate(torch.tensor(prompt), 9).response.tolist()

    async def go():
        eng = GenerationEngine(_paged(kv_cache_tokens=64, share_prefixes=False), model=model)         # one request at a time
        outs = await _generate(eng, [prompt] * 3, greedy)
        assert all(o.token_ids == want for o in outs) and eng.steps == 27 and _all_pages_back(eng._paged)
        eng = GenerationEngine(_paged(), model=model)
        first = asyncio.create_task(eng.generate(prompt, request_id="a", sampling_config=greedy))
        await asyncio.sleep(0)
        await asyncio.sleep(0)
        assert eng._paged.shared_tokens(prompt) == 32
        await eng.pull_model_state_dict(1)
        assert eng._paged.shared_tokens(prompt) == 0                                                  # computed under other weights
        second = await eng.generate(prompt, request_id="b", sampling_config=greedy)
        assert (await first).token_ids == second.token_ids == want
        with pytest.raises(ValueError, match="paged cache holds"):
            small = GenerationEngine(_paged(kv_cache_tokens=32), model=model)
            await small.generate(prompt, request_id="c", sampling_config=greedy)
        # a request that reaches the pool's length ends there
        eng2 = GenerationEngine(_paged(kv_cache_tokens=48), model=model)
        done = await eng2.generate(prompt, request_id="d", sampling_config=SamplingConfig(temperature=0.0, max_tokens=100))
        assert done.finish_reason == "length" and len(done.token_ids) == 48 - 35 + 1 and done.token_ids[:9] == want
        await eng.close()
        await eng2.close()
        assert _all_pages_back(eng._paged) and _all_pages_back(eng2._paged)

    _run(go())


def test_a_failed_step_gives_all_pages_back():
    model = _model("llama3", "debugmodel")

    async def go():
        eng = GenerationEngine(_paged(), model=model)
        with pytest.raises(RuntimeError, match="generation failed"):
            await eng.generate([1, 5000], request_id="bad", sampling_config=SamplingConfig(temperature=0.0, max_tokens=2))
        assert _all_pages_back(eng._paged)
        ok = await eng.generate([5, 6], request_id="good", sampling_config=SamplingConfig(temperature=0.0, max_tokens=3))
        assert len(ok.token_ids) == 3
        await eng.close()

    _run(go())


def test_paged_cache_refusals():
    with pytest.raises(ValueError, match="grouped-query layers"):
        PagedKVCache.for_model(_model("deepseek_v3", "debugmodel"), tokens=64, max_seqs=2, max_length=64, device="cpu")
    kw = dict(tokens=64, max_seqs=2, max_length=64, device="cpu")
    with pytest.raises(ValueError, match="page size"):
        PagedKVCache((4, 2), (0,), page_size=48, **kw)
    cache = PagedKVCache((4, 2), (0,), page_size=16, **kw)
    with pytest.raises(ValueError, match="prompt"):
        cache.add(list(range(65)), 1)
    slot, cached = cache.add(list(range(20)), 100)                    # the whole pool
    assert cached == 0 and not cache.can_add([1], 1)
    with pytest.raises(RuntimeError, match="full"):
        cache.add([1], 1)
    with pytest.raises(RuntimeError, match="reserved"):
        cache.begin_step([slot], [65])
    cache.release(slot)
    assert _all_pages_back(cache)


def test_prefix_entries_outlive_their_first_holder():
    cache = PagedKVCache((4, 2), (0,), tokens=256, max_seqs=4, max_length=128, page_size=16, device="cpu")
    prompt = list(range(40))
    a, n0 = cache.add(prompt, 5)
    b, n1 = cache.add(prompt + [7], 5)
    assert (n0, n1) == (0, 32) and cache._pages[a][:2] == cache._pages[b][:2] and cache.group_of(a) == cache.group_of(b)
    shared = cache._pages[a][:2]
    cache.release(a)
    assert not set(shared) & set(cache._free)                         # still held by the second sequence
    c, n2 = cache.add(prompt, 5)
    assert n2 == 32 and cache._pages[c][:2] == shared
    cache.release(b)
    cache.release(c)
    assert _all_pages_back(cache) and cache.add(prompt, 5)[1] == 0


# ------------------------------------------------------------------------------------------- query / key norms in the models
@pytest.mark.parametrize("name,flavor,layers", [("qwen3", "debugmodel", 2), ("muse_glimmer", "debugmodel", 4), ("qwen3_5", "debugmodel", 4),
                                                ("qwen3_5", "debugmodel_vl", 4)])
def test_fused_norms_give_the_separate_kernels_results(name, flavor, layers):
    """fp32 on the CPU: loss and every gradient, with three-axis positions on the vision-language flavor."""
    out = {}
    calls = []
    real = OF.qk_norm_rope
    for mode in ("separate", "fused"):
        model = _model(name, flavor, layers)
        OF.settings.qk_norm_rope = mode
        OF.qk_norm_rope = lambda *a, **k: (calls.append(mode), real(*a, **k))[1]
        try:
            g = torch.Generator().manual_seed(0)
            tokens = torch.randint(0, 300, (24,), generator=g)
            pos = torch.arange(24) % 13
            ctx = AttentionContext()
            if flavor.endswith("vl"):
                ctx.rope_positions = torch.stack([pos, (pos * 2) % 11, (pos * 3) % 7])
                body = model
                h = type(model).__mro__[1].forward(body, tokens, pos, ctx)
            else:
                h = model(tokens, pos, ctx)
            loss = h.float().square().mean()
            loss.backward()
        finally:
            OF.settings.qk_norm_rope, OF.qk_norm_rope = "separate", real
        out[mode] = (loss.detach(), {n: p.grad.clone() for n, p in model.named_parameters() if p.grad is not None})
    assert set(calls) == {"fused"}
    (l0, g0), (l1, g1) = out["separate"], out["fused"]
    assert abs(float(l0 - l1)) <= 1e-5 * abs(float(l0)) and g0.keys() == g1.keys()
    for n in g0:
        assert (g0[n] - g1[n]).abs().max() <= 1e-4 * g0[n].abs().max() + 1e-7, n


def test_the_switch_is_a_config_field():
    from torchtitan_b200.config import ConfigManager

    cfg = ConfigManager().parse_args(["--module", "qwen3", "--config", "qwen3_debugmodel", "--kernels.qk_norm_rope", "fused"])
    assert cfg.kernels.qk_norm_rope == "fused"


# ------------------------------------------------------------------------------------------------------------ on the GPU
@pytest.mark.gpu
@pytest.mark.parametrize("name,flavor,layers", [("qwen3", "debugmodel", 2), ("llama3", "debugmodel_hd128", 2), ("gpt_oss", "debugmodel", 2),
                                                ("gpt_oss", "debugmodel:hd64", 2), ("qwen3_5", "debugmodel", 4)])
def test_generation_on_the_kernels(name, flavor, layers, fused):
    """bf16 on the kernels: plan, norms, page writes and attention together, as the engine runs them.  Every sampled token's
    log-probability against one uncached pass over the finished sequence (two bf16 paths through a few layers: logits of
    order one differ by some 2^-8 of themselves per layer)."""
    from torchtitan_b200.experiments.rl.engine import place_model_

    model = place_model_(_model(name, flavor, layers), "cuda", torch.bfloat16)
    base = [(7 * i) % 200 + 1 for i in range(150)]
    prompts = [base, base, base[:128] + [3], [9], base[:77], base]
    eng = GenerationEngine(_paged(kv_page_size=64, kv_cache_tokens=4096), model=model)
    n0 = OF.settings.library_fallbacks
    outs = _run(_generate(eng, prompts, SamplingConfig(temperature=1.0, top_k=0, max_tokens=6, seed=3)))
    if flavor in ("debugmodel_hd128", "debugmodel:hd64") or name == "qwen3":        # head dimensions of the attention kernels
        assert OF.settings.library_fallbacks == n0
    assert _all_pages_back(eng._paged)
    with torch.no_grad():
        for p, o in zip(prompts, outs):
            ids = torch.tensor(p + o.token_ids, device="cuda")
            logits = model(ids, torch.arange(ids.numel(), device="cuda"))[len(p) - 1:-1].float()
            want = torch.log_softmax(logits, -1).gather(1, ids[len(p):, None])[:, 0]
            assert (want.cpu() - torch.tensor(o.token_logprobs)).abs().max() < 0.1


@pytest.mark.gpu
def test_training_step_with_the_fused_norms(fused):
    """A qwen3 step on the kernels with the norms fused: loss and gradients of the fp32 CPU model within bf16 noise."""
    losses, grads = [], []
    for device in ("cpu", "cuda"):
        model = _model("qwen3", "debugmodel")
        model = model.to(device)
        if device == "cuda":
            for p in model.parameters():
                p.data = p.data.bfloat16()
        tokens = torch.randint(0, 300, (256,), generator=torch.Generator().manual_seed(0)).to(device)
        loss = model(tokens, torch.arange(256, device=device)).float().logsumexp(-1).mean()
        loss.backward()
        losses.append(float(loss.detach()))
        grads.append({n: p.grad.float().cpu() for n, p in model.named_parameters() if "_norm" in n and "layers" in n})
    assert abs(losses[0] - losses[1]) <= 2e-2 * abs(losses[0])
    for n, g in grads[0].items():
        assert (grads[1][n] - g).norm() <= 0.1 * g.norm() + 1e-6, n


# --------------------------------------------------------------------------------------------------- batch-invariant mode
def test_batch_invariant_mode_refuses_the_paged_cache():
    from torchtitan_b200.experiments.rl import batch_invariant, config_registry

    model = _model("llama3", "debugmodel")
    with batch_invariant():
        with pytest.raises(ValueError, match="batch-invariant"):
            GenerationEngine(_paged(), model=model)
        GenerationEngine(GenerationEngine.Config(threaded=False), model=model)
    GenerationEngine(_paged(), model=model)
    cfg = config_registry.rl_grpo_qwen3_0_6b_alphabet_sort_batch_invariant()
    cfg.validate()
    cfg.generator.kv_cache = "paged"
    with pytest.raises(ValueError, match="contiguous"):
        cfg.validate()
    cfg.trainer.debug.batch_invariant = False
    cfg.validate()


@pytest.mark.gpu
def test_batch_invariant_mode_refuses_paged_attention():
    from torchtitan_b200.experiments.rl import batch_invariant
    from torchtitan_b200.ops import paged

    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    kp = torch.zeros(2, 2, 16, 64, device="cuda", dtype=torch.bfloat16)
    q = torch.zeros(1, 4, 64, device="cuda", dtype=torch.bfloat16)
    plan = paged.page_plan(i32([3]), i32([1]), i32([[0]]), i32([0]), i32([]), 16, 1, num_pages=2, mapped=i32([1]), n_heads=4, n_kv_heads=2)
    with batch_invariant(), pytest.raises(RuntimeError, match="batch-invariant"):
        paged.attention(q, kp, kp, plan, 0.1)
    paged.attention(q, kp, kp, plan, 0.1)


# ------------------------------------------------------------------------------------- groups and their workspace in a step
def _step_plan(cache, slots, rows):
    cache.begin_step(slots, rows)
    plan = cache.plan
    cache.end_step()
    return plan


def test_a_step_that_shares_nothing_has_no_groups():
    """Workspace for rows of sharing groups is there for those rows only: not in a step whose sequences are alone, not in the step
    that computes a prefix, and not for a long prompt beside a group."""
    kw = dict(tokens=2048, max_seqs=8, max_length=1024, page_size=16, device="cpu")
    prompt = list(range(40))
    for share in (True, False):
        cache = PagedKVCache((4, 2), (0,), share_prefixes=share, **kw)
        a, b = (cache.add(p, 20)[0] for p in (prompt, [7] * 35))
        plan = _step_plan(cache, [a, b], [40, 35])
        assert (plan.groups, plan.shared_rows, plan.max_rows) == (0, 0, 40)
        c, n = cache.add(prompt + [9], 20)
        assert n == (32 if share else 0)
        plan = _step_plan(cache, [a, c, b], [1, 41 - n, 1])
        assert (plan.groups, plan.shared_rows) == ((2, 10) if share else (0, 0)) and plan.max_rows == (10 if share else 41)
    cache = PagedKVCache((4, 2), (0,), **kw)
    (a, _), (b, n) = cache.add(prompt, 20), cache.add(prompt, 20)
    assert _step_plan(cache, [a, b], [40, 40 - n]).groups == 0            # the prefix is among the new rows of this step
    long, _ = cache.add([5] * 700, 20)
    plan = _step_plan(cache, [long, a, b], [700, 1, 1])
    assert (plan.groups, plan.shared_rows, plan.max_rows) == (2, 2, 700)
    other, _ = cache.add([6] * 50, 20)
    plan = _step_plan(cache, [a, b, long, other], [1, 1, 1, 50])
    assert (plan.groups, plan.shared_rows) == (2, 2)                      # the two single sequences are one group without a prefix
    plan = _step_plan(cache, [a, b, long], [1, 0, 1])                     # one member of the group waits this step out
    assert (plan.groups, plan.shared_rows) == (0, 0)


# -------------------------------------------------------------------------------------------------- flags of a step's kernels
def test_flags_are_taken_on_the_models_device(monkeypatch):
    """An engine on another GPU than the current one looks at that GPU's flags, and leaves those of others alone."""
    from contextlib import contextmanager
    from types import SimpleNamespace

    from torchtitan_b200.ops import ext

    at, asked, bits = [None], [], [0]

    @contextmanager
    def device(d):
        at[0] = d
        yield
        at[0] = None

    def take(mask):
        asked.append((at[0], mask))
        return bits[0] & mask

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(ext, "require", lambda: SimpleNamespace(take_status=take))
    eng = GenerationEngine(_paged(), model=_model("llama3", "debugmodel"))
    dev = torch.device("cuda:1")
    for bits[0], said in ((15, None), (16, "out of range"), (32, "wait"), (63, "out of range")):
        if said:
            with pytest.raises(RuntimeError, match=said):
                eng._check_pages(dev)
        else:
            eng._check_pages(dev)
    assert asked == [(dev, 48)] * 4


@pytest.mark.gpu
def test_flags_are_read_behind_the_stream_of_the_step():
    """Bad pages of a step on a side stream that is still at work, beside a flag of somebody else."""
    from torchtitan_b200.experiments.rl.engine import place_model_
    from torchtitan_b200.ops import ext, paged

    ops = ext.require()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    args = (i32([0]), i32([1]), i32([[0]]), i32([0]), i32([7]), 16, 1)              # page 7 of a pool of two
    eng = GenerationEngine(_paged(), model=place_model_(_model("llama3", "debugmodel"), "cuda", torch.bfloat16))
    dev = torch.device("cuda")
    ops.status(True)
    OF.rope(torch.zeros(1, 1, 64, device="cuda"), torch.zeros(4, 64, device="cuda"), torch.tensor([9], device="cuda"), False)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)                                               # some 25 ms
        paged.page_plan(*args, num_pages=2)
        with pytest.raises(RuntimeError, match="out of range"):
            eng._check_pages(dev)
        eng._check_pages(dev)
    assert ops.status(False) == 1 and ops.take_status(15) == 1 and ops.status(True) == 0


def test_more_sequences_than_a_step_takes_are_refused_at_once():
    """Not by the step that first has them all in flight."""
    kw = dict(tokens=64, max_length=64, device="cpu")
    PagedKVCache((4, 2), (0,), max_seqs=4096, **kw)
    with pytest.raises(ValueError, match="4096"):
        PagedKVCache((4, 2), (0,), max_seqs=4097, **kw)


def test_a_failed_pull_ends_the_sharing_too():
    """The weights may be half replaced: later requests compute their prompts themselves."""
    prompt = list(range(1, 40))

    def source(engine):
        raise RuntimeError("half the weights")

    async def go():
        eng = GenerationEngine(_paged(), model=_model("llama3", "debugmodel"), weight_source=source)
        first = asyncio.create_task(eng.generate(prompt, request_id="a", sampling_config=SamplingConfig(temperature=0.0, max_tokens=9)))
        await asyncio.sleep(0)
        await asyncio.sleep(0)
        assert eng._paged.shared_tokens(prompt) == 32
        with pytest.raises(RuntimeError, match="half"):
            await eng.pull_model_state_dict(1)
        assert eng._paged.shared_tokens(prompt) == 0
        await first
        await eng.close()

    _run(go())


def test_training_after_an_evaluation_in_inference_mode(fused):
    """The map of position axes is made once per module; made under inference_mode it could not be saved for a backward."""
    model = _model("qwen3_5", "debugmodel_vl", 4)
    tokens, pos = torch.arange(12), torch.arange(12)

    def run():
        ctx = AttentionContext()
        ctx.rope_positions = torch.stack([pos, pos % 5, pos % 3])
        return type(model).__mro__[1].forward(model, tokens, pos, ctx)

    with torch.inference_mode():
        want = run().clone()
    got = run()
    got.float().square().mean().backward()
    assert torch.equal(got.detach(), want)
    assert all(p.grad is not None for n, p in model.named_parameters() if "q_norm" in n)
