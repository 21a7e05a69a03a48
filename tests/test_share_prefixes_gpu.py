"""Requests that begin alike through the engine: the pages of a common beginning are held once, attention reads them once, and the logits are
those of requests that share nothing."""
import pytest
import torch

from conftest import TINY, tokens_for

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def small_groups_too(monkeypatch):
    """Models this small never spare enough keys for the kernels to be chosen."""
    from lucciola_b200.engine import step
    monkeypatch.setattr(step, "SHARED_ELEMENTS", 0)


def engine(folder, name, **kw):
    from lucciola_b200 import Engine, EngineOptions
    kw = dict(max_blocks=400, block_size=TINY[name][4], max_num_seqs=40, **kw)
    return Engine(folder, options=EngineOptions(**kw))


def answers(eng, prompts, params):
    out = eng.generate(prompts, params)
    return out, eng.stats()


@pytest.mark.parametrize("name", ["A", "B"])
@pytest.mark.parametrize("graph", [True, False])
def test_float32_answers_are_those_of_requests_that_share_nothing(tiny_models, name, graph):
    """Eight draws and greedy answers behind one prompt, two behind a part of it, one of its own: the same tokens.  (A draw or a largest
    logit could only differ where two scores are within the rounding of 32-bit sums of each other, which no token here comes near.)"""
    from lucciola_b200 import SamplingParams
    prompt = tokens_for(name, 70, 3)
    half = prompt[:40]
    prompts = [prompt] * 8 + [half + tokens_for(name, 5, 4), half + tokens_for(name, 9, 5), tokens_for(name, 17, 6)]
    params = [SamplingParams(max_new_tokens=20, ignore_eos=True, temperature=0.8 if i % 3 else 0.0, seed=i, top_p=0.9, top_k=40 if i % 2 else 0)
              for i in range(len(prompts))]
    alone, stats = answers(engine(tiny_models[name], name, dtype="float32", use_cuda_graph=graph), prompts, params)
    assert stats["shared_tokens"] == 0
    eng = engine(tiny_models[name], name, dtype="float32", use_cuda_graph=graph, share_prefixes=True)
    together, stats = answers(eng, prompts, params)
    page = TINY[name][4]
    assert stats["shared_tokens"] == 7 * (69 // page * page) + 2 * (40 // page * page)
    assert together == alone
    eng.runner.manager.check_invariants()
    assert stats["free_pages"] == 400


def logits_of(folder, name, share, prompt, tails, dtype):
    """Prompt, then every request's tail, then three decoded tokens each: the wanted logits of all steps."""
    from lucciola_b200 import EngineOptions
    from lucciola_b200.engine.load import build_runner
    from lucciola_b200.engine.step import StepEntry
    r = build_runner(folder, EngineOptions(dtype=dtype, block_size=TINY[name][4], max_blocks=300, max_num_seqs=24, share_prefixes=share))
    out = [r.step([StepEntry(0, prompt, (len(prompt) - 1,))]).clone()]
    pages = (len(prompt) - 1) // TINY[name][4]
    at = pages * TINY[name][4]
    for i in range(1, len(tails)):
        if share:
            r.manager.admit(i)
            r.manager.share_prefix(i, 0, pages)
    first = [StepEntry(0, tails[0], (len(tails[0]) - 1,))]
    first += [StepEntry(i, (prompt[at:] if share else prompt) + t, (len((prompt[at:] if share else prompt) + t) - 1,)) for i, t in enumerate(tails) if i]
    out.append(r.step(first).clone())
    for k in range(3):
        out.append(r.step([StepEntry(i, [7 * k + i], (0,)) for i in range(len(tails))]).clone())
    return torch.cat(out).double().cpu(), r


@pytest.mark.parametrize("name", ["A", "B", "D"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_logits_beside_those_of_requests_that_share_nothing(tiny_models, name, dtype):
    """The two ways differ by the order of sums, and in bfloat16 by roundings of weights and results that fall differently: a relative 2^-8
    each in a layer of two or three; float32: 2^-24 times the few hundred terms of a sum."""
    prompt = tokens_for(name, 100 if name != "A" else 70, 1)
    tails = [tokens_for(name, n, n) for n in (1, 2, 5, 20, 1, 1, 3)]
    a, _ = logits_of(tiny_models[name], name, False, prompt, tails, dtype)
    b, r = logits_of(tiny_models[name], name, True, prompt, tails, dtype)
    off = (a - b).norm() / a.norm()
    assert off <= (2 ** -15 if dtype == "float32" else 6 * 2 ** -8), float(off)


def test_shared_attention_is_what_runs(tiny_models):
    """Steps with groups launch the shared kernels, one plan for all layers; recordings of steps with and without groups lie side by side."""
    from lucciola_b200 import ops
    from lucciola_b200 import SamplingParams
    calls = {"plan": 0, "attention": 0}
    plan, attention = ops.shared_plan, ops.attention_shared

    def counted(kind, f):
        def g(*a, **k):
            calls[kind] += 1
            return f(*a, **k)
        return g
    eng = engine(tiny_models["D"], "D", share_prefixes=True)
    ops.shared_plan, ops.attention_shared = counted("plan", plan), counted("attention", attention)
    try:
        eng.generate([tokens_for("D", 130, 1)] * 6, SamplingParams(max_new_tokens=8, ignore_eos=True))
    finally:
        ops.shared_plan, ops.attention_shared = plan, attention
    layers = TINY["D"][0]["num_hidden_layers"]
    assert calls["plan"] > 0 and calls["attention"] == layers * calls["plan"]
    assert eng.runner.graph_replays > 0
    assert ops.device_error() == 0


def test_under_page_pressure(tiny_models):
    """Preemptions while pages are shared: the same tokens, and every page comes back."""
    from lucciola_b200 import Engine, EngineOptions, SamplingParams
    prompts = [tokens_for("B", 60, 2)] * 6 + [tokens_for("B", 50, 3)] * 3
    params = SamplingParams(max_new_tokens=40, ignore_eos=True)
    want = Engine(tiny_models["B"], options=EngineOptions(dtype="float32", block_size=8, max_blocks=400, max_num_seqs=16)).generate(prompts, params)
    eng = Engine(tiny_models["B"], options=EngineOptions(dtype="float32", block_size=8, max_blocks=36, max_num_seqs=16, share_prefixes=True))
    assert eng.generate(prompts, params) == want
    assert eng.stats()["preemptions"] > 0 and eng.stats()["free_pages"] == 36
    eng.runner.manager.check_invariants()


def test_a_model_with_windows_refuses(tiny_models):
    with pytest.raises(ValueError, match="share_prefixes"):
        engine(tiny_models["C"], "C", share_prefixes=True)


def test_groups_that_spare_little_take_the_ordinary_kernels(tiny_models, monkeypatch):
    """The pages are held once all the same, and the tokens are those of requests that share nothing."""
    from lucciola_b200 import SamplingParams, ops
    from lucciola_b200.engine import step
    monkeypatch.setattr(step, "SHARED_ELEMENTS", 1 << 24)
    called = []
    plan = ops.shared_plan
    monkeypatch.setattr(ops, "shared_plan", lambda *a: called.append(1) or plan(*a))
    prompts = [tokens_for("D", 100, 3)] * 4
    params = SamplingParams(max_new_tokens=12, ignore_eos=True)
    eng = engine(tiny_models["D"], "D", dtype="bfloat16", share_prefixes=True)
    eng.generate(prompts, params)
    assert not called and eng.stats()["shared_tokens"] > 0


def test_long_portions_stay_with_their_kernel(tiny_models):
    from types import SimpleNamespace as N
    from lucciola_b200.parts.attention import SHARED_PORTION, GQAttention
    part = N(num_heads=8, num_kv_heads=2, head_dim=128, window=0, scale=0.1, plan_key=lambda: ("attention tiles", 4))
    takes = lambda tokens, dim=128, page=16, dtype=torch.bfloat16, of=True, seqs=4: GQAttention._attend_shared(
        N(**{**vars(part), "head_dim": dim}), torch.empty(tokens, 8, dim, dtype=dtype, device="cuda"),
        N(prefix_of=of or None, num_seqs=seqs, max_q_len=tokens), N(page_size=page))
    assert takes(1) and takes(SHARED_PORTION) and not takes(SHARED_PORTION + 1)
    assert takes(SHARED_PORTION + 1, dim=64)                 # no other kernel for such heads but the mma.sync ones
    assert not takes(1, dim=96) and not takes(1, page=12)    # bfloat16 that the tensor-core kernel does not take
    assert takes(1, dim=256) and takes(1, dim=96, dtype=torch.float32)
    assert not takes(1, of=False) and not takes(1, seqs=513)
