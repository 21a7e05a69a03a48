"""The sampler with top-k, top-p and min-p against its restatement in 64 bits: the tokens are equal, whatever way a row takes through the
kernel (a short list ranked, a border found digit by digit, candidates looked for and rejected)."""
import itertools

import numpy as np
import pytest
import torch

import plain_operators as plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from lucciola_b200 import ops
    return ops


def call(ops, logits, temperature, keys, counters, top_k=None, top_p=None, min_p=None, tokens=None):
    R = logits.shape[0]
    dev = logits.device

    def row(v, dtype):
        if v is None or torch.is_tensor(v):
            return v
        return torch.tensor(np.broadcast_to(np.asarray(v), (R,)).copy(), dtype=dtype, device=dev)
    if tokens is None:
        tokens = torch.full((R,), -7, dtype=torch.int32, device=dev)
    ops.sample(tokens, logits, ops.current_stream(), row(temperature, torch.float32), row(keys, torch.int64), row(counters, torch.int32),
               row(top_k, torch.int32), row(top_p, torch.float32), row(min_p, torch.float32))
    return tokens.tolist()


def numbers(R, seed=0):
    rng = np.random.default_rng(seed)
    return rng.integers(-2 ** 63, 2 ** 63 - 1, R), rng.integers(0, 1000, R)


def check(ops, logits, temperature, top_k, top_p, min_p, seed=0):
    R = logits.shape[0]
    keys, counters = numbers(R, seed)
    # as the kernel gets them: 32-bit numbers
    t, p, m = (np.broadcast_to(np.asarray(v, dtype=np.float32), (R,)) for v in (temperature, top_p, min_p))
    k = np.broadcast_to(np.asarray(top_k), (R,))
    got = call(ops, logits.cuda(), t, keys, counters, k, p, m)
    rows = logits.numpy()
    want = [plain.draw(rows[r], float(t[r]), int(keys[r]), int(counters[r]), int(k[r]), float(p[r]), float(m[r])) for r in range(R)]
    assert got == want


FILTERS = [(1, 1.0, 0.0), (7, 1.0, 0.0), (50, 0.9, 0.0), (256, 1.0, 0.02), (0, 0.9, 0.0), (0, 0.05, 0.0), (0, 0.999, 0.0), (0, 1.0, 0.1),
           (0, 1.0, 1.0), (300, 0.8, 0.01), (257, 1.0, 0.0), (100000, 0.99, 0.0), (0, 0.7, 0.2)]


@pytest.mark.parametrize("vocab", [1, 2, 3, 5, 255, 503, 2047, 8193, 32000, 50003, 151936])
@pytest.mark.parametrize("kind", ["smooth", "flat", "stepped"])
def test_the_token_of_every_filter(ops, vocab, kind):
    R = len(FILTERS)
    x = torch.randn(R, vocab) * 3
    if kind == "flat":
        x = torch.randn(R, vocab) * 0.05
    if kind == "stepped":
        x = x.round()                                  # many equal logits: the lower index comes first
    k, p, m = zip(*FILTERS)
    for T in (0.3, 1.0, 4.0):
        check(ops, x, T, k, p, m, seed=int(T * 10))


@pytest.mark.parametrize("vocab", [64, 1000, 40000])
def test_equal_logits_are_kept_by_index(ops, vocab):
    """All logits equal: top_k keeps the first k indices, top_p = 1/2 the first half (the border falls between two tokens exactly)."""
    x = torch.full((6, vocab), 1.25)
    check(ops, x, 1.0, [3, 300, vocab // 2, 0, 0, 7], [1.0, 1.0, 1.0, 0.5, 0.25, 0.5], 0.0)


@pytest.mark.parametrize("vocab", [9, 4096, 70001])
def test_masked_and_infinite_logits(ops, vocab):
    """-inf, the type's lowest value and NaN in masked places; a row with nothing left; +inf."""
    low = torch.finfo(torch.float32).min
    rows = []
    for fill in (float("-inf"), low, float("nan")):
        for allowed in (1, 3, vocab // 2):
            x = torch.full((vocab,), fill)
            at = torch.randperm(vocab)[:allowed]
            x[at] = torch.randn(allowed) * 2
            rows.append(x)
    x = torch.stack(rows)
    for k, p, m in ((2, 1.0, 0.0), (0, 0.9, 0.0), (0, 1.0, 0.05), (400, 0.95, 0.0), (5, 0.5, 0.5)):
        check(ops, x, 0.8, k, p, m)
    nothing = torch.stack([torch.full((vocab,), float("-inf")), torch.full((vocab,), float("nan")), torch.full((vocab,), low)])
    keys, counters = numbers(3)
    got = call(ops, nothing.cuda(), 1.0, keys, counters, top_p=0.5)
    assert got[:2] == [0, 0]
    assert got[2] == plain.draw(nothing[2].numpy(), 1.0, int(keys[2]), int(counters[2]), top_p=0.5)
    x = torch.randn(1, vocab)
    x[0, vocab - 1] = x[0, vocab // 2] = float("inf")
    assert call(ops, x.cuda(), 1.0, [5], [0], top_k=3) == [vocab // 2]


def test_logits_of_wide_range(ops):
    """One outlier, exponents over the type's whole range, temperatures from tiny to huge."""
    V = 30000
    x = torch.randn(8, V)
    x[0, 17] = 1e30
    x[1, 5] = -3e38
    x[2] = torch.exp2(torch.randint(-120, 120, (V,)).float()) * torch.sign(torch.randn(V))
    x[3] = torch.randn(V) * 1e-6
    x[4] = 1e6 + torch.randn(V)
    x[5, ::2] = -0.0
    x[5, 1::2] = 0.0
    x[6] = -1e4 + torch.arange(V) * 1e-3
    for T in (1e-3, 0.7, 50.0, 1e6):
        for k, p, m in ((20, 1.0, 0.0), (0, 0.9, 0.0), (1000, 0.9, 0.0), (0, 1.0, 0.3)):
            check(ops, x, T, k, p, m, seed=3)


def test_a_row_draws_the_same_in_any_batch(ops):
    """The token depends on the row's own logits, key, counter and filters: alone, among others, at another place, and without filters
    the same as from the sampler that knows none."""
    R, V = 24, 32000
    x = (torch.randn(R, V) * 2).cuda()
    keys, counters = numbers(R)
    k = np.where(np.arange(R) % 4 == 1, 40, 0)
    p = np.where(np.arange(R) % 4 == 2, 0.9, 1.0)
    t = np.where(np.arange(R) % 6 == 5, 0.0, 0.9)
    together = call(ops, x, t, keys, counters, k, p, 0.0)
    alone = [call(ops, x[r:r + 1], t[r:r + 1], keys[r:r + 1], counters[r:r + 1], k[r:r + 1], p[r:r + 1], 0.0)[0] for r in range(R)]
    assert together == alone
    back = list(range(R))[::-1]
    assert call(ops, x.flip(0).contiguous(), t[back].copy(), keys[back].copy(), counters[back].copy(), k[back].copy(), p[back].copy(), 0.0) == together[::-1]
    free = [r for r in range(R) if k[r] == 0 and p[r] == 1.0]
    plain_tokens = call(ops, x, t, keys, counters)
    assert [plain_tokens[r] for r in free] == [together[r] for r in free]


def test_rows_of_a_wider_matrix_and_any_alignment(ops):
    wide = torch.randn(5, 4099) * 2
    for a, n in ((0, 4096), (1, 4001), (3, 4096), (2, 17)):
        view = wide.cuda()[:, a:a + n]
        keys, counters = numbers(5)
        got = call(ops, view, 1.0, keys, counters, top_k=[0, 3, 300, 0, 64], top_p=[0.9, 1.0, 1.0, 0.8, 0.5])
        want = [plain.draw(wide[r, a:a + n].numpy(), 1.0, int(keys[r]), int(counters[r]), [0, 3, 300, 0, 64][r],
                           float(np.float32([0.9, 1.0, 1.0, 0.8, 0.5][r]))) for r in range(5)]
        assert got == want


def test_rows_too_long_for_shared_memory(ops):
    V = 500_000
    x = torch.randn(4, V) * 2
    check(ops, x, 1.0, [30, 0, 5000, 0], [1.0, 0.9, 0.95, 1.0], [0.0, 0.0, 0.0, 0.1])


def test_draws_follow_the_kept_distribution(ops):
    """8192 counters of one row: every kept token's share is within five standard deviations of its probability (the chance that one of
    the nine is not: below 10^-5), and no other token comes."""
    V, n = 400, 8192
    row = torch.randn(V) * 1.5
    p = np.exp(row.double().numpy() / 0.9)
    kept = plain.kept_tokens(row.numpy(), float(np.float32(0.9)), 9, 1.0, 0.0)
    got = np.bincount(call(ops, row.cuda().expand(n, V).contiguous(), 0.9, np.full(n, 77), np.arange(n), top_k=9), minlength=V)
    assert got.sum() == got[kept].sum() == n
    q = p[kept] / p[kept].sum()
    assert (np.abs(got[kept] - n * q) <= 5 * np.sqrt(n * q * (1 - q))).all()


def test_filters_out_of_range_keep_the_first_token(ops):
    """The device's numbers cannot be refused: top_p <= 0 and min_p > 1 keep the likeliest token, top_k beyond the row all of it."""
    x = torch.randn(4, 1000)
    keys, counters = numbers(4)
    got = call(ops, x.cuda(), 1.0, keys, counters, top_k=[0, 0, 5000, -3], top_p=[0.0, 1.0, 1.0, -1.0], min_p=[0.0, 2.0, 0.0, 0.0])
    free = call(ops, x.cuda(), 1.0, keys, counters)
    assert got == [int(x[0].argmax()), int(x[1].argmax()), free[2], int(x[3].argmax())]


def test_replayed_from_a_graph_and_on_another_stream(ops):
    R, V = 5, 32000
    x = torch.randn(R, V, device="cuda") * 2
    keys, counters = (torch.tensor(v, device="cuda") for v in numbers(R))
    counters = counters.int()
    t = torch.full((R,), 0.8, device="cuda")
    k = torch.tensor([0, 20, 500, 0, 3], dtype=torch.int32, device="cuda")
    p = torch.tensor([0.9, 1.0, 0.9, 0.5, 1.0], device="cuda")
    tokens = torch.zeros(R, dtype=torch.int32, device="cuda")
    call(ops, x, t, keys, counters, k, p, tokens=tokens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.sample(tokens, x, ops.current_stream(), t, keys, counters, k, p)
    for step in range(3):
        x.copy_(torch.randn(R, V, device="cuda") * 2)
        counters.add_(1)
        graph.replay()
        replayed = tokens.tolist()
        assert replayed == call(ops, x, t, keys, counters, k, p)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            assert call(ops, x, t, keys, counters, k, p) == replayed


def test_refusals(ops):
    x = torch.randn(3, 64, device="cuda")
    t = torch.ones(3, device="cuda")
    keys, counters = torch.zeros(3, dtype=torch.int64, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    k = torch.full((3,), 4, dtype=torch.int32, device="cuda")
    tokens = torch.zeros(3, dtype=torch.int32, device="cuda")
    s = ops.current_stream()
    for bad in (dict(top_k=k[:2]), dict(top_k=k.long()), dict(top_p=t.double()), dict(min_p=t.cpu()), dict(top_k=k.cpu())):
        with pytest.raises(ops.KernelError):
            ops.sample(tokens, x, s, t, keys, counters, **bad)
    with pytest.raises(ops.KernelError):
        ops.sample(tokens, x.bfloat16(), s, t, keys, counters, top_k=k)
    with pytest.raises(ops.KernelError):
        ops.sample(tokens, x.t(), s, t, keys, counters, top_k=k)
    with pytest.raises(ops.KernelError):
        ops.sample(tokens, x, s, t, None, None, top_k=k)
    with pytest.raises(ops.KernelError):
        ops.sample(tokens.long(), x, s, t, keys, counters, top_k=k)
    with pytest.raises(ops.KernelError):
        ops.sample(tokens, torch.empty(3, 0, device="cuda"), s, t, keys, counters, top_k=k)
    ops.sample(tokens[:0], x[:0], s, t[:0], keys[:0], counters[:0], top_k=k[:0])           # no rows: nothing to do


def test_the_sampler_takes_each_requests_filters(ops):
    from lucciola_b200.sampling.params import SamplingParams
    from lucciola_b200.sampling.sampler import Sampler, sampling_key
    V = 1000
    x = torch.randn(4, V) * 2
    params = [SamplingParams(temperature=0.9, seed=3, top_k=5), SamplingParams(), SamplingParams(temperature=0.7, seed=4),
              SamplingParams(temperature=1.1, seed=5, top_p=0.6, min_p=0.05)]
    got = Sampler(torch.device("cuda:0")).sample(x.cuda(), params, [0, 1, 2, 3])
    want = [plain.draw(x[r].numpy(), float(np.float32(q.temperature)), sampling_key(q.seed), r, q.top_k, float(np.float32(q.top_p)),
                       float(np.float32(q.min_p))) for r, q in enumerate(params)]
    assert got == want


def test_engine_generates_with_filters(ops, tiny_models):
    """Through Engine: top_k = 1 is greedy whatever the seed; a request's tokens do not depend on who shares its steps."""
    from lucciola_b200 import Engine, SamplingParams
    from conftest import TINY, tokens_for
    engine = Engine(tiny_models["D"], max_blocks=64, block_size=TINY["D"][4])
    prompts = [tokens_for("D", n) for n in (5, 17, 33)]
    greedy = engine.generate(prompts, SamplingParams(max_new_tokens=6, ignore_eos=True))
    one = engine.generate(prompts, SamplingParams(max_new_tokens=6, ignore_eos=True, temperature=1.0, seed=9, top_k=1))
    assert one == greedy
    mixed = [SamplingParams(max_new_tokens=6, ignore_eos=True, temperature=1.0, seed=1, top_p=0.8),
             SamplingParams(max_new_tokens=6, ignore_eos=True),
             SamplingParams(max_new_tokens=6, ignore_eos=True, temperature=0.7, seed=2, min_p=0.1, top_k=30)]
    assert engine.generate(prompts, mixed)[1] == greedy[1]


@pytest.mark.parametrize("vocab", [4097, 20011, 70001])
def test_a_row_draws_the_same_among_many(ops, vocab):
    """Batches so large that a row has fewer and fewer CTAs."""
    gen = torch.Generator().manual_seed(vocab)
    rows = 6
    x = (torch.randn(rows, vocab, generator=gen) * 2).cuda()
    t, keys = torch.tensor([0.7, 1.0, 1.3, 0.9, 1.0, 0.0]).cuda(), torch.arange(rows).cuda()
    counters, k = torch.arange(rows, dtype=torch.int32).cuda(), torch.tensor([0, 40, 0, vocab // 3, 0, 5], dtype=torch.int32).cuda()
    p, m = torch.tensor([0.95, 0.9, 1.0, 0.999, 0.5, 0.9]).cuda(), torch.tensor([0.0, 0.01, 0.02, 0.0, 0.0, 0.0]).cuda()
    draws = []
    for times in (1, 5, 10, 25, 60, 120):
        out = torch.full((rows * times,), -1, dtype=torch.int32, device="cuda")
        many = [a.repeat(times) for a in (t, keys, counters, k, p, m)]
        ops.sample(out, x.repeat(times, 1), ops.current_stream(), *many[:3], top_k=many[3], top_p=many[4], min_p=many[5])
        draws.append(out.view(times, rows))
    assert all(torch.equal(d, draws[0].expand_as(d)) for d in draws)
