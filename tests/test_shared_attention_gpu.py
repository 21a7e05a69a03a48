"""Attention of requests that share prefixes against its restatement in 64 bits.

Tolerances.  float32: sums of up to a few hundred products in 32 bits; a score is off by less than 2^-20 (|q . k| scale is a few), a weight
as much relatively, a result (a mean of values of size 1 to 4) by less than 2^-18.  bfloat16: the same where the products run on the ordinary
pipes; on the tensor cores each weight is rounded to bfloat16, by at most half a step, 2^-8 of itself, so the mean of values |v| <= V moves by
at most 2^-8 V (and its denominator, summed before the rounding, not at all); and the output is rounded once, by at most 2^-8 of itself, also
V at most.  Together 2^-7 V, and 2^-18."""
import random

import pytest
import torch

import plain_operators as plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from lucciola_b200 import ops
    return ops


class Batch:
    """Requests with pages of their own and of their groups; every page slot that no request's keys lie in is NaN."""

    def __init__(self, heads, kv_heads, dim, page, requests, groups, dtype, extra_rows=0, spare=3):
        """requests: (group or -1, new tokens, length); groups: prefix length.  The first page of a request's own part holds the end of
        a prefix that is no whole number of pages too (a copy, as a cache would make one)."""
        rng = random.Random(7)
        S = len(requests)
        self.heads, self.kv_heads, self.dim, self.page, self.dtype = heads, kv_heads, dim, page, dtype
        need = [-(-n // page) for _, _, n in requests]
        total = sum(need) + sum(-(-p // page) for p in groups) + spare
        ids = list(range(total))
        rng.shuffle(ids)
        k = torch.full((total, kv_heads, page, dim), float("nan"))
        v = k.clone()
        self.table = torch.full((S, max(max(need), 1) + 2), -1, dtype=torch.int32)
        common = [(torch.randn(p, kv_heads, dim), torch.randn(p, kv_heads, dim), [ids.pop() for _ in range(-(-p // page))]) for p in groups]
        leader, self.prefix_of, self.prefix_lens = {}, [-1] * S, [0] * S
        self.cu, self.ctx = [0], [n for _, _, n in requests]
        for kk, vv, pages in common:
            for j in range(kk.shape[0]):
                k[pages[j // page], :, j % page] = kk[j]
                v[pages[j // page], :, j % page] = vv[j]
        for s, (g, new, n) in enumerate(requests):
            whole = groups[g] // page if g >= 0 else 0           # pages shared outright
            row = (common[g][2][:whole] if g >= 0 else [])
            row = row + [ids.pop() for _ in range(max(need[s] - len(row), 0))]
            self.table[s, :len(row)] = torch.tensor(row, dtype=torch.int32)
            for j in range(whole * page, n):
                mine = torch.randn(2, kv_heads, dim)
                if g >= 0 and j < groups[g]:
                    mine = torch.stack([common[g][0][j], common[g][1][j]])
                k[row[j // page], :, j % page], v[row[j // page], :, j % page] = mine
            if g >= 0:
                self.prefix_of[s] = leader.setdefault(g, s)
                self.prefix_lens[self.prefix_of[s]] = groups[g]
            self.cu.append(self.cu[-1] + new)
        self.T = self.cu[-1] + extra_rows
        self.q = torch.randn(self.T, heads, dim).to(dtype)
        self.k, self.v = k.to(dtype), v.to(dtype)
        self.max_new = max(r[1] for r in requests)
        self.scale = dim ** -0.5

    def device(self):
        ints = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (self.cu, self.ctx, self.prefix_of, self.prefix_lens)]
        return [self.q.cuda(), self.k.cuda(), self.v.cuda(), self.table.cuda()] + ints

    def launch(self, ops, dev, out, stream=None):
        q, k, v, table, cu, ctx, of, lens = dev
        ops.attention_shared(q, out, k, v, table, cu, ctx, of, lens, self.max_new, self.heads, self.kv_heads, self.dim, self.page, self.scale,
                             stream if stream is not None else ops.current_stream())
        return out

    def want(self):
        return plain.shared_attention(self.q, self.k, self.v, self.table, self.cu, self.ctx, self.prefix_of, self.prefix_lens, self.scale)

    def compare(self, got, want=None):
        want = self.want() if want is None else want
        n = self.cu[-1]
        got, want = got[:n].double().cpu(), want[:n]
        top = float(self.v[~self.v.isnan()].abs().max())
        off = 2 ** -18 * max(top, 1) + (2 ** -7 * top if self.dtype == torch.bfloat16 else 0)
        assert got.isfinite().all()
        assert (got - want).abs().max() <= off

    def check(self, ops):
        dev = self.device()
        got = self.launch(ops, dev, torch.full_like(dev[0], float("nan")))
        self.compare(got)
        return got


LAYOUTS = [(8, 2, 128, 16, torch.bfloat16), (8, 2, 64, 16, torch.bfloat16), (10, 2, 128, 8, torch.bfloat16), (4, 4, 128, 32, torch.bfloat16),
           (16, 1, 64, 64, torch.bfloat16), (48, 1, 128, 128, torch.bfloat16), (6, 2, 128, 12, torch.bfloat16), (4, 2, 48, 16, torch.bfloat16),
           (4, 2, 256, 16, torch.bfloat16), (8, 2, 128, 16, torch.float32), (5, 5, 40, 7, torch.float32), (40, 1, 64, 8, torch.float32),
           (2, 1, 256, 16, torch.float32)]


@pytest.mark.parametrize("layout", LAYOUTS, ids=str)
def test_decode_in_groups(ops, layout):
    """Single tokens: two groups whose members stand in mixed order, and requests of their own; prefixes of whole blocks, whole pages and
    neither; own parts of one key and of several blocks."""
    requests = [(0, 1, 193), (1, 1, 260), (-1, 1, 1), (0, 1, 192 + 64), (1, 1, 251), (0, 1, 400), (-1, 1, 130), (1, 1, 251 + 63)]
    Batch(*layout[:4], requests, [192, 250], layout[4]).check(ops)


@pytest.mark.parametrize("layout", LAYOUTS, ids=str)
def test_portions_in_groups(ops, layout):
    """Portions of one to forty tokens beside single ones, a request without new tokens, a portion that follows its prefix at once."""
    requests = [(0, 37, 200 + 37), (0, 1, 230), (-1, 5, 5), (0, 40, 300), (1, 2, 130), (0, 0, 210), (-1, 70, 90), (1, 17, 129 + 17)]
    Batch(*layout[:4], requests, [200, 129], layout[4]).check(ops)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("prefix", [1, 63, 64, 65, 127, 128, 129, 640, 1000])
def test_prefixes_around_blocks(ops, dtype, prefix):
    requests = [(0, 1, prefix + own) for own in (1, 2, 63, 64, 65)]
    Batch(8, 2, 128, 16, requests, [prefix], dtype).check(ops)


@pytest.mark.parametrize("members", [2, 3, 31, 32, 33, 65, 130])
def test_many_members(ops, members):
    """More rows than a tile of either kernel has."""
    requests = [(0, 1, 200 + 1 + i % 5) for i in range(members)]
    Batch(8, 2, 128, 16, requests, [200], torch.bfloat16).check(ops)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_no_groups_at_all(ops, dtype):
    Batch(8, 2, 128, 16, [(-1, 1, n) for n in (1, 2, 64, 65, 500)] + [(-1, 30, 90)], [], dtype).check(ops)
    Batch(8, 2, 128, 16, [(-1, 1, 1)], [], dtype).check(ops)
    Batch(8, 2, 128, 16, [(0, 1, 300)], [256], dtype).check(ops)             # a group of one


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_that_see_nothing_and_rows_of_nobody(ops, dtype):
    """Entries that pad a step own no page: zeros.  Rows behind the last request keep what they held.  Pages missing in the middle."""
    b = Batch(8, 2, 128, 16, [(0, 1, 200), (0, 1, 190), (-1, 1, 1), (-1, 1, 100), (-1, 1, 1)], [128], dtype, extra_rows=5)
    b.table[2] = -1
    b.table[4] = -1
    b.table[3, 2] = -1
    b.table[1, 9] = 10 ** 6                                                    # outside the pool
    dev = b.device()
    out = torch.full_like(dev[0], 3.25)
    b.launch(ops, dev, out)
    b.compare(out)
    assert (out[2] == 0).all() and (out[4] == 0).all()
    assert (out[b.cu[-1]:] == 3.25).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_odd_groups(ops, dtype):
    """A leader that is no member itself, a leader that leads nobody, ids outside the batch, a prefix longer than some member's tokens."""
    b = Batch(8, 2, 128, 16, [(0, 1, 300), (0, 1, 280), (0, 1, 260), (-1, 1, 150)], [256], dtype)
    b.prefix_of = [-1, 0, 0, 99]
    b.check(ops)
    b.prefix_of = [0, 0, -5, 3]
    b.prefix_lens = [256, 0, 0, 64]
    b.check(ops)
    c = Batch(8, 2, 128, 16, [(0, 1, 256), (0, 1, 100), (0, 3, 300)], [256], dtype)
    c.check(ops)


@pytest.mark.parametrize("dim", [64, 128])
def test_long_runs_of_blocks(ops, dim):
    """More blocks of keys for every CTA than its ring holds, in segments of one tile and of two, long ones beside short ones."""
    rng = random.Random(dim)
    requests = [(0, 1, 4096 + rng.randint(1, 2000)) for _ in range(9)] + [(-1, 1, rng.randint(1, 3000)) for _ in range(6)] + \
               [(1, 20, 1500 + rng.randint(20, 900)) for _ in range(4)] + [(-1, 90, 1200)]
    rng.shuffle(requests)
    Batch(16, 8, dim, 16, requests, [4096, 1500], torch.bfloat16).check(ops)


def test_large_scores_and_equal_keys(ops):
    """A running maximum that grows from block to block, and one that is the first key's; all keys alike."""
    for sign in (1.0, -1.0):
        b = Batch(8, 2, 128, 16, [(0, 1, 700), (0, 1, 650), (0, 20, 690)], [640], torch.bfloat16)
        ramp = torch.ones(128) * 0.5
        for s in range(3):
            for j in range(b.ctx[s]):
                b.k[b.table[s, j // 16], :, j % 16] = (sign * ramp * (j % 640) / 64).to(torch.bfloat16)
        b.q = torch.full_like(b.q, 0.75)
        b.check(ops)
    b = Batch(8, 2, 128, 16, [(0, 1, 200), (0, 1, 230)], [192], torch.bfloat16)
    b.k = torch.where(b.k.isnan(), b.k, torch.ones_like(b.k))
    b.check(ops)


def test_the_result_does_not_depend_on_the_order_of_runs(ops):
    """Twice the same call: the same bits."""
    b = Batch(8, 2, 128, 16, [(0, 1, 3000 + 7 * i) for i in range(12)], [2944], torch.bfloat16)
    dev = b.device()
    first = b.launch(ops, dev, torch.empty_like(dev[0]))
    for _ in range(3):
        assert torch.equal(first, b.launch(ops, dev, torch.empty_like(dev[0])))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_replayed_with_other_groups_and_lengths(ops, dtype):
    """One recording: its replays follow the device's groups, lengths and tables."""
    batches = [Batch(8, 2, 128, 16, reqs, groups, dtype, spare=40) for reqs, groups in (
        ([(0, 1, 300), (0, 1, 310), (-1, 1, 40), (0, 1, 299)], [256]),
        ([(-1, 1, 1), (-1, 1, 2), (-1, 1, 3), (-1, 1, 4)], []),
        ([(0, 1, 100), (1, 1, 200), (0, 1, 101), (1, 1, 222)], [96, 160]))]
    pages = max(b.k.shape[0] for b in batches)
    width = max(b.table.shape[1] for b in batches)
    for b in batches:
        b.k, b.v = (torch.cat([x, torch.full((pages - x.shape[0], *x.shape[1:]), float("nan"), dtype=dtype)]) for x in (b.k, b.v))
        b.table = torch.cat([b.table, torch.full((4, width - b.table.shape[1]), -1, dtype=torch.int32)], 1)
    dev = batches[0].device()
    out = torch.empty_like(dev[0])
    batches[0].launch(ops, dev, out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        batches[0].launch(ops, dev, out)
    for b in batches[::-1]:
        for x, y in zip(dev, b.device()):
            x.copy_(y)
        out.fill_(float("nan"))
        graph.replay()
        b.compare(out)


def test_two_streams_at_once(ops):
    """Calls on two streams have partial results of their own."""
    a = Batch(8, 2, 128, 16, [(0, 1, 1500 + i) for i in range(9)], [1408], torch.bfloat16)
    b = Batch(8, 2, 128, 16, [(0, 1, 900 + i) for i in range(5)], [832], torch.bfloat16)
    da, db = a.device(), b.device()
    wa, wb = a.launch(ops, da, torch.empty_like(da[0])), b.launch(ops, db, torch.empty_like(db[0]))
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    oa, ob = [torch.empty_like(da[0]) for _ in range(10)], [torch.empty_like(db[0]) for _ in range(10)]
    torch.cuda.synchronize()
    for x, y in zip(oa, ob):
        with torch.cuda.stream(s1):
            a.launch(ops, da, x)
        with torch.cuda.stream(s2):
            b.launch(ops, db, y)
    # a stream that is not the current one
    oc = torch.empty_like(da[0])
    torch.cuda.synchronize()
    a.launch(ops, da, oc, stream=s1.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(x, wa) for x in oa + [oc]) and all(torch.equal(y, wb) for y in ob)


def test_refusals(ops):
    b = Batch(8, 2, 128, 16, [(0, 1, 200), (0, 1, 190)], [128], torch.bfloat16)
    q, k, v, table, cu, ctx, of, lens = b.device()
    out = torch.empty_like(q)

    def call(q=q, out=out, k=k, v=v, table=table, cu=cu, ctx=ctx, of=of, lens=lens, heads=8, kv_heads=2, dim=128, page=16):
        ops.attention_shared(q, out, k, v, table, cu, ctx, of, lens, 1, heads, kv_heads, dim, page, 0.1, ops.current_stream())
    call()
    for bad in (dict(out=out.float()), dict(q=q.half(), out=out.half()), dict(k=k.float()), dict(v=v[:-1]), dict(table=table.long()), dict(table=table[:1]),
                dict(cu=cu[:2]), dict(of=of[:1]), dict(lens=lens.cpu()), dict(ctx=ctx.long()), dict(heads=6), dict(kv_heads=3), dict(dim=64),
                dict(page=8), dict(q=q.transpose(0, 1)), dict(out=out[:1]), dict(q=q.cpu())):
        with pytest.raises(ops.KernelError):
            call(**bad)
    many = torch.zeros(600, dtype=torch.int32, device="cuda")
    with pytest.raises(ops.KernelError, match="512"):
        call(table=table[:1].expand(600, -1).contiguous(), cu=torch.zeros(601, dtype=torch.int32, device="cuda"), ctx=many, of=many, lens=many)
    wide = torch.empty(2, 1, 264, dtype=torch.bfloat16, device="cuda")
    pool = torch.empty(4, 1, 16, 264, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ops.KernelError):
        call(q=wide, out=wide.clone(), k=pool, v=pool, heads=1, kv_heads=1, dim=264)
    call(q=q[:0], out=out[:0])                                                 # no tokens: nothing to do


def a_batch():
    return Batch(8, 2, 128, 16, [(0, 1, 193), (0, 3, 260), (-1, 5, 40), (0, 1, 400)], [192], torch.bfloat16)


def plan_of(ops, b, dev, **other):
    q, k, v, table, cu, ctx, of, lens = dev
    sizes = dict(dtype=b.dtype, num_tokens=b.T, num_q_heads=b.heads, num_kv_heads=b.kv_heads, head_dim=b.dim, page_size=b.page,
                 pages_a_seq=table.shape[1], stream=ops.current_stream())
    return ops.shared_plan(cu_tokens=cu, context_lens=ctx, prefix_of=of, prefix_lens=lens, **{**sizes, **other})


def with_plan(ops, b, dev, plan):
    q, k, v, table, cu, ctx, of, lens = dev
    out = torch.empty_like(q)
    ops.attention_shared(q, out, k, v, table, cu, ctx, of, lens, b.max_new, b.heads, b.kv_heads, b.dim, b.page, b.scale, ops.current_stream(), plan=plan)
    return out


def test_a_plan_serves_calls_of_its_sizes_only(ops):
    b = a_batch()
    dev = b.device()
    plan = plan_of(ops, b, dev)
    first = with_plan(ops, b, dev, plan)
    b.compare(first)
    assert torch.equal(first, with_plan(ops, b, dev, plan)) and torch.equal(first, b.launch(ops, dev, torch.empty_like(dev[0])))
    for other in (dict(dtype=torch.float32), dict(num_tokens=b.T + 1), dict(num_q_heads=16), dict(num_kv_heads=4), dict(head_dim=64),
                  dict(page_size=32), dict(pages_a_seq=dev[3].shape[1] + 1)):
        with pytest.raises(ops.KernelError, match="other sizes"):
            with_plan(ops, b, dev, plan_of(ops, b, dev, **other))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_tokens_that_belong_to_two_requests(ops, dtype):
    """cu_tokens that fall: there is no room for what would come of it, and nothing is computed."""
    b = Batch(8, 2, 128, 16, [(0, 4, 300)] * 8, [192], dtype)
    dev = b.device()
    for cu in ([0, 32] * 4 + [32], [0, 30, 2, 31, 3, 32, 0, 32, 32], [32, 28, 24, 20, 16, 12, 8, 4, 0], [0, -5, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 0, 40, 5, 32]):
        dev[4] = torch.tensor(cu, dtype=torch.int32, device="cuda")
        out = b.launch(ops, dev, torch.full_like(dev[0], 7.0))
        assert (out == 7).all()
    assert ops.device_error() == 0


def test_lengths_written_right_in_front(ops):
    """Lengths and groups that kernels on the same stream write directly ahead of the call, through a chain of the library's own launches."""
    b = a_batch()
    dev = b.device()
    ints = [t.clone() for t in dev[4:]]
    want = b.launch(ops, dev, torch.empty_like(dev[0]))
    alone = b.launch(ops, dev[:6] + [torch.full_like(ints[2], -1), torch.zeros_like(ints[3])], torch.empty_like(dev[0]))
    for turn in range(30):
        for t, keep in zip(dev[4:], ints):
            t.zero_()
        b.launch(ops, dev, torch.empty_like(dev[0]))
        for t, keep in zip(dev[4:], ints):
            t.copy_(keep)
        if turn % 2:
            dev[6].fill_(-1)
        assert torch.equal(b.launch(ops, dev, torch.empty_like(dev[0])), alone if turn % 2 else want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_pages_behind_four_gigabytes(ops, dtype):
    """The same keys at the beginning and at the end of pools whose offsets pass 32 bits: the same result."""
    b = Batch(8, 2, 128, 16, [(0, 1, 193), (0, 3, 260), (-1, 5, 40), (0, 1, 400)], [192], dtype)
    dev = b.device()
    near = b.launch(ops, dev, torch.empty_like(dev[0]))
    b.compare(near)
    pages = dev[1].shape[0]
    total = 2 ** 32 // (2 * 16 * 128 * dev[1].element_size()) + 2 * pages
    k, v = torch.empty(total, 2, 16, 128, dtype=dtype, device="cuda"), torch.empty(total, 2, 16, 128, dtype=dtype, device="cuda")
    k[-pages:], v[-pages:] = dev[1], dev[2]
    k[:2 * pages], v[:2 * pages] = float("nan"), float("nan")
    table = torch.where(dev[3] >= 0, dev[3] + (total - pages), dev[3]).to(torch.int32)
    far = b.launch(ops, [dev[0], k, v, table] + dev[4:], torch.empty_like(dev[0]))
    assert torch.equal(near, far)
