"""Attention of requests that share prefixes where a CTA walks many short segments: requests in pairs or in one group behind a block of keys, with up to a
block of their own, on so many kv heads that tile B of a CTA has no block for dozens of steps in a row.

Every row of partial results is NaN before the call, so that one that nobody writes shows.  Tolerance as in test_shared_attention_gpu: the weights are
rounded to bfloat16 (2^-8 of a mean of values of at most V), and so is the output; 32-bit sums of a few hundred products: 2^-18."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

PAGE = 16


@pytest.fixture(scope="module")
def ops():
    from lucciola_b200 import ops
    return ops


class Short:
    """S requests with `new` tokens each, `members` behind every prefix of `prefix` keys, own[s] keys of their own in front of the new tokens' last.  Slots
    behind a request's end are NaN."""

    def __init__(self, S, kv_heads, group, dim, new, members, prefix, own):
        dev = "cuda"
        self.S, self.kv_heads, self.heads, self.dim, self.new = S, kv_heads, kv_heads * group, dim, new
        shared = prefix // PAGE
        groups = -(-S // members)
        length = torch.tensor([prefix + n + new - 1 for n in own])
        behind = (-(-length // PAGE) - shared).tolist()
        count = groups * shared + sum(behind)
        ids = torch.randperm(count).tolist()
        common = [[ids.pop() for _ in range(shared)] for _ in range(groups)]
        self.width = shared + max(behind)
        table = torch.full((S, self.width), -1, dtype=torch.int32)
        for s in range(S):
            row = common[s // members] + [ids.pop() for _ in range(behind[s])]
            table[s, :len(row)] = torch.tensor(row, dtype=torch.int32)
        kv = (count, kv_heads, PAGE, dim)
        self.k, self.v = (torch.randn(kv, device=dev).to(torch.bfloat16) for _ in range(2))
        last = table[torch.arange(S), -(-length // PAGE) - 1].long().to(dev)
        past = (torch.arange(PAGE)[None] >= ((length - 1) % PAGE + 1)[:, None]).to(dev)          # [S, PAGE]
        for pool in (self.k, self.v):
            pool[last] = pool[last].masked_fill(past[:, None, :, None], float("nan"))
        self.q = torch.randn(S * new, self.heads, dim, device=dev).to(torch.bfloat16)
        ints = dict(cu=[s * new for s in range(S + 1)], ctx=length.tolist(), of=[s // members * members for s in range(S)],
                    lens=[0 if s % members else prefix for s in range(S)])
        self.ints = {k: torch.tensor(v, dtype=torch.int32, device=dev) for k, v in ints.items()}
        self.table, self.length, self.scale = table.to(dev), length.to(dev), dim ** -0.5

    def call(self, ops):
        """Through the library's entry point, on partial results of this test's own."""
        T = self.S * self.new
        sizes = (T, self.S, self.heads, self.kv_heads, self.dim, PAGE, self.width)
        dt = ops.dtype_code(torch.bfloat16)
        n_ints, n_floats = ops._shared_sizes(0, dt, *sizes)
        plan = torch.full((n_ints,), -1, dtype=torch.int32, device="cuda")
        floats = torch.full((n_floats,), float("nan"), device="cuda")
        out = torch.full_like(self.q, float("nan"))
        lengths = [self.ints[n].data_ptr() for n in ("cu", "ctx", "of", "lens")]
        ops._call("lb_attention_shared", dt, self.q.data_ptr(), out.data_ptr(), self.k.data_ptr(), self.v.data_ptr(), self.table.data_ptr(), plan.data_ptr(), n_ints,
                  *lengths, *sizes[:6], self.k.shape[0], self.width, self.scale, floats.data_ptr(), n_floats, ops.current_stream())
        torch.cuda.synchronize()
        assert ops.device_error() == 0
        return out

    def want(self):
        """In 64 bits, some requests at a time, each through its own table."""
        out = torch.empty(self.q.shape, dtype=torch.float64, device="cuda")
        key = torch.arange(self.width * PAGE, device="cuda")
        g = self.heads // self.kv_heads
        for a in range(0, self.S, 32):
            b = min(a + 32, self.S)
            pages = self.table[a:b].long().clamp(min=0)
            k, v = (x[pages].transpose(2, 3).reshape(b - a, -1, self.kv_heads, self.dim).double() for x in (self.k, self.v))
            there = key < self.length[a:b, None]
            k, v = (x.masked_fill(~there[:, :, None, None], 0.0) for x in (k, v))
            q = self.q[a * self.new:b * self.new].double().view(b - a, self.new, self.kv_heads, g, self.dim)
            position = self.length[a:b, None] - self.new + torch.arange(self.new, device="cuda")
            score = torch.einsum("snkgd,slkd->skgnl", q, k) * self.scale
            score = score.masked_fill((key > position[:, :, None])[:, None, None], -torch.inf)
            o = torch.einsum("skgnl,slkd->snkgd", torch.softmax(score, -1), v)
            out[a * self.new:b * self.new] = o.reshape(-1, self.heads, self.dim)
        return out

    def check(self, ops):
        got = self.call(ops)
        assert got.isfinite().all()
        top = float(self.v.nan_to_num(0.0).abs().max())
        assert (got.double() - self.want()).abs().max() <= 2 ** -7 * top + 2 ** -18 * top
        return got


# requests, kv heads, query heads a kv head, new tokens, members of a group
SHAPES = [(512, 8, 4, 1, 2), (512, 8, 8, 1, 2), (256, 16, 1, 1, 2), (256, 32, 1, 1, 2), (128, 32, 1, 1, 2), (512, 16, 8, 5, 512), (256, 32, 1, 40, 4)]


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_many_short_segments(ops, shape, dim):
    S, kv_heads, group, new, members = shape
    Short(S, kv_heads, group, dim, new, members, 64, torch.randint(1, 65, (S,)).tolist()).check(ops)


@pytest.mark.parametrize("shape", SHAPES[:5], ids=str)
def test_longer_ones_among_them(ops, shape):
    """Every eighth request has several blocks of its own: tile B has work, then dozens of steps without any, then work again."""
    S, kv_heads, group, new, members = shape
    own = torch.randint(1, 65, (S,))
    own[::8] = torch.randint(65, 400, (len(own[::8]),))
    Short(S, kv_heads, group, 128, new, members, 64, own.tolist()).check(ops)


def test_the_same_bits_every_time(ops):
    b = Short(256, 16, 1, 128, 1, 2, 64, [1 + s % 64 for s in range(256)])
    first = b.call(ops)
    for _ in range(10):
        assert torch.equal(first, b.call(ops))
