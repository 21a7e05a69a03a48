"""Which sizes attention_shared takes: what can be told without a GPU."""
import pytest
import torch

from lucciola_b200 import ops

BF16 = ops.dtype_code(torch.bfloat16)


def refused(tokens, seqs, heads, kv_heads, page, pages):
    """The library's message for heads of 128; a machine without a GPU gets as far as that."""
    try:
        ops._shared_sizes(0, BF16, tokens, seqs, heads, kv_heads, 128, page, pages)
    except ops.KernelError as e:
        return str(e)
    return ""


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("seqs,kv_heads", [(512, 1024), (512, 64), (40, 8192), (1, 65535)])
def test_the_line_of_blocks_fits_32_bits(seqs, kv_heads, page):
    """The longest tables that are taken, tables of whole blocks of 64 keys and others: every tile of 256 rows (a tile costs 3 units, and 2
    a block), at one query head a kv head, with all the keys there can be, in a line of fewer than 2^31 units."""
    tokens = 512
    lo, hi = 1, (2 ** 31 - 65) // page                       # taken, refused
    assert "too much for one launch" in refused(tokens, seqs, kv_heads, kv_heads, page, hi)
    while hi - lo > 1:
        mid = (lo + hi) // 2
        if "too much for one launch" in refused(tokens, seqs, kv_heads, kv_heads, page, mid):
            hi = mid
        else:
            lo = mid
    for pages in range(max(lo - 4, 1), lo + 1):
        tiles = 2 * (tokens // 256 + seqs)
        assert tiles * (3 + 2 * -(-pages * page // 64)) * kv_heads < 2 ** 31


@pytest.mark.parametrize("pages,shared", [(1 << 13, True), (1 << 17, False)])
def test_a_step_that_is_too_much_for_a_launch_takes_the_ordinary_kernels(monkeypatch, pages, shared):
    """512 requests of 64 kv heads on tables of 2^17 and of 2^21 keys: the second step is none that attention_shared takes."""
    from types import SimpleNamespace as N
    from lucciola_b200.parts.attention import GQAttention
    called = []
    monkeypatch.setattr(ops, "attention", lambda *a, **k: called.append("ordinary"))
    monkeypatch.setattr(ops, "shared_plan", lambda *a, **k: called.append("plan"))
    monkeypatch.setattr(ops, "attention_shared", lambda *a, **k: called.append("shared"))
    part = N(num_heads=64, num_kv_heads=64, head_dim=128, window=0, scale=0.1, plan_key=lambda: ("attention tiles", 1), rt=N(stream=0))
    part._attend_shared = lambda *a: GQAttention._attend_shared(part, *a)
    q = torch.empty(512, 64, 128, dtype=torch.bfloat16)
    step = N(prefix_of=q, prefix_lens=q, num_seqs=512, max_q_len=1, cu_tokens=None, context_lens=None, memo={}, plans={},
             block_tables=[torch.empty(512, 1, dtype=torch.int32).expand(512, pages)])
    GQAttention._attend(part, q, q, step, N(page_size=16, group=0, k=None, v=None))
    assert called == (["plan", "shared"] if shared else ["ordinary"])
