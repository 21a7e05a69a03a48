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
