"""Plain restatements, in 64 bits on the CPU, of the filtered sampler and of attention whose requests share a prefix."""
import math

import numpy as np
import torch

M64 = (1 << 64) - 1


def _mix(x: np.ndarray) -> np.ndarray:
    x = (x ^ (x >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
    x = (x ^ (x >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
    return x ^ (x >> np.uint64(31))


def uniforms(key: int, counter: int, vocab: int) -> np.ndarray:
    """The samplers' numbers in (0, 1) for every vocabulary index."""
    with np.errstate(over="ignore"):
        row = _mix(np.uint64(key & M64) + np.uint64(0x9E3779B97F4A7C15) * np.uint64(counter + 1))
        h = _mix(row ^ (np.uint64(0xD6E8FEB86659FD93) * (np.arange(vocab, dtype=np.uint64) + np.uint64(1))))
    return ((h >> np.uint64(41)).astype(np.float64) + 0.5) / 2 ** 23


def kept_tokens(logits, temperature: float, top_k: int, top_p: float, min_p: float) -> np.ndarray:
    """The tokens a row keeps, in the order of falling logits."""
    x = np.where(np.isnan(logits), -np.inf, np.asarray(logits, dtype=np.float64))
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if top_k > 0:
        order = order[:top_k]
    w = np.exp((x[order] - x[order[0]]) / temperature)
    n = len(order)
    if top_p < 1:
        n = min(n, max(1, int(((np.cumsum(w) - w) < top_p * w.sum()).sum())))
    if min_p > 0:
        n = min(n, max(1, int((w >= min_p).sum())))
    return order[:n]


def draw(logits, temperature, key, counter, top_k=0, top_p=1.0, min_p=0.0) -> int:
    x = np.where(np.isnan(logits), -np.inf, np.asarray(logits, dtype=np.float64))
    if not (x > -np.inf).any():
        return 0
    if not temperature > 0 or x.max() == np.inf:
        return int(np.argmax(x))
    kept = kept_tokens(logits, temperature, top_k, top_p, min_p)
    score = (x[kept] - x.max()) / temperature - np.log(-np.log(uniforms(key, counter, len(x))[kept]))
    return int(kept[score == score.max()].min())


def shared_attention(q, k_cache, v_cache, table, cu, ctx, prefix_of, prefix_lens, scale):
    """[T, heads, dim] in 64 bits; rows of no request are NaN.  Key j of request s lies in the table row of its prefix if j is one of the
    prefix's keys, else in its own; keys whose page is not in the pool are not there."""
    heads, dim = q.shape[1:]
    pages, kv_heads, ps = k_cache.shape[:3]
    out = torch.full(q.shape, math.nan, dtype=torch.float64)
    for s in range(len(ctx)):
        n = cu[s + 1] - cu[s]
        length = min(ctx[s], table.shape[1] * ps)
        lead = prefix_of[s]
        keys = []
        for j in range(length):
            row = table[lead] if 0 <= lead < len(ctx) and j < prefix_lens[lead] else table[s]
            page = int(row[j // ps])
            keys.append((page, j % ps) if 0 <= page < pages else None)
        for i in range(n):
            position = ctx[s] - n + i
            seen = [at for at in keys[:max(position + 1, 0)] if at is not None]
            t = cu[s] + i
            if not seen:
                out[t] = 0.0
                continue
            page, slot = torch.tensor(seen).T
            k = k_cache[page, :, slot].double().repeat_interleave(heads // kv_heads, 1)       # [keys, heads, dim]
            v = v_cache[page, :, slot].double().repeat_interleave(heads // kv_heads, 1)
            w = torch.softmax(torch.einsum("hd,jhd->hj", q[t].double(), k) * scale, 1)
            out[t] = torch.einsum("hj,jhd->hd", w, v)
    return out
