"""Plain restatements, in 64 bits on the CPU, of the filtered sampler and of attention whose requests share a prefix."""
import math

import numpy as np

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
