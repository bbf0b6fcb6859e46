"""Plain 64-bit restatements of the 4-bit cache, of decode attention with key weights and of eviction, in numpy, straight from their definitions
(include/nvk.h).  Values of a 16-bit type come in as float64 arrays that hold them exactly."""
import numpy as np

D = 128
HALF_STEP = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}    # half a unit in the last place, relative


def to_type(x, dtype):
    """float64 -> fp32 -> the 16-bit type -> float64, each to nearest even."""
    import torch
    with np.errstate(over="ignore"):
        return torch.from_numpy(np.asarray(x, np.float64).astype(np.float32)).to(getattr(torch, dtype)).double().numpy()


def quantise(x, dtype):
    """Head vectors [..., 128] -> (bytes [..., 64], params [..., 2])."""
    x = np.asarray(x, np.float64)
    low, high = x.min(-1), x.max(-1)                           # (NaN where there is one)
    with np.errstate(all="ignore"):
        span = np.float32(high) - np.float32(low)
        fine = np.isfinite(span)
        step = np.where(fine, to_type(span / np.float32(15), dtype), np.nan)
        n = np.minimum(np.floor((x - low[..., None]) / step[..., None] + 0.5), 15)
    n = np.where(fine[..., None] & (step > 0)[..., None], n, 0).astype(np.uint8)
    return n[..., 0::2] | (n[..., 1::2] << 4), np.stack([step, np.where(fine, low, np.nan)], -1)


def numbers(data):
    n = np.empty((*data.shape[:-1], 2 * data.shape[-1]))
    n[..., 0::2], n[..., 1::2] = data & 15, data >> 4
    return n


def values(data, params):
    return params[..., 1:] + params[..., :1] * numbers(data)


def places(table, n, block_size, blocks):
    """Cache rows of keys 0 .. n - 1 of a sequence; -1 where there is none."""
    pos = np.arange(n)
    blk = pos // block_size
    ids = np.where(blk < len(table), np.asarray(table, np.int64)[np.minimum(blk, len(table) - 1)], -1)
    return np.where((ids >= 0) & (ids < blocks), ids * block_size + pos % block_size, -1)


def context(cache_rows, at):
    """Rows of [rows, Hkv, D], zeros where there are none."""
    return np.where((at >= 0)[:, None, None], cache_rows[np.maximum(at, 0)], 0.0)


def attend(q, k, v, scale):
    """One sequence: q [Hq, D], k and v [n, Hkv, D] -> (out [Hq, D], probabilities [Hq, n])."""
    hq, hkv = q.shape[0], k.shape[1]
    if k.shape[0] == 0:
        return np.zeros_like(q), np.zeros((hq, 0))
    s = np.einsum("jgd,njd->jgn", q.reshape(hkv, hq // hkv, -1), k) * scale
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    return np.einsum("jgn,njd->jgd", p, v).reshape(hq, -1), p.reshape(hq, -1)


def keep(weights, n, budget, sinks, recent):
    """Which keys of one KV head stay, in order."""
    if n <= budget:
        return np.arange(n)
    middle = np.arange(sinks, n - recent)
    w = np.asarray(weights, np.float64)[middle]
    best = sorted(range(len(middle)), key=lambda i: (bool(np.isnan(w[i])), -w[i] if not np.isnan(w[i]) else 0.0, i))[:budget - sinks - recent]
    return np.sort(np.concatenate([np.arange(sinks), middle[np.asarray(best, int)], np.arange(n - recent, n)])).astype(int)


def score_error(q, k_abs, scale):
    """How far an fp32 score can be off: the sum of 128 products (and of the two terms of a 4-bit key) of magnitudes |q| `k_abs`, each addition by 2^-24
    of the sum of the magnitudes at most, with 8 operations more for the scaling."""
    return 136 * 2.0 ** -24 * float(np.abs(q).sum(-1).max()) * float(k_abs) * abs(scale)
