"""Plain 64-bit restatements of the 8-bit cache with scales of blocks, of rotary positions and of a step's metadata, in numpy, straight from their definitions
(include/nvk.h).  Values of a narrower type come in as float64 arrays that hold them exactly."""
import math

import numpy as np

D = 128
TOP = {"int8": 127.0, "e4m3": 448.0}
HALF_STEP = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11, "float32": 2.0 ** -24}    # half a unit in the last place, relative


def scale_for(top, kind):
    """The smallest power of two, at least 2^-126, that `top` is at most TOP times; NaN for what is not finite."""
    out = np.empty(np.shape(top))
    for i, a in np.ndenumerate(top):
        e = -126
        if np.isfinite(a):
            while a > TOP[kind] * 2.0 ** e:
                e += 1
        out[i] = 2.0 ** e if np.isfinite(a) else np.nan
    return out


def nearest(x, kind):
    """Elements of the 8-bit type next to x, ties to even; NaN: 0 (int8), NaN (e4m3)."""
    x = np.asarray(x, np.float64)
    if kind == "int8":
        return np.where(np.isnan(x), 0.0, np.rint(x))
    with np.errstate(all="ignore"):
        grid = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -6))) - 3)
        return np.clip(np.rint(x / grid) * grid, -448, 448)


class Cache:
    """K or V: elements [blocks, block_size, Hkv, 128] and scales [blocks, Hkv]."""

    def __init__(self, blocks, block_size, hkv, kind):
        self.kind, self.bs = kind, block_size
        self.data, self.scale = np.zeros((blocks, block_size, hkv, D)), np.zeros((blocks, hkv))

    def store(self, x, cu, lens, tables):
        """Returns the blocks that were written."""
        written = []
        for s, total in enumerate(lens):
            n = cu[s + 1] - cu[s]
            start = int(total) - n
            for blk in range(max(start, 0) // self.bs, -(-max(int(total), 0) // self.bs)):
                first, last = max(start, 0, blk * self.bs), min(int(total), (blk + 1) * self.bs)
                if first >= last or blk >= len(tables[s]) or not 0 <= tables[s][blk] < len(self.data):
                    continue
                block, row = int(tables[s][blk]), first - blk * self.bs
                rows = x[cu[s] + first - start:cu[s] + last - start]
                now = scale_for(np.abs(rows).max((0, 2)), self.kind)
                if row > 0:
                    old = self.scale[block]
                    now = np.where(np.isnan(old) | np.isnan(now), np.nan, np.maximum(old, now))
                    with np.errstate(all="ignore"):
                        again = nearest(self.data[block, :row] * (old / now)[:, None], self.kind)
                    grown = ~(old == now) & ~np.isnan(old)
                    self.data[block, :row] = np.where(grown[:, None], again, self.data[block, :row])
                with np.errstate(all="ignore"):
                    self.data[block, row:row + last - first] = nearest(rows / now[:, None], self.kind)
                self.scale[block] = now
                written.append(block)
        return written

    def rows(self, table, n):
        """Values of positions 0 .. n - 1 of a sequence; zeros where there is no block."""
        out = np.zeros((n, *self.data.shape[2:]))
        for i in range(0, n, self.bs):
            if i // self.bs < len(table) and 0 <= table[i // self.bs] < len(self.data):
                block = int(table[i // self.bs])
                out[i:i + self.bs] = self.data[block, :min(self.bs, n - i)] * self.scale[block][:, None]
        return out


def attend(q, k, v, scale):
    """One sequence: q [Hq, D], k and v [n, Hkv, D] -> (out [Hq, D], the largest p |v| sums [Hq, D])."""
    hq, hkv = q.shape[0], k.shape[1]
    if k.shape[0] == 0:
        return np.zeros_like(q), np.zeros_like(q)
    s = np.einsum("jgd,njd->jgn", q.reshape(hkv, hq // hkv, -1), k) * scale
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    return (np.einsum("jgn,njd->jgd", p, x).reshape(hq, -1) for x in (v, np.abs(v)))


def rotary(x, positions, inv_freq, pairs, factor):
    """x [rows, heads, D] -> the same with its first 2 len(inv_freq) elements turned."""
    rot = 2 * len(inv_freq)
    angle = np.asarray([[float(p) * float(f) for f in inv_freq] for p in positions]).reshape(len(positions), len(inv_freq))
    c, s = (np.asarray(f(np.asarray(angle, np.longdouble)), np.float64)[:, None] * factor for f in (np.cos, np.sin))
    y = np.array(x, np.float64)
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if pairs else (x[..., :rot // 2], x[..., rot // 2:rot])
    first, second = a * c - b * s, b * c + a * s
    if pairs:
        y[..., 0:rot:2], y[..., 1:rot:2] = first, second
    else:
        y[..., :rot // 2], y[..., rot // 2:rot] = first, second
    return y


def inv_freq(rot, base, scaling, factor, original, low, high):
    out = []
    for i in range(rot // 2):
        theta = base ** (-2.0 * i / rot)
        if scaling == "base":
            theta = (base * factor ** (rot / (rot - 2))) ** (-2.0 * i / rot)
        elif scaling == "linear":
            theta /= factor
        elif scaling in ("parts", "yarn"):
            g = min(max((original * theta / (2 * math.pi) - low) / (high - low), 0.0), 1.0)
            theta = (1 - g) * theta / factor + g * theta
        out.append(theta)
    return out, 0.1 * math.log(factor) + 1 if scaling == "yarn" else 1.0


class Requests:
    """Tables of requests and the list of free blocks."""

    def __init__(self, lens, held, free, count, block_size):
        self.lens, self.held, self.free, self.count, self.bs = list(lens), [list(h) for h in held], list(free), count, block_size

    def blocks(self, n):
        return -(-n // self.bs)

    def step(self, new, rows, width, tokens, pool):
        """(block_tables, context_lens, cu_q, cu_k, positions, slots)"""
        room = min(len(self.held[0]), width) * self.bs
        tables, ctx, cu_q, cu_k = [], [], [0], [0]
        positions, slots = [0] * tokens, [-1] * tokens
        stack, wanted, taken = self.count, 0, 0
        for b, n in enumerate(new):
            row = b if rows is None else rows[b]
            line, length, at = [0] * width, 0, cu_q[-1]
            if 0 <= row < len(self.lens) and self.lens[row] + n <= room:
                had, want = self.blocks(self.lens[row]), self.blocks(self.lens[row] + n)
                first, wanted = wanted, wanted + want - had
                if want == had or wanted <= stack:
                    for j in range(had, want):
                        self.held[row][j] = self.free[stack - 1 - first - (j - had)]
                    taken = max(taken, wanted if want > had else 0)
                    line[:want] = self.held[row][:want]
                    for i in range(n):
                        pos = self.lens[row] + i
                        if at + i < tokens:
                            positions[at + i] = pos
                            if 0 <= line[pos // self.bs] < pool:
                                slots[at + i] = line[pos // self.bs] * self.bs + pos % self.bs
                    self.lens[row] += n
                    length = self.lens[row]
            tables.append(line)
            ctx.append(length)
            cu_q.append(at + n)
            cu_k.append(cu_k[-1] + length)
        self.count -= taken
        return tables, ctx, cu_q, cu_k, positions, slots

    def release(self, rows, first):
        for b, row in enumerate(range(len(self.lens)) if rows is None else rows):
            if not 0 <= row < len(self.lens):
                continue
            for j in range(first[b] if first is not None else 0, self.blocks(self.lens[row])):
                if self.count < len(self.free):
                    self.free[self.count] = self.held[row][j]
                    self.count += 1
            self.lens[row] = 0
