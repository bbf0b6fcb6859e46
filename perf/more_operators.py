"""A serving step that the host need not prepare, over an 8-bit cache whose scales belong to blocks of tokens.

A case is one pass of one kind:

  step     the metadata of one step from the lengths of its requests: requests that ended give their cache blocks back, those that
           grow take new ones from the list of free blocks, and out come block tables, context lengths, cumulative lengths, positions
           and slots
  rotary   rotary positions on the query and key heads of one layer's packed projections: halves of a vector or neighbours as
           pairs, all of a head or its first part, plain frequencies or ones scaled for long contexts
  chunk    one layer of a prefill step over the 8-bit cache, without its attention: the new tokens' K / V rows are quantised into the
           cache, then the contexts come out of it as dense 16-bit rows, cached prefixes and new tokens alike
  decode   one layer of a decode step over the 8-bit cache: the step's K / V rows go into it, then every row attends over its whole
           context

Of the 8-bit cache, a (cache block, KV head) has one scale, a power of two: the smallest 2^e, at least 2^-126, of which the largest
absolute value among its rows is at most 127 times (int8) or 448 times (e4m3).  Elements are x / scale, rounded to nearest, ties to
even.  A block begins with its first row; rows that join it later may raise its scale, and the rows that were there are then brought
to the new one, rounded again.

Heads are those of the 32 / 8 and 16 / 8 head configurations and of their tensor-parallel shards, and groups of other sizes;
head_dim 128 and cache blocks of 256 tokens where nothing else is said.  Lengths are spread evenly over their range, in an order
that comes from the seed.
"""
import importlib
import math
import random

import numpy as np
import torch

own = False   # whether run() calls this library's operators; otherwise it computes them from elementary ones

D = 128
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
TOP = {"int8": 127.0, "e4m3": 448.0}
HEADS = ((32, 8), (16, 4), (8, 2), (4, 1), (16, 8), (8, 4), (8, 8), (8, 1), (6, 2), (14, 2))


def listed():
    return [
        # One user's next token.
        step("step-1", 1, 300, 300, 1, 1),
        # A decode step of the headline configuration's batch, some requests just ended.
        step("step-256", 256, 1024, 8192, 1, 1, ended=5),
        # A prefill step of 16 prompts, some behind what an earlier chunk has left.
        step("step-prefill-16", 16, 0, 768, 512, 4096, ended=2, index="i64"),
        # A large batch over small blocks, with some speculated tokens for each.
        step("step-1024", 1024, 200, 8192, 1, 4, ended=30, block_size=16),
        # One user's next token, then a batch with partly rotated heads, neighbours as pairs.
        rotary("rotary-1", 1, 32, 8, 300),
        rotary("rotary-256", 256, 16, 8, 8192, head_dim=64, part=0.5, layout="pairs", dtype="fp16"),
        # A long prefill step far out in a long context, frequencies scaled for it.
        rotary("rotary-16384", 16384, 32, 8, 1000000, scaled="yarn"),
        # A short question behind a cached prompt that ends inside a block.
        chunk("blocks8-chunk-1", 32, 8, 1, 77, 77, prefix=600),
        # A prefill step of 16 prompts of 512 to 4096 tokens, half of them behind a cached prefix.
        chunk("blocks8-chunk-16", 32, 8, 16, 512, 4096, prefix=768, prefix_share=0.5, kv="e4m3", dtype="fp16"),
        # One user, a short conversation.
        decode("blocks8-decode-1", 32, 8, 1, 300, 300),
        # One of eight tensor-parallel ranks (one KV head), fp16, e4m3, 64-bit indices.
        decode("blocks8-decode-rank", 4, 1, 256, 100, 2048, kv="e4m3", dtype="fp16", index="i64"),
        # The largest: the batch and the contexts of the headline configuration.
        decode("blocks8-decode-256", 32, 8, 256, 1024, 8192),
    ]


def step(name, batch, ctx_lo, ctx_hi, new_lo, new_hi, ended=0, block_size=256, index="i32", free_share=1.0, padding=0):
    return dict(name=name, kind="step", batch=batch, ctx_lo=ctx_lo, ctx_hi=ctx_hi, new_lo=new_lo, new_hi=new_hi, ended=ended, block_size=block_size,
                index=index, free_share=free_share, padding=padding)


def rotary(name, rows, q_heads, kv_heads, far, head_dim=D, part=1.0, layout="halves", scaled="plain", dtype="bf16", index="i32"):
    return dict(name=name, kind="rotary", rows=rows, q_heads=q_heads, kv_heads=kv_heads, far=far, head_dim=head_dim, part=part, layout=layout,
                scaled=scaled, dtype=dtype, index=index)


def chunk(name, q_heads, kv_heads, batch, q_lo, q_hi, prefix=0, prefix_share=1.0, dtype="bf16", index="i32", block_size=256, kv="int8"):
    return dict(name=name, kind="chunk", q_heads=q_heads, kv_heads=kv_heads, batch=batch, q_lo=q_lo, q_hi=q_hi, prefix=prefix,
                prefix_share=prefix_share, dtype=dtype, index=index, block_size=block_size, kv=kv)


def decode(name, q_heads, kv_heads, batch, ctx_lo, ctx_hi, dtype="bf16", index="i32", block_size=256, kv="int8"):
    return dict(name=name, kind="decode", q_heads=q_heads, kv_heads=kv_heads, batch=batch, ctx_lo=ctx_lo, ctx_hi=ctx_hi, dtype=dtype, index=index,
                block_size=block_size, kv=kv)


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Another case of the same ranges; none is more work than the largest listed one of its kind."""
    kind = rng.choice(("step", "rotary", "chunk", "decode", "decode"))
    index = rng.choice(("i32", "i32", "i64"))
    block_size = rng.choice((256, 256, 128, 64, 16))
    if kind == "step":
        batch = _log(rng, 1, 1024)
        hi = _log(rng, 16, min(40000, 500000 * block_size // batch))
        new = rng.choice((1, 1, rng.randint(1, 8), _log(rng, 1, max(1, min(8192, 40000 // batch)))))
        c = step("", batch, rng.randint(0, hi), hi, rng.randint(0, new), new, rng.choice((0, rng.randint(1, max(1, batch // 8)))), block_size, index,
                 rng.choice((1.0, 1.0, 0.6)), rng.choice((0, 0, rng.randint(1, 16))))
    elif kind == "rotary":
        hq, hkv = rng.choice(HEADS)
        head_dim = rng.choice((64, 80, 96, 128, 128, 192, 256))
        dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        rows = _log(rng, 1, min(16384, 16384 * 40 * 128 * 2 // ((hq + hkv) * head_dim * (4 if dtype == "fp32" else 2))))
        c = rotary("", rows, hq, hkv, _log(rng, 100, 4000000), head_dim, rng.choice((1.0, 0.5, 0.25)), rng.choice(("halves", "pairs")),
                   rng.choice(("plain", "linear", "yarn")), dtype, index)
    else:
        hq, hkv = rng.choice(HEADS)
        more = dict(dtype=rng.choice(("bf16", "bf16", "fp16")), index=index, block_size=block_size, kv=rng.choice(("int8", "e4m3")))
        if kind == "chunk":
            batch = _log(rng, 1, 32)
            hi = _log(rng, 1, min(8192, 36000 // batch))
            prefix = rng.choice((0, rng.randint(1, 700), 2 * block_size))
            c = chunk("", hq, hkv, batch, rng.randint(max(1, hi // 8), hi), hi, prefix, rng.choice((0.5, 1.0)) if prefix else 0.0, **more)
        else:
            batch = _log(rng, 1, 256)
            hi = _log(rng, 1, min(40000, 256 * 4608 // batch))
            c = decode("", hq, hkv, batch, rng.randint(max(1, hi // 20), hi), hi, **more)
    del c["name"]
    return c


# ---- lengths and sizes ------------------------------------------------------------------------------------------------------

def _spread(lo, hi, n):
    """n lengths over [lo, hi], the middles of n equal parts."""
    return [lo + int((hi - lo) * (i + 0.5) / n) for i in range(n)]


def _prompts(c):
    """(new tokens, cached prefix) of every prompt."""
    q = _spread(c["q_lo"], c["q_hi"], c["batch"])
    hits = round(c["batch"] * c["prefix_share"])
    return [(n, c["prefix"] if (i * hits) // len(q) != ((i + 1) * hits) // len(q) else 0) for i, n in enumerate(q)]


def _new_tokens(c):
    """New tokens of a step's requests: single ones over a small range, an even spread over a wide one."""
    lo, hi, n = c["new_lo"], c["new_hi"], c["batch"]
    return [lo + i % (hi - lo + 1) for i in range(n)] if hi - lo < 8 else _spread(lo, hi, n)


def _rotary_dim(c):
    return max(2, int(c["head_dim"] * c["part"]) // 2 * 2)


def _blocks(n, bs):
    return -(-n // bs)


def work(c):
    wide = 8 if c["index"] == "i64" else 4
    if c["kind"] == "rotary":
        size = 4 if c["dtype"] == "fp32" else 2
        heads, rot = c["q_heads"] + c["kv_heads"], _rotary_dim(c)
        return {"bytes": 2 * c["rows"] * heads * c["head_dim"] * size + c["rows"] * wide + rot // 2 * 4, "flops": c["rows"] * heads * rot * 3}
    bs = c["block_size"]
    if c["kind"] == "step":
        old, new = _spread(c["ctx_lo"], c["ctx_hi"], c["batch"]), _new_tokens(c)
        total = [a + b for a, b in zip(old, new)]
        used, tokens = sum(_blocks(t, bs) for t in total), sum(new)
        width = max(1, max(_blocks(t, bs) for t in total))
        given = sum(_blocks(t, bs) for t in _spread(c["ctx_lo"], c["ctx_hi"], c["ended"])) if c["ended"] else 0
        numbers = used + c["batch"] * (width + 7) + 2 * tokens + 2 * given + 4 * c["ended"]
        return {"bytes": numbers * wide, "flops": 8 * c["batch"] + 4 * tokens}
    hq, hkv = c["q_heads"], c["kv_heads"]
    row16, row8 = hkv * 2 * D * 2, hkv * 2 * D   # a token's K and V
    if c["kind"] == "chunk":
        lens = _prompts(c)
        new, cached = sum(n for n, _ in lens), sum(p for _, p in lens)
        scales = sum(_blocks(n + p, bs) for n, p in lens) * hkv * 8
        return {"bytes": new * (row16 + row8) + cached * row8 + (new + cached) * row16 + 2 * scales, "flops": 4 * new * hkv * D}
    ctx = _spread(c["ctx_lo"], c["ctx_hi"], c["batch"])
    blocks = sum(_blocks(t, bs) for t in ctx)
    return {"bytes": sum(ctx) * row8 + blocks * (hkv * 8 + wide) + 2 * c["batch"] * hq * D * 2 + c["batch"] * (row16 + row8 + wide),
            "flops": 4 * hq * D * sum(ctx)}


# ---- inputs -----------------------------------------------------------------------------------------------------------------

class _State:
    pass


class _Maker:
    """Seeded inputs on the GPU and the host-side metadata of a step."""

    def __init__(self, c, seed):
        self.c, self.rng, self.order = c, np.random.default_rng(seed), random.Random(seed)
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)
        self.index = torch.int64 if c["index"] == "i64" else torch.int32

    def normal(self, *shape, dtype=None):
        return torch.empty(shape, device="cuda", dtype=dtype or DTYPES[self.c["dtype"]]).normal_(generator=self.gen)

    def up(self, a, dtype=None):
        return torch.from_numpy(np.ascontiguousarray(a)).to("cuda", dtype or self.index)

    def zeros(self, *shape):
        return torch.zeros(shape, device="cuda", dtype=self.index)

    def shuffled(self, v):
        v = list(v)
        self.order.shuffle(v)
        return v

    def tables(self, need):
        """Block tables of sequences of so many blocks, a random permutation of the pool."""
        perm, at = self.rng.permutation(max(1, sum(need))), 0
        out = np.zeros((len(need), max(1, max(need))), np.int64)
        for i, n in enumerate(need):
            out[i, :n] = perm[at:at + n]
            at += n
        return out

    def cache(self, blocks):
        """Elements and scales of a cache of normal keys (or values), some blocks' twice or half as large."""
        c = self.c
        scale = torch.pow(2.0, self.up(self.rng.integers(-1, 2, (blocks, c["kv_heads"])) - (4 if c["kv"] == "int8" else 6), torch.float32))
        data = torch.empty((blocks, c["block_size"], c["kv_heads"], D), device="cuda", dtype=torch.int8 if c["kv"] == "int8" else torch.float8_e4m3fn)
        for first in range(0, blocks, 512):
            part = data[first:first + 512]
            x = self.normal(*part.shape, dtype=torch.float16) * (16.0 if c["kv"] == "int8" else 64.0)
            part.copy_(x.round().clamp(-127, 127) if c["kv"] == "int8" else x)
        return data, scale


def _frequencies(c):
    """Radians per position of every pair, and what the rotated part is multiplied by.  Scaled linearly, or as in YaRN (Peng et al., 2023):
    slow pairs as by linear scaling, fast ones left as they are, a ramp between them."""
    rot, base, factor, before = _rotary_dim(c), 10000.0, 32.0, 32768
    f = base ** (-np.arange(0, rot, 2) / rot)
    if c["scaled"] == "plain":
        return f, 1.0
    if c["scaled"] == "linear":
        return f / factor, 1.0
    turns = before * f / (2 * math.pi)
    keep = np.clip((turns - 1.0) / (32.0 - 1.0), 0.0, 1.0)
    return f * keep + f / factor * (1.0 - keep), 0.1 * math.log(factor) + 1.0


def _prepare_step(c, m, s):
    bs, b, ended, pad = c["block_size"], c["batch"], c["ended"], c["padding"]
    order = m.shuffled(range(b))
    old, new = ([v[i] for i in order] for v in (_spread(c["ctx_lo"], c["ctx_hi"], b), _new_tokens(c)))
    gone = m.shuffled(_spread(c["ctx_lo"], c["ctx_hi"], ended)) if ended else []
    s.width = max(1, max(_blocks(x + y, bs) for x, y in zip(old, new)))
    rows = m.rng.permutation(b + ended + 3)
    lens, need = np.zeros(len(rows), np.int64), np.zeros(len(rows), np.int64)
    for row, n in zip(rows, old + gone):
        lens[row], need[row] = n, _blocks(n, bs)
    row_blocks = max(s.width, int(need.max()))
    more = sum(_blocks(x + y, bs) - _blocks(x, bs) for x, y in zip(old, new))
    spare = max(1, int(more * c["free_share"]) + (3 if c["free_share"] == 1.0 else 0))
    perm = m.rng.permutation(int(need.sum()) + spare)
    held = np.full((len(rows), row_blocks), -1, np.int64)
    at = 0
    for row, n in enumerate(need):
        held[row, :n] = perm[at:at + n]
        at += n
    free = np.zeros(len(perm), np.int64)
    free[:spare] = perm[at:]
    s.pool, s.tokens = len(perm), _blocks(sum(new) + 1, 16) * 16   # (rows of a captured graph: some more than there are tokens)
    s.rows, s.new = m.up(np.concatenate([rows[:b], np.full(pad, -1)])), m.up(np.concatenate([np.array(new), np.zeros(pad, np.int64)]))
    s.ended = m.up(rows[b:b + ended]) if ended else None
    s.lens, s.held, s.free, s.count = m.up(lens), m.up(held), m.up(free), m.up(np.array([spare]))
    s.mid_lens, s.mid_count = torch.empty_like(s.lens), torch.empty_like(s.count)
    s.out_lens, s.out_count = torch.empty_like(s.lens), torch.empty_like(s.count)
    s.tables, s.ctx, s.cu_q, s.cu_k = m.zeros(b + pad, s.width), m.zeros(b + pad), m.zeros(b + pad + 1), m.zeros(b + pad + 1)
    s.positions, s.slots = m.zeros(s.tokens), m.zeros(s.tokens)
    return s


def _prepare_rotary(c, m, s):
    hq, hkv, hd = c["q_heads"], c["kv_heads"], c["head_dim"]
    qkv = m.normal(c["rows"], (hq + 2 * hkv) * hd)   # a projection's packed rows: queries, keys, values
    s.q, s.k = qkv[:, :hq * hd].unflatten(1, (hq, hd)), qkv[:, hq * hd:(hq + hkv) * hd].unflatten(1, (hkv, hd))
    s.q_out, s.k_out = torch.empty((c["rows"], hq, hd), device="cuda", dtype=qkv.dtype), torch.empty((c["rows"], hkv, hd), device="cuda", dtype=qkv.dtype)
    first = int(m.rng.integers(0, max(1, c["far"] - c["rows"]) + 1))
    # Runs of positions, each of some sequence.
    s.positions = m.up(np.concatenate([(first + 7919 * i) % c["far"] + np.arange(min(2048, c["rows"] - r)) for i, r in enumerate(range(0, c["rows"], 2048))]))
    f, s.factor = _frequencies(c)
    s.frequencies = m.up(f, torch.float32)
    return s


def prepare(case, seed):
    c, m, s = case, _Maker(case, seed), _State()
    s.c = c
    if c["kind"] == "step":
        return _prepare_step(c, m, s)
    if c["kind"] == "rotary":
        return _prepare_rotary(c, m, s)
    hq, hkv, b, bs = c["q_heads"], c["kv_heads"], c["batch"], c["block_size"]
    s.scale, s.workspace = 1.0 / math.sqrt(D), None
    if c["kind"] == "chunk":
        lens = m.shuffled(_prompts(c))
        new, total = np.array([n for n, _ in lens]), np.array([n + p for n, p in lens])
    else:
        total = np.array(m.shuffled(_spread(c["ctx_lo"], c["ctx_hi"], b)))
        new = np.ones(b, np.int64)
    tables = m.tables([_blocks(int(t), bs) for t in total])
    blocks = int(tables.max()) + 1
    (s.k_cache, s.k_scale), (s.v_cache, s.v_scale) = m.cache(blocks), m.cache(blocks)
    s.lens, s.tables, s.longest, s.total = m.up(total), m.up(tables), int(total.max()), int(total.sum())
    s.cu_q, s.cu_k = (m.up(np.concatenate([[0], np.cumsum(v)])) for v in (new, total))
    s.k, s.v = m.normal(int(new.sum()), hkv, D), m.normal(int(new.sum()), hkv, D)
    # Where the new rows go, and by blocks: which block, and how many rows of it were there.
    seq, pos = np.repeat(np.arange(b), new), np.concatenate([np.arange(t - n, t) for n, t in zip(new, total)])
    s.slots = m.up(tables[seq, pos // bs] * bs + pos % bs, torch.int64)
    unit = np.cumsum((np.diff(seq * (int(total.max()) // bs + 2) + pos // bs, prepend=-1) != 0)) - 1
    first = np.unique(unit, return_index=True)[1]
    there = pos[first] % bs
    s.unit, s.unit_block = m.up(unit, torch.int64), m.up(tables[seq, pos // bs][first], torch.int64)
    s.unit_new = m.up(there == 0, torch.bool)
    go_on = np.flatnonzero(there)
    s.go_on = m.up(go_on, torch.int64)
    s.go_on_rows = m.up(there[go_on], torch.int64)
    if c["kind"] == "chunk":
        s.row_seq = m.up(np.repeat(np.arange(b), total), torch.int64)
        s.row_pos = m.up(np.concatenate([np.arange(t) for t in total]), torch.int64)
        s.key, s.value = (torch.empty((s.total, hkv, D), device="cuda", dtype=s.k.dtype) for _ in range(2))
    else:
        s.q, s.out = m.normal(b, hq, D), torch.empty((b, hq, D), device="cuda", dtype=s.k.dtype)
    return s


# ---- the operators in plain form --------------------------------------------------------------------------------------------

def _release(s):
    """Blocks of the requests that ended onto the list of free ones, in their order."""
    s.mid_lens.copy_(s.lens)
    s.mid_count.copy_(s.count)
    if s.ended is None:
        return
    rows, bs = s.ended.long(), s.c["block_size"]
    n = (s.lens[rows].long() + bs - 1) // bs
    j = torch.arange(s.held.shape[1], device="cuda")
    to = s.count.long() + (torch.cumsum(n, 0) - n)[:, None] + j
    room = torch.cat([s.free, s.free[:1]])   # (what is no block goes behind the end)
    room[torch.where(j < n[:, None], to, len(room) - 1).flatten()] = s.held[rows].flatten()
    s.free.copy_(room[:-1])
    s.mid_lens[rows] = 0
    s.mid_count.copy_(s.count + n.sum())


def _step(s):
    bs, rows = s.c["block_size"], s.rows.long()
    known = rows >= 0
    row = rows.clamp(min=0)
    old, new = torch.where(known, s.mid_lens[row], 0).long(), s.new.long()
    total = old + new
    fits = known & (total <= s.width * bs)
    had = (old + bs - 1) // bs
    need = torch.where(fits, (total + bs - 1) // bs - had, 0)
    upto = torch.cumsum(need, 0)
    taken = fits & ((need == 0) | (upto <= s.mid_count))
    # The new blocks: the list's last first.
    j = torch.arange(s.width, device="cuda")
    nth = upto[:, None] - need[:, None] + j - had[:, None]
    fresh = taken[:, None] & (j >= had[:, None]) & (j < (had + need)[:, None])
    ids = s.free[torch.where(fresh, s.mid_count - 1 - nth, 0).clamp(min=0)]
    held = torch.where(fresh, ids, s.held[row, :s.width])
    s.tables.copy_(torch.where(taken[:, None] & (j < (had + need)[:, None]), held, 0))
    # (A request that has no place writes what is there, to a row of its own; padding to one behind the end.)
    room = torch.cat([s.held, s.held[:1]])
    room[torch.where(known, row, len(room) - 1), :s.width] = held
    s.held.copy_(room[:-1])
    s.ctx.copy_(torch.where(taken, total, 0))
    s.cu_q[1:] = torch.cumsum(new, 0)
    s.cu_k[1:] = torch.cumsum(s.ctx, 0)
    lens = torch.cat([s.mid_lens, s.mid_lens[:1]])
    lens[torch.where(taken, row, len(lens) - 1)] = total.to(lens.dtype)
    s.out_lens.copy_(lens[:-1])
    s.out_count.copy_(s.mid_count - torch.where(taken, upto, 0).max())
    t = torch.arange(s.tokens, device="cuda")
    seq = torch.searchsorted(s.cu_q[1:].long(), t, right=True).clamp(max=len(rows) - 1)
    there = (t < s.cu_q[-1]) & taken[seq]
    pos = torch.where(there, old[seq] + t - s.cu_q[seq], 0)
    s.positions.copy_(pos)
    s.slots.copy_(torch.where(there, s.tables[seq, pos // bs].long() * bs + pos % bs, -1))


def _rotary(s):
    c, rot = s.c, _rotary_dim(s.c)
    angle = s.positions.double()[:, None] * s.frequencies.double()
    cos, sin = ((f(angle) * s.factor).float()[:, None] for f in (torch.cos, torch.sin))
    for x, out in ((s.q, s.q_out), (s.k, s.k_out)):
        turned, rest = x[..., :rot].float(), x[..., rot:]
        if c["layout"] == "halves":
            a, b = turned[..., :rot // 2], turned[..., rot // 2:]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        else:
            a, b = turned[..., 0::2], turned[..., 1::2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        out.copy_(torch.cat([turned.to(x.dtype), rest], -1))


def _scale_for(top, kv):
    """The smallest power of two, at least 2^-126, that `top` is at most TOP times."""
    part, e = torch.frexp(top)
    whole, bits = math.frexp(TOP[kv])
    e = e - bits + (part > whole).to(e.dtype)
    return torch.ldexp(torch.ones_like(top), torch.where(top > 0, e, -126).clamp(min=-126))


def _round(x, kv):
    """Elements in 32 bits -> the cache's type."""
    return x.round().clamp(-127, 127).to(torch.int8) if kv == "int8" else x.clamp(-448, 448).to(torch.float8_e4m3fn)


def _bytes(cache):
    return cache.view(torch.uint8)


def _numbers(cache):
    """A cache as whole numbers: int8 ones as they are, e4m3 ones' bits."""
    return cache if cache.dtype == torch.int8 else _bytes(cache)


def _rows_of(cache, at):
    """Rows `at` of a cache of [rows, heads, D], in 32 bits (indexing by bytes: e4m3 has none of its own)."""
    return _bytes(cache)[at].view(cache.dtype).float()


def _store(s):
    kv, bs = s.c["kv"], s.c["block_size"]
    for x, cache, scale in ((s.k, s.k_cache, s.k_scale), (s.v, s.v_cache, s.v_scale)):
        top = x.float().abs().amax(-1)
        by_block = torch.zeros((len(s.unit_block), x.shape[1]), device="cuda").scatter_reduce(0, s.unit[:, None].expand_as(top), top, "amax")
        old = torch.where(s.unit_new[:, None], 0.0, scale[s.unit_block])
        now = torch.maximum(old, _scale_for(by_block, kv))
        for first in range(0, len(s.go_on), 64):   # rows that were there, brought to the block's new scale
            unit = s.go_on[first:first + 64]
            there = torch.arange(bs, device="cuda") < s.go_on_rows[first:first + 64, None]
            was = _bytes(cache)[s.unit_block[unit]]
            again = _bytes(_round(was.view(cache.dtype).float() * (old[unit] / now[unit])[:, None, :, None], kv))
            _bytes(cache)[s.unit_block[unit]] = torch.where(there[..., None, None], again, was)
        scale[s.unit_block] = now
        _bytes(cache).flatten(0, 1)[s.slots] = _bytes(_round(x.float() / now[s.unit][..., None], kv))


def _values(cache, scale, rows, bs):
    """Cache rows `rows` as the values they stand for, in 32 bits."""
    return _rows_of(cache.flatten(0, 1), rows) * scale[rows // bs][..., None]


def _gather(s):
    bs = s.c["block_size"]
    rows = s.tables.long()[s.row_seq, s.row_pos // bs] * bs + s.row_pos % bs
    s.key.copy_(_values(s.k_cache, s.k_scale, rows, bs))
    s.value.copy_(_values(s.v_cache, s.v_scale, rows, bs))


def _attend(s):
    c, bs = s.c, s.c["block_size"]
    hkv = c["kv_heads"]
    some = max(1, 400000 // (s.longest * hkv))   # sequences at a time
    for first in range(0, c["batch"], some):
        lens, tables = s.lens[first:first + some, None].long(), s.tables[first:first + some].long()
        pos = torch.arange(s.longest, device="cuda").expand(len(lens), -1)
        rows = tables.gather(1, pos // bs) * bs + pos % bs   # (behind a sequence's end those of some other block)
        q = s.q[first:first + some].float().unflatten(1, (hkv, -1))
        scores = torch.einsum("bjgd,bljd->bjgl", q, _values(s.k_cache, s.k_scale, rows, bs)) * s.scale
        scores = scores.masked_fill((pos >= lens)[:, None, None], -math.inf)
        p = torch.exp(scores - scores.amax(-1, keepdim=True))
        o = torch.einsum("bjgl,bljd->bjgd", p, _values(s.v_cache, s.v_scale, rows, bs)) / p.sum(-1, keepdim=True)
        s.out[first:first + some] = o.flatten(1, 2).to(s.out.dtype)


# ---- one pass ---------------------------------------------------------------------------------------------------------------

def _outputs(s):
    kind = s.c["kind"]
    if kind == "step":
        return s.tables, s.ctx, s.cu_q, s.cu_k, s.positions, s.slots, s.out_lens, s.out_count, s.held, s.free
    if kind == "rotary":
        return s.q_out, s.k_out
    if kind == "chunk":   # (the 8-bit elements show in the dense rows)
        return s.key, s.value, s.k_scale, s.v_scale
    # One new row among thousands hardly shows in the output: with the caches it went into.  An element is its number times its block's scale.
    return s.out, s.k_scale, s.v_scale, _numbers(s.k_cache), _numbers(s.v_cache)


def _own(s):
    """One pass by this library."""
    nvk = importlib.import_module("nano-vllm-cpp_b200")
    c = s.c
    kind = c["kind"]
    if kind == "step":
        lens, count = s.lens, s.count
        if s.ended is not None:
            nvk.release_blocks(s.ended, None, lens, s.held, s.free, count, c["block_size"], s.mid_lens, s.mid_count)
            lens, count = s.mid_lens, s.mid_count
        nvk.step_metadata(s.new, s.rows, lens, s.held, s.free, count, c["block_size"], s.pool, s.tables, s.ctx, s.cu_q, s.cu_k, s.positions, s.slots,
                          s.out_lens, s.out_count)
    elif kind == "rotary":
        nvk.rotary_embedding(s.q, s.k, s.positions, s.frequencies, c["layout"] == "pairs", s.factor, s.q_out, s.k_out)
    else:
        cache, shape = (s.k_cache, s.v_cache, s.k_scale, s.v_scale), (c["kv_heads"], D, c["block_size"])
        nvk.store_kvcache_blocks8(s.k, s.v, *cache, s.cu_q if kind == "chunk" else None, s.lens, s.tables)
        if kind == "chunk":
            nvk.gather_kvcache_blocks8(*cache, s.cu_k, s.tables, *shape, s.key, s.value)
        else:
            if s.workspace is None:   # kept from the first step on
                size = nvk.decode_attention_workspace_bytes(c["batch"], c["q_heads"], c["kv_heads"], D, s.tables.shape[1], c["block_size"])
                s.workspace = torch.empty(max(16, size), dtype=torch.uint8, device="cuda")
            nvk.launch_decode_attention_paged_blocks8(s.q, *cache, s.lens, s.tables, *shape, s.scale, s.out, s.workspace)
    return _outputs(s)


def run(s):
    if own:
        return _own(s)
    kind = s.c["kind"]
    if kind == "step":
        _release(s)
        _step(s)
    elif kind == "rotary":
        _rotary(s)
    else:
        _store(s)
        _gather(s) if kind == "chunk" else _attend(s)
    return _outputs(s)


# ---- the same from the definitions, in 64 bits --------------------------------------------------------------------------------

def _exact_step(s):
    bs, pool = s.c["block_size"], s.free.tolist()
    lens, held, count = s.lens.tolist(), s.held.tolist(), int(s.count)
    for row in s.ended.tolist() if s.ended is not None else []:
        for j in range(_blocks(lens[row], bs)):
            pool[count] = held[row][j]
            count += 1
        lens[row] = 0
    stack, wanted = count, 0
    tables, ctx, cu_q, cu_k, positions, slots = [], [], [0], [0], [0] * s.tokens, [-1] * s.tokens
    for row, n in zip(s.rows.tolist(), s.new.tolist()):
        line, length, at = [0] * s.width, 0, cu_q[-1]
        if row >= 0 and lens[row] + n <= s.width * bs:
            had, want = _blocks(lens[row], bs), _blocks(lens[row] + n, bs)
            first, wanted = wanted, wanted + want - had
            if want == had or wanted <= stack:
                for j in range(had, want):
                    held[row][j] = pool[stack - 1 - first - (j - had)]
                count = min(count, stack - wanted) if want > had else count
                line[:want] = held[row][:want]
                for i in range(n):
                    positions[at + i] = lens[row] + i
                    slots[at + i] = line[(lens[row] + i) // bs] * bs + (lens[row] + i) % bs
                lens[row] = length = lens[row] + n
        tables.append(line)
        ctx.append(length)
        cu_q.append(at + n)
        cu_k.append(cu_k[-1] + length)
    return tuple(torch.tensor(v, device="cuda", dtype=s.lens.dtype) for v in (tables, ctx, cu_q, cu_k, positions, slots, lens, [count], held, pool))


def _exact_rotary(s):
    rot, out = _rotary_dim(s.c), []
    turn = torch.exp(1j * (s.positions.to(torch.float64)[:, None, None] * s.frequencies.to(torch.float64))) * s.factor
    for x in (s.q, s.k):
        x = x.to(torch.float64)
        y = x.clone()
        first, second = (slice(0, rot // 2), slice(rot // 2, rot)) if s.c["layout"] == "halves" else (slice(0, rot, 2), slice(1, rot, 2))
        z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
        y[..., first], y[..., second] = z.real, z.imag
        out.append(y)
    return tuple(out)


def _nearest(x, kv):
    """x rounded to the elements of the 8-bit type, ties to even, in 64 bits."""
    if kv == "int8":
        return torch.round(x)
    grid = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)   # spacing of the type around x
    return torch.round(x / grid) * grid


class _ExactCache:
    """Elements (in 64 bits) and scales of the blocks that a case's new rows touch; everything else as it is in the cache."""

    def __init__(self, s, x, cache, scale):
        self.s, self.cache, self.bs = s, cache, s.c["block_size"]
        self.scale, self.fresh = scale.to(torch.float64).clone(), {}
        kv, tables = s.c["kv"], s.tables.tolist()
        x, cu = x.to(torch.float64), s.cu_q.tolist()
        for b, total in enumerate(s.lens.tolist()):
            n = cu[b + 1] - cu[b]
            at = total - n
            while at < total:
                block, row = tables[b][at // self.bs], at % self.bs
                end = min(total, at - row + self.bs)
                rows = x[cu[b] + at - (total - n):cu[b] + end - (total - n)]
                top = rows.abs().amax((0, 2))
                e = torch.floor(torch.log2(top / TOP[kv])).clamp(min=-130) - 1   # (below the one that is looked for)
                for _ in range(3):
                    e = torch.where(top > TOP[kv] * torch.exp2(e), e + 1, e)
                now = torch.exp2(e.clamp(min=-126))
                data = self.elements(block)
                if row > 0:
                    was = self.scale[block]
                    now = torch.maximum(was, now)
                    data[:row] = _nearest(data[:row] * (was / now)[:, None], kv)
                data[row:row + end - at] = _nearest(rows / now[:, None], kv)
                self.scale[block], self.fresh[block] = now, data
                at = end

    def elements(self, block):
        if block in self.fresh:
            return self.fresh[block]
        return _rows_of(self.cache, torch.tensor([block], device="cuda"))[0].to(torch.float64)

    def whole(self):
        """All of the cache, as whole numbers."""
        cache = self.cache.clone()
        for block, data in self.fresh.items():
            cache[block] = data.to(cache.dtype)
        return _numbers(cache)

    def rows(self, b, total):
        """Values of sequence b's first `total` positions."""
        blocks = self.s.tables[b, :_blocks(total, self.bs)].long()
        data = _rows_of(self.cache, blocks).to(torch.float64)
        for i, block in enumerate(blocks.tolist()):
            if block in self.fresh:
                data[i] = self.fresh[block]
        return (data * self.scale[blocks][:, None, :, None]).flatten(0, 1)[:total]


def exact(case, seed):
    s = prepare(case, seed)
    c = s.c
    if c["kind"] == "step":
        return _exact_step(s)
    if c["kind"] == "rotary":
        return _exact_rotary(s)
    k, v = _ExactCache(s, s.k, s.k_cache, s.k_scale), _ExactCache(s, s.v, s.v_cache, s.v_scale)
    lens = s.lens.tolist()
    if c["kind"] == "chunk":
        return tuple(torch.cat([x.rows(b, n) for b, n in enumerate(lens)]) for x in (k, v)) + (k.scale, v.scale)
    out = torch.empty(s.q.shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        keys, values = (x.rows(b, n).transpose(0, 1) for x in (k, v))
        p = torch.softmax(s.q[b].to(torch.float64).reshape(c["kv_heads"], -1, D) @ keys.transpose(1, 2) / math.sqrt(D), -1)
        out[b] = (p @ values).reshape(c["q_heads"], D)
    return out, k.scale, v.scale, k.whole(), v.whole()
