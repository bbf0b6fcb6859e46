"""Long contexts in little memory: a paged KV cache of 4 bits, and a cache that keeps the keys that attention uses.

A case is one pass of one kind:

  decode   one layer of a decode step over a 4-bit cache: the step's new K / V rows are quantised into it, then every row
           attends over its whole context
  chunk    one layer of a prefill step over a 4-bit cache, without its attention: the new tokens' K / V rows are quantised
           into the cache, then the contexts come out of it as dense 16-bit rows, cached prefixes and new tokens alike
  weights  one layer of a decode step whose attention weights are added up for every key of every KV head, over a 16-bit or a
           4-bit cache: what an eviction later goes by
  evict    one eviction: of every sequence and KV head the first keys, the last ones and those of the largest weight stay,
           and close up in other blocks, their weights with them (4-bit caches: then they are read back)

A head vector x of a 4-bit cache is stored as whole numbers n from 0 to 15 with a step and a lowest value of its own, in the type
of x: low = min x, step = (max x - min x) / 15 rounded to that type, n = floor((x - low) / step + 1/2), 15 at most, 0 where the step
is 0; it stands for low + step n.  Where max x - min x is not finite, step and low are NaN.

Heads are those of the 32 / 8 and 16 / 8 head configurations and of their tensor-parallel shards, and groups of other sizes;
head_dim 128, cache blocks of 256 tokens where nothing else is said.  Lengths are spread evenly over their range, in an order that
comes from the seed.
"""
import importlib
import math
import random

import numpy as np
import torch

own = False   # whether run() calls this library's operators; otherwise it computes them from elementary ones

D = 128
LEVELS = 15
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
HEADS = ((32, 8), (16, 4), (8, 2), (4, 1), (16, 8), (8, 4), (8, 8), (8, 1), (6, 2), (14, 2))


def listed():
    return [
        # One user, a short conversation: what a call costs when there is next to nothing to read.
        decode("int4-decode-1", 32, 8, 1, 300, 300),
        # Some dozens of users with contexts of mixed length, the bulk of a server's day.
        decode("int4-decode-64", 32, 8, 64, 500, 4096),
        # The largest: the batch and the contexts of the repository's headline configuration, over the 4-bit cache.
        decode("int4-decode-256", 32, 8, 256, 1024, 8192),
        # One of eight tensor-parallel ranks (one KV head), fp16, 64-bit indices.
        decode("int4-decode-rank", 4, 1, 256, 100, 2048, dtype="fp16", index="i64"),
        # A handful of long documents.
        decode("int4-decode-long-3", 16, 8, 3, 9000, 40000),
        # A short question behind a cached prompt.
        chunk("int4-chunk-1", 32, 8, 1, 77, 77, prefix=512),
        # A prefill step of 16 prompts of 512 to 4096 tokens, half of them behind a cached prefix.
        chunk("int4-chunk-16", 32, 8, 16, 512, 4096, prefix=768, prefix_share=0.5, dtype="fp16"),
        # One user again, with the weights of its keys.
        weights("weights-1", 32, 8, 1, 300, 300),
        # The step of some dozens of users, 16-bit cache.
        weights("weights-64", 32, 8, 64, 500, 4096),
        # The same over the 4-bit cache, 16 / 8 heads.
        weights("weights-int4-100", 16, 8, 100, 500, 4096, kv="int4"),
        # Four conversations that have outgrown their share of the cache.
        evict("evict-4", 32, 8, 4, 2000, 4096, budget=1024, sinks=4, recent=256),
        # A round of evictions over a whole batch; some of its sequences are still short enough.
        evict("evict-32", 16, 8, 32, 1000, 8192, budget=2048, sinks=4, recent=512),
    ]


def decode(name, q_heads, kv_heads, batch, ctx_lo, ctx_hi, dtype="bf16", index="i32", block_size=256, kv="int4", kind="decode"):
    return dict(name=name, kind=kind, q_heads=q_heads, kv_heads=kv_heads, batch=batch, ctx_lo=ctx_lo, ctx_hi=ctx_hi, dtype=dtype, index=index,
                block_size=block_size, kv=kv)


def weights(name, q_heads, kv_heads, batch, ctx_lo, ctx_hi, dtype="bf16", index="i32", block_size=256, kv="same"):
    return decode(name, q_heads, kv_heads, batch, ctx_lo, ctx_hi, dtype, index, block_size, kv, kind="weights")


def chunk(name, q_heads, kv_heads, batch, q_lo, q_hi, prefix=0, prefix_share=1.0, dtype="bf16", index="i32", block_size=256):
    return dict(name=name, kind="chunk", q_heads=q_heads, kv_heads=kv_heads, batch=batch, q_lo=q_lo, q_hi=q_hi, prefix=prefix,
                prefix_share=prefix_share, dtype=dtype, index=index, block_size=block_size, kv="int4")


def evict(name, q_heads, kv_heads, batch, ctx_lo, ctx_hi, budget, sinks, recent, dtype="bf16", index="i32", block_size=256, kv="same"):
    return dict(name=name, kind="evict", q_heads=q_heads, kv_heads=kv_heads, batch=batch, ctx_lo=ctx_lo, ctx_hi=ctx_hi, budget=budget, sinks=sinks,
                recent=recent, dtype=dtype, index=index, block_size=block_size, kv=kv)


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Another case of the same ranges; none is more work than the largest listed one of its kind."""
    kind = rng.choice(("decode", "decode", "chunk", "weights", "weights", "evict"))
    hq, hkv = rng.choice(HEADS)
    more = dict(dtype=rng.choice(("bf16", "bf16", "fp16")), index=rng.choice(("i32", "i32", "i64")), block_size=rng.choice((256, 256, 128, 64, 16)))
    if kind == "decode":
        batch = _log(rng, 1, 256)
        hi = _log(rng, 1, min(40000, 256 * 4608 // batch))
        c = decode("", hq, hkv, batch, rng.randint(max(1, hi // 20), hi), hi, **more)
    elif kind == "weights":
        batch = _log(rng, 1, 100)
        hi = _log(rng, 1, min(40000, 64 * 2298 // batch))
        c = weights("", hq, hkv, batch, rng.randint(max(1, hi // 20), hi), hi, kv=rng.choice(("same", "int4")), **more)
    elif kind == "chunk":
        batch = _log(rng, 1, 32)
        hi = _log(rng, 1, min(8192, 40000 // batch))
        prefix = rng.choice((0, rng.randint(1, 1024), 4 * more["block_size"]))
        c = chunk("", hq, hkv, batch, rng.randint(max(1, hi // 8), hi), hi, prefix, rng.choice((0.5, 1.0)) if prefix else 0.0, **more)
    else:
        batch = _log(rng, 1, 32)
        hi = _log(rng, 16, min(40000, 100000 // batch))
        budget = rng.randint(max(1, hi // 8), hi)
        sinks = min(rng.choice((0, 1, 4, 16)), budget // 2)
        c = evict("", hq, hkv, batch, rng.randint(max(1, hi // 8), hi), hi, budget, sinks, rng.randint(0, budget - sinks), kv=rng.choice(("same", "same", "int4")),
                  **more)
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


def work(c):
    hq, hkv = c["q_heads"], c["kv_heads"]
    row16, row4 = hkv * 2 * D * 2, hkv * 2 * (D // 2 + 4)   # a token's K and V
    row = row4 if c["kv"] == "int4" else row16
    if c["kind"] == "chunk":
        lens = _prompts(c)
        new, cached = sum(n for n, _ in lens), sum(p for _, p in lens)
        return {"bytes": new * (row16 + row4) + cached * row4 + (new + cached) * row16, "flops": 8 * new * hkv * D}
    ctx = _spread(c["ctx_lo"], c["ctx_hi"], c["batch"])
    ids = sum(-(-t // c["block_size"]) for t in ctx) * 4
    if c["kind"] == "evict":
        # The weights of all, the rows of the keys that stay; what is read back (4-bit caches), in 16 bits.
        kept = [min(t, c["budget"]) for t in ctx]
        return {"bytes": (sum(ctx) + sum(kept)) * hkv * 4 + sum(kept) * (2 * row + (row16 if c["kv"] == "int4" else 0)) + ids, "flops": sum(ctx) * hkv}
    sums = 2 * 4 * hkv * sum(ctx) if c["kind"] == "weights" else 0
    return {"bytes": sum(ctx) * row + sums + 2 * c["batch"] * hq * D * 2 + c["batch"] * (row16 + row) + ids, "flops": 4 * hq * D * sum(ctx)}


# ---- inputs -----------------------------------------------------------------------------------------------------------------

class _State:
    pass


class _Maker:
    """Seeded inputs on the GPU and the host-side metadata of a step."""

    def __init__(self, c, seed):
        self.c, self.rng, self.order = c, np.random.default_rng(seed), random.Random(seed)
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)
        self.dtype = DTYPES[c["dtype"]]
        self.index = torch.int64 if c["index"] == "i64" else torch.int32

    def normal(self, *shape, std=1.0, mean=0.0, dtype=None):
        return torch.empty(shape, device="cuda", dtype=dtype or self.dtype).normal_(mean, std, generator=self.gen)

    def up(self, a, dtype=torch.int32):
        return torch.from_numpy(np.ascontiguousarray(a)).to("cuda", dtype)

    def shuffled(self, v):
        v = list(v)
        self.order.shuffle(v)
        return v

    def tables(self, need):
        """Block tables of sequences of so many blocks, a random permutation of the pool."""
        perm, at = self.rng.permutation(sum(need)), 0
        out = np.zeros((len(need), max(need)), np.int64)
        for i, n in enumerate(need):
            out[i, :n] = perm[at:at + n]
            at += n
        return out

    def cache(self, s, blocks):
        """A cache of normal keys and values; of a 4-bit one the numbers and the steps and lowest values that go with them."""
        shape = blocks, self.c["block_size"], self.c["kv_heads"]
        s.k_params = s.v_params = None
        if self.c["kv"] == "same":
            s.k_cache, s.v_cache = self.normal(*shape, D), self.normal(*shape, D)
            return
        s.k_cache, s.v_cache = (torch.randint(0, 256, (*shape, D // 2), device="cuda", dtype=torch.uint8, generator=self.gen) for _ in range(2))
        s.k_params, s.v_params = (torch.stack([self.normal(*shape, std=0.02, mean=0.3), self.normal(*shape, std=0.3, mean=-2.25)], -1) for _ in range(2))


def _slots(tables, seq, pos, bs):
    return tables[seq, pos // bs] * bs + pos % bs


def prepare(case, seed):
    c, m, s = case, _Maker(case, seed), _State()
    hq, hkv, b, bs = c["q_heads"], c["kv_heads"], c["batch"], c["block_size"]
    s.c, s.scale, s.workspace = c, 1.0 / math.sqrt(D), None
    if c["kind"] == "chunk":
        lens = m.shuffled(_prompts(c))
        new, total = np.array([n for n, _ in lens]), np.array([n + p for n, p in lens])
        seq, pos = np.repeat(np.arange(b), new), np.concatenate([np.arange(t - n, t) for n, t in zip(new, total)])
    else:
        total = np.array(m.shuffled(_spread(c["ctx_lo"], c["ctx_hi"], b)))
        seq, pos = np.arange(b), total - 1
    need = [-(-int(t) // bs) for t in total]
    kept = np.minimum(total, c["budget"]) if c["kind"] == "evict" else total
    tables = m.tables(need + [-(-int(t) // bs) for t in kept]) if c["kind"] == "evict" else m.tables(need)
    m.cache(s, int(tables.max()) + 1)
    s.lens, s.tables = m.up(total, m.index), m.up(tables[:b], m.index)
    s.longest, s.rows = int(total.max()), int(kept.sum())
    # Where the rows of all (kept) keys lie, sequence after sequence: what a gather brings together.
    s.cu = m.up(np.concatenate([[0], np.cumsum(kept)]), m.index)
    s.row_seq = m.up(np.repeat(np.arange(b), kept), torch.int64)
    s.row_pos = m.up(np.concatenate([np.arange(t) for t in kept]), torch.int64)
    if c["kind"] == "evict":
        s.new_tables, s.new_lens = m.up(tables[b:, :-(-int(kept.max()) // bs)], m.index), torch.empty_like(s.lens)
        # Attention falls on few keys: sums of weights over a long-tailed range.
        s.weights = m.normal(b, hkv, tables.shape[1] * bs, std=2.0, dtype=torch.float32).exp_()
        s.new_weights = torch.zeros_like(s.weights)
    else:
        s.k, s.v = m.normal(len(pos), hkv, D), m.normal(len(pos), hkv, D)
        s.slots = m.up(_slots(tables, seq, pos, bs))
    if c["kv"] == "int4" and c["kind"] in ("chunk", "evict"):
        s.key, s.value = (torch.empty((s.rows, hkv, D), device="cuda", dtype=m.dtype) for _ in range(2))
    if c["kind"] in ("decode", "weights"):
        s.q, s.out = m.normal(b, hq, D), torch.empty((b, hq, D), device="cuda", dtype=m.dtype)
    if c["kind"] == "weights":   # what some steps have left
        s.weights = m.normal(b, hkv, tables.shape[1] * bs, std=2.0, dtype=torch.float32).exp_().mul_(hq / hkv / s.longest)
        s.new_weights = torch.zeros_like(s.weights)
    return s


# ---- the operators in plain form --------------------------------------------------------------------------------------------

def _quantise(x):
    """(bytes, (step, low)) of head vectors; in 64 bits, where a value can lie next to the border between two numbers."""
    lo, hi = x.float().amin(-1, keepdim=True), x.float().amax(-1, keepdim=True)
    span = hi - lo
    step = (span / LEVELS).to(x.dtype)
    fine = torch.isfinite(span)
    n = torch.floor((x.double() - lo.double()) / step.double() + 0.5).clamp(max=LEVELS)
    n = torch.where(fine & (step > 0), n, 0.0).to(torch.uint8)
    params = torch.cat([step, lo.to(x.dtype)], -1)
    return n[..., 0::2] | (n[..., 1::2] << 4), torch.where(fine, params, math.nan)


def _values(data, params):
    n = torch.stack([data & 15, data >> 4], -1).flatten(-2).float()
    return params[..., 1:].float() + params[..., :1].float() * n


def _store(s):
    """The new rows into the cache; slots are those of the plan, all of them in the cache."""
    at = s.slots.long()
    for new, cache, params in ((s.k, s.k_cache, s.k_params), (s.v, s.v_cache, s.v_params)):
        if params is None:
            cache.flatten(0, 1)[at] = new
        else:
            cache.flatten(0, 1)[at], params.flatten(0, 1)[at] = _quantise(new)


def _row_of(tables, pos, bs):
    """Cache rows of the positions `pos` [batch, n] of every sequence."""
    return tables.long().gather(1, pos // bs) * bs + pos % bs


def _contexts(s, cache, params):
    """All sequences' rows in 32 bits, [batch, longest, heads, D]; behind a sequence's end those of some other row."""
    pos = torch.arange(s.longest, device="cuda").expand(s.lens.shape[0], -1)
    rows = _row_of(s.tables, pos, s.c["block_size"])
    if params is None:
        return cache.flatten(0, 1)[rows].float()
    return _values(cache.flatten(0, 1)[rows], params.flatten(0, 1)[rows])


def _attend(s):
    """(output, probabilities [batch, KV heads, group, longest])"""
    hkv = s.c["kv_heads"]
    q = s.q.float().unflatten(1, (hkv, -1))
    scores = torch.einsum("bjgd,bljd->bjgl", q, _contexts(s, s.k_cache, s.k_params)) * s.scale
    hidden = torch.arange(s.longest, device="cuda") >= s.lens[:, None, None, None]
    p = torch.exp(scores.masked_fill(hidden, -math.inf) - scores.masked_fill(hidden, -math.inf).amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    return torch.einsum("bjgl,bljd->bjgd", p, _contexts(s, s.v_cache, s.v_params)).flatten(1, 2).to(s.q.dtype), p


def _gather(s, tables):
    rows = tables.long()[s.row_seq, s.row_pos // s.c["block_size"]] * s.c["block_size"] + s.row_pos % s.c["block_size"]
    return tuple(_values(cache.flatten(0, 1)[rows], params.flatten(0, 1)[rows]).to(params.dtype)
                 for cache, params in ((s.k_cache, s.k_params), (s.v_cache, s.v_params)))


def _evict(s):
    c, n = s.c, s.weights.shape[-1]
    pos, lens = torch.arange(n, device="cuda"), s.lens[:, None, None]
    new_lens = lens.clamp(max=c["budget"])
    # The first and the last before the others, what is not there behind them; of equal weights the lower index first.
    rank = torch.where((pos < c["sinks"]) | (pos >= lens - c["recent"]), math.inf, s.weights)
    rank = torch.where(pos < lens, rank, -math.inf)
    kept = torch.zeros_like(rank, dtype=torch.bool).scatter_(2, torch.sort(rank, dim=-1, descending=True, stable=True)[1], pos < new_lens.expand_as(rank))
    to = torch.arange(s.new_tables.shape[1] * c["block_size"], device="cuda")
    order = torch.sort((~kept).to(torch.uint8), dim=-1, stable=True)[1][..., :len(to)]   # kept keys, in their order
    s.new_weights.zero_()
    s.new_weights[..., :len(to)] = torch.where(to < new_lens, s.weights.gather(2, order), 0.0)
    # (Places behind a sequence's end repeat its last key.)
    to = torch.minimum(to, new_lens[:, 0] - 1)
    order = order.gather(2, to[:, None].expand_as(order))
    from_rows = _row_of(s.tables, order.flatten(1), c["block_size"]).view_as(order)
    to_rows, head = _row_of(s.new_tables, to, c["block_size"])[:, None].expand_as(order), torch.arange(c["kv_heads"], device="cuda")[:, None].expand_as(order)
    _move(s.k_cache, to_rows, from_rows, head)
    _move(s.v_cache, to_rows, from_rows, head)
    if s.k_params is not None:
        _move(s.k_params, to_rows, from_rows, head)
        _move(s.v_params, to_rows, from_rows, head)
    s.new_lens.copy_(new_lens[:, 0, 0])


def _move(cache, to_rows, from_rows, head):
    rows = cache.flatten(0, 1)
    rows[to_rows, head] = rows[from_rows, head]


# ---- one pass ---------------------------------------------------------------------------------------------------------------

def _state(s):
    """What a step leaves in the cache: its rows, or the steps and lowest values (the 4-bit numbers between them show in the output)."""
    return (s.k_cache, s.v_cache) if s.c["kv"] == "same" else (s.k_params, s.v_params)


def _own(s):
    """One pass by this library."""
    nvk = importlib.import_module("nano-vllm-cpp_b200")
    c = s.c
    kind, shape, b = c["kind"], (c["kv_heads"], D, c["block_size"]), c["batch"]
    cache = s.k_cache, s.v_cache, s.k_params, s.v_params
    if kind == "evict":
        nvk.evict_kvcache(*cache, s.weights, None, s.lens, s.tables, s.new_weights, s.new_tables, s.new_lens, *shape, c["budget"], c["sinks"], c["recent"])
        if c["kv"] == "same":
            return s.k_cache, s.v_cache, s.new_weights, s.new_lens
        nvk.gather_kvcache_int4(*cache, s.cu, s.new_tables, *shape, s.key, s.value)
        return s.key, s.value, s.new_weights, s.new_lens
    if c["kv"] == "same":
        nvk.store_kvcache(s.k, s.v, s.k_cache, s.v_cache, s.slots)
    else:
        nvk.store_kvcache_int4(s.k, s.v, *cache, s.slots)
    if kind == "chunk":
        nvk.gather_kvcache_int4(*cache, s.cu, s.tables, *shape, s.key, s.value)
        return s.key, s.value
    if s.workspace is None:   # kept from the first step on
        size = nvk.decode_attention_weights_workspace_bytes if kind == "weights" else nvk.decode_attention_workspace_bytes
        s.workspace = torch.empty(max(16, size(b, c["q_heads"], c["kv_heads"], D, s.tables.shape[1], c["block_size"])), dtype=torch.uint8, device="cuda")
    if kind == "weights":
        nvk.launch_decode_attention_paged_weights(s.q, *cache, s.lens, s.tables, *shape, s.scale, s.weights, None, s.new_weights, s.out, s.workspace)
        return (s.out, *_state(s), s.new_weights)
    nvk.launch_decode_attention_paged_int4(s.q, *cache, s.lens, s.tables, *shape, s.scale, s.out, s.workspace)
    return (s.out, *_state(s))


def run(s):
    if own:
        return _own(s)
    kind = s.c["kind"]
    if kind == "evict":
        _evict(s)
        return (s.k_cache, s.v_cache, s.new_weights, s.new_lens) if s.c["kv"] == "same" else (*_gather(s, s.new_tables), s.new_weights, s.new_lens)
    _store(s)
    if kind == "chunk":
        return _gather(s, s.tables)
    out, p = _attend(s)
    if kind == "decode":
        return (out, *_state(s))
    seen = torch.arange(s.longest, device="cuda") < s.lens[:, None, None]
    s.new_weights[..., :s.longest] = torch.where(seen, s.weights[..., :s.longest] + p.sum(2), s.new_weights[..., :s.longest])
    return (out, *_state(s), s.new_weights)


# ---- the same from the definitions, in 64 bits --------------------------------------------------------------------------------

class _Exact:
    """Key and value rows of single sequences in 64 bits, the step's new rows among them as the format has them."""

    def __init__(self, s):
        self.s, self.bs = s, s.c["block_size"]
        self.lens, self.tables = s.lens.tolist(), s.tables.long()
        self.caches = [self.with_new(*x) for x in ((s.k_cache, s.k_params, getattr(s, "k", None)), (s.v_cache, s.v_params, getattr(s, "v", None)))]

    def with_new(self, cache, params, new):
        cache = cache.reshape(-1, *cache.shape[2:]).clone()
        if params is None:
            if new is not None:
                cache[self.s.slots.long()] = new
            return cache, None, None
        params = params.reshape(-1, *params.shape[2:]).clone()
        if new is None:
            return cache, params, None
        x = new.to(torch.float64)
        low, top = x.min(-1).values[..., None], x.max(-1).values[..., None]
        step = ((top - low) / LEVELS).to(torch.float32).to(new.dtype).to(torch.float64)
        number = torch.where(step > 0, torch.floor((x - low) / torch.where(step > 0, step, 1.0) + 0.5), torch.zeros_like(x))
        values = low + step * number.clamp(0, LEVELS)
        params[self.s.slots.long()] = torch.cat([step, low], -1).to(new.dtype)
        at = torch.full((cache.shape[0],), -1, dtype=torch.int64, device=cache.device)
        at[self.s.slots.long()] = torch.arange(new.shape[0], device=cache.device)
        return cache, params, (at, values)

    def rows(self, which, at):
        """Rows `at` of the keys (0) or of the values (1)."""
        cache, params, new = self.caches[which]
        if params is None:
            return cache[at].to(torch.float64)
        data, p = cache[at].to(torch.int64), params[at].to(torch.float64)
        n = torch.empty((*data.shape[:-1], D), dtype=torch.float64, device=data.device)
        n[..., 0::2], n[..., 1::2] = (data % 16).to(torch.float64), (data // 16).to(torch.float64)
        x = p[..., 0, None] * n + p[..., 1, None]
        if new is not None:
            fresh = new[0][at]
            x = torch.where((fresh >= 0)[:, None, None], new[1][fresh.clamp(min=0)], x)
        return x

    def places(self, i, tables=None, length=None):
        pos = torch.arange(self.lens[i] if length is None else length, device=self.tables.device)
        return (self.tables if tables is None else tables)[i][pos // self.bs] * self.bs + pos % self.bs


def exact(case, seed):
    s = prepare(case, seed)
    c, e = s.c, _Exact(s)
    hkv, b = c["kv_heads"], c["batch"]
    if c["kind"] == "chunk":
        at = torch.cat([e.places(i) for i in range(b)])
        return e.rows(0, at), e.rows(1, at)
    if c["kind"] == "evict":
        return _exact_evict(s, e)
    out = torch.empty((b, hkv, c["q_heads"] // hkv, D), dtype=torch.float64, device="cuda")
    sums = s.new_weights.to(torch.float64) if c["kind"] == "weights" else None
    for i in range(b):
        at = e.places(i)
        keys, values = e.rows(0, at).transpose(0, 1), e.rows(1, at).transpose(0, 1)
        p = torch.softmax(s.q[i].to(torch.float64).reshape(hkv, -1, D) @ keys.transpose(1, 2) / math.sqrt(D), -1)
        out[i] = p @ values
        if sums is not None:
            sums[i, :, :len(at)] = s.weights[i, :, :len(at)].to(torch.float64) + p.sum(1)
    state = [x[0].view_as(s.k_cache) if c["kv"] == "same" else x[1].view_as(s.k_params) for x in e.caches]
    return (out.reshape(b, c["q_heads"], D), *state, *([] if sums is None else [sums]))


def _exact_evict(s, e):
    c = s.c
    hkv, budget = c["kv_heads"], c["budget"]
    weights, new_tables = s.weights.cpu().numpy().astype(np.float64), s.new_tables.long()
    new_weights, new_lens = np.zeros_like(weights), [min(n, budget) for n in e.lens]
    k, v = (x[0].clone() for x in e.caches)
    dense = [[], []]
    for i, n in enumerate(e.lens):
        places = e.places(i)
        to = e.places(i, new_tables, new_lens[i])
        picked = []
        for j in range(hkv):
            keep = np.arange(n)
            if n > budget:
                first, last = keep[:c["sinks"]], keep[n - c["recent"]:]
                middle = keep[c["sinks"]:n - c["recent"]]
                best = np.lexsort((middle, -weights[i, j, middle]))[:budget - len(first) - len(last)]
                keep = np.sort(np.concatenate([first, middle[best], last]))
            new_weights[i, j, :len(keep)] = weights[i, j, keep]
            picked.append(places[torch.from_numpy(keep).to("cuda")])
            if c["kv"] == "same":
                k[to, j], v[to, j] = e.caches[0][0][picked[j], j], e.caches[1][0][picked[j], j]
        if c["kv"] != "same":
            for which in (0, 1):
                dense[which].append(torch.stack([e.rows(which, picked[j])[:, j] for j in range(hkv)], 1))
    tail = torch.from_numpy(new_weights).to("cuda"), torch.tensor(new_lens, device="cuda", dtype=s.lens.dtype)
    if c["kv"] == "same":
        return (k.view_as(s.k_cache), v.view_as(s.v_cache), *tail)
    return (torch.cat(dense[0]), torch.cat(dense[1]), *tail)
