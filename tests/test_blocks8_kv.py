"""8-bit paged KV cache with scales of blocks: nvk_store_kvcache_blocks8, nvk_gather_kvcache_blocks8, nvk_decode_attention_paged_blocks8.

The reference has no such cache, so the format is pinned by the 64-bit restatement of its definition in ref_blocks8.py (checked by hand on the CPU): the
store and the gather bit for bit, the decode within what its roundings allow."""
import ctypes

import numpy as np
import pytest

import ref_blocks8 as ref
from util import entry, nvk

D = 128
TINY = {"bfloat16": 2.0 ** -134, "float16": 2.0 ** -25}       # half of the smallest number


@pytest.fixture(scope="module")
def built():
    entry.build()
    return nvk()


# ---- on the CPU --------------------------------------------------------------------------------------------------------------
def test_scales_by_hand():
    for kind, top in ref.TOP.items():
        a = np.array([0.0, top, top * 1.0001, top / 2, top / 2 * 1.0001, 1.0, 2.0 ** -133, np.inf, np.nan, 3.3895313892515355e38])
        s = ref.scale_for(a, kind)
        assert s[:5].tolist() == [2.0 ** -126, 1.0, 2.0, 0.5, 1.0] and s[6] == 2.0 ** -126 and np.isnan(s[7:9]).all()
        assert s[5] == (2.0 ** -6 if kind == "int8" else 2.0 ** -8) and s[9] == (2.0 ** 122 if kind == "int8" else 2.0 ** 120)


def test_elements_by_hand():
    assert ref.nearest([0.5, 1.5, -2.5, 126.5, np.nan], "int8").tolist() == [0, 2, -2, 126, 0]
    x = ref.nearest([0.0, 1.0625, 1.1875, 2.0 ** -10, 2.0 ** -9, 1.5 * 2.0 ** -9, 447.0, 432.0, -17.0], "e4m3")
    assert x.tolist() == [0.0, 1.0, 1.25, 0.0, 2.0 ** -9, 2.0 ** -8, 448.0, 448.0, -16.0]   # (432 and -17 lie between two: to the even one)


def test_a_block_that_grows():
    c = ref.Cache(2, 4, 1, "int8")
    row = lambda v: np.full((1, 1, D), v)
    c.store(row(127.0), [0, 1], [1], [[1]])
    assert c.scale[1, 0] == 1.0 and c.data[1, 0, 0, 0] == 127
    c.store(row(129.0), [0, 1], [2], [[1]])
    assert c.scale[1, 0] == 2.0 and c.data[1, 0, 0, 0] == 64 and c.data[1, 1, 0, 0] == 64     # 63.5 and 64.5, to even
    c.store(row(1.0), [0, 1], [3], [[1]])
    assert c.scale[1, 0] == 2.0 and c.data[1, 2, 0, 0] == 0
    c.store(row(np.inf), [0, 1], [4], [[1]])
    assert np.isnan(c.rows([1], 4)).all()
    c.store(row(3.0), [0, 1], [1], [[1]])                                                     # anew
    assert c.scale[1, 0] == 2.0 ** -5 and c.rows([1], 1)[0, 0, 0] == 3.0


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_less_than_a_step_off(kind):
    """However often a block grew: int8 by less than one step, e4m3 by less than twice its half step (or by one step of its smallest numbers)."""
    rng = np.random.default_rng(5)
    c = ref.Cache(1, 64, 2, kind)
    x = rng.standard_normal((64, 2, D)) * 2.0 ** np.linspace(-4, 4, 64)[:, None, None]
    for i in range(64):
        c.store(x[i:i + 1], [0, 1], [i + 1], [[0]])
    step = c.scale[0][:, None]
    most = step if kind == "int8" else np.maximum(np.abs(x) * 2.0 ** -3, step * 2.0 ** -9)
    assert (np.abs(c.rows([0], 64) - x) < most).all()


def _call(lib, name, *args):
    rc = getattr(lib.lib(), name)(*args)
    return rc, lib.lib().nvk_last_error().decode()


L, I = ctypes.c_int64, ctypes.c_int
P, ODD = ctypes.c_void_p(256), ctypes.c_void_p(264)


def _store_args(**change):
    a = dict(key=P, value=P, ks=L(256), vs=L(256), k_cache=P, v_cache=P, k_scale=P, v_scale=P, kind=I(5), cu=P, cu_dtype=I(3), ctx=P, ctx_dtype=I(3), bt=P, bt_dtype=I(4),
             seqs=L(2), total=L(5), max_blocks=L(3), blocks=L(4), hkv=I(2), d=I(128), bs=I(16), dtype=I(1), stream=None)
    a.update(change)
    return a.values()


def _gather_args(**change):
    a = dict(k_cache=P, v_cache=P, k_scale=P, v_scale=P, kind=I(6), cu=P, cu_dtype=I(3), bt=P, bt_dtype=I(4), seqs=L(2), total=L(10), max_blocks=L(2), blocks=L(4),
             hkv=I(2), d=I(128), bs=I(16), key=P, value=P, dtype=I(0), stream=None)
    a.update(change)
    return a.values()


def _decode_args(**change):
    a = dict(q=P, k_cache=P, v_cache=P, k_scale=P, v_scale=P, kind=I(5), ctx=P, ctx_dtype=I(3), bt=P, bt_dtype=I(3), batch=L(2), max_blocks=L(40), blocks=L(4), hq=I(8),
             hkv=I(2), d=I(128), bs=I(256), scale=ctypes.c_float(1.0), out=P, dtype=I(1), ws=None, ws_bytes=ctypes.c_size_t(0), stream=None)
    a.update(change)
    return a.values()


@pytest.mark.parametrize("change,code,word", [
    (dict(key=None), 1, "defined"), (dict(v_scale=None), 1, "defined"), (dict(bt=None), 1, "defined"), (dict(kind=I(1)), 1, "int8 or e4m3"), (dict(dtype=I(2)), 3, "F16 or BF16"),
    (dict(d=I(64)), 3, "128"), (dict(hkv=I(0)), 1, "positive"), (dict(ctx_dtype=I(5)), 1, "int32 or int64"), (dict(cu_dtype=I(1)), 1, "int32 or int64"),
    (dict(seqs=L(-1)), 1, "positive"), (dict(blocks=L(0)), 1, "positive"), (dict(bs=I(0)), 1, "positive"), (dict(cu=None), 1, "one row for every"),
    (dict(ks=L(248)), 1, "strides"), (dict(vs=L(260)), 1, "strides"), (dict(key=ODD), 1, "aligned"), (dict(k_scale=ctypes.c_void_p(258)), 1, "aligned"),
    (dict(total=L(1 << 31)), 3, "too many"), (dict(max_blocks=L(1 << 30)), 3, "too many"), (dict(seqs=L(1 << 30)), 3, "too many"), (dict(total=L(0)), 0, ""),
    (dict(seqs=L(0)), 0, "")])
def test_store_refuses(built, change, code, word):
    rc, said = _call(built, "nvk_store_kvcache_blocks8", *_store_args(**change))
    assert rc == code and (rc == 0 or word in said), said


@pytest.mark.parametrize("change,code,word", [
    (dict(cu=None), 1, "defined"), (dict(k_scale=None), 1, "defined"), (dict(kind=I(0)), 1, "int8 or e4m3"), (dict(dtype=I(2)), 3, "F16 or BF16"), (dict(d=I(256)), 3, "128"),
    (dict(cu_dtype=I(0)), 1, "int32 or int64"), (dict(seqs=L(0)), 1, "positive"), (dict(total=L(-1)), 1, "positive"), (dict(max_blocks=L(0)), 1, "positive"),
    (dict(value=ODD), 1, "aligned"), (dict(total=L(0)), 0, ""), (dict(total=L(1 << 40)), 3, "too many")])
def test_gather_refuses(built, change, code, word):
    rc, said = _call(built, "nvk_gather_kvcache_blocks8", *_gather_args(**change))
    assert rc == code and (rc == 0 or word in said), said


@pytest.mark.parametrize("change,code,word", [
    (dict(q=None), 1, "requires"), (dict(v_scale=None), 1, "requires"), (dict(kind=I(4)), 1, "int8 or e4m3"), (dict(scale=ctypes.c_float(float("inf"))), 1, "finite"),
    (dict(scale=ctypes.c_float(float("nan"))), 1, "finite"), (dict(ctx_dtype=I(1)), 1, "int32 or int64"),
    (dict(batch=L(-1)), 1, "positive"), (dict(hq=I(7)), 1, "divisible"), (dict(dtype=I(2)), 3, "F16 / BF16"), (dict(d=I(64)), 3, "head_dim"),
    (dict(hq=I(18)), 3, "8 query heads"), (dict(bs=I(24)), 3, "multiple"), (dict(q=ODD), 3, "aligned"), (dict(ws=P, ws_bytes=ctypes.c_size_t(64)), 1, "workspace"),
    (dict(ws=ODD, ws_bytes=ctypes.c_size_t(1 << 30)), 1, "aligned"), (dict(batch=L(0)), 0, "")])
def test_decode_refuses(built, change, code, word):
    rc, said = _call(built, "nvk_decode_attention_paged_blocks8", *_decode_args(**change))
    assert rc == code and (rc == 0 or word in said), said


# ---- on the GPU --------------------------------------------------------------------------------------------------------------
def _typed(x, dtype):
    """float64 -> the 16-bit type, on the GPU, and as float64 again."""
    import torch
    t = torch.from_numpy(np.ascontiguousarray(x, np.float64)).to(getattr(torch, dtype))
    return t.cuda(), t.double().numpy()


class Both:
    """K and V caches on the GPU and here."""

    def __init__(self, blocks, bs, hkv, kind, garbage=True):
        import torch
        self.kind, self.bs, self.hkv, self.blocks = kind, bs, hkv, blocks
        self.ref = [ref.Cache(blocks, bs, hkv, kind) for _ in range(2)]
        self.data, self.scale = [], []
        for _ in range(2):   # what was there before: anything
            d = torch.randint(0, 256, (blocks, bs, hkv, D), dtype=torch.uint8, device="cuda") if garbage else torch.zeros((blocks, bs, hkv, D), dtype=torch.uint8, device="cuda")
            self.data.append(d.view(torch.int8 if kind == "int8" else torch.float8_e4m3fn))
            self.scale.append(torch.full((blocks, hkv), 2.0 ** 60 if garbage else 0.0, device="cuda"))
        self.seen = {}       # rows of a block that mean something

    def store(self, x, cu, lens, tables, index="int32", one=False):
        """x: (k, v) on the GPU and here."""
        import torch
        up = lambda v: torch.as_tensor(np.asarray(v), dtype=getattr(torch, index)).cuda()
        behind = [d.view(torch.uint8).clone() for d in self.data]
        nvk().store_kvcache_blocks8(x[0][0], x[1][0], *self.data, *self.scale, None if one else up(cu), up(lens), up(tables))
        for w in range(2):
            for block in self.ref[w].store(x[w][1], cu, lens, tables):
                self.seen[block] = 0
        for s, total in enumerate(lens):
            for pos in range(max(int(total) - (cu[s + 1] - cu[s]), 0), int(total)):
                if pos // self.bs < len(tables[s]) and 0 <= tables[s][pos // self.bs] < self.blocks:
                    self.seen[int(tables[s][pos // self.bs])] = pos % self.bs + 1
        self.same(behind)

    def same(self, behind):
        import torch
        for w in range(2):
            got, scale = self.data[w].double() if self.kind == "int8" else self.data[w].float().double(), self.scale[w].double().cpu().numpy()
            got = got.cpu().numpy()
            for block in range(self.blocks):
                n = self.seen.get(block, 0)
                if n:
                    assert np.array_equal(scale[block], self.ref[w].scale[block], equal_nan=True), (w, block, scale[block], self.ref[w].scale[block])
                    assert np.array_equal(got[block, :n], self.ref[w].data[block, :n], equal_nan=True), (w, block)
                # rows behind the last one, and blocks of nobody
                assert torch.equal(self.data[w].view(torch.uint8)[block, n:], behind[w][block, n:]), (w, block)


def _tables(rng, need, width, blocks):
    perm, out, at = rng.permutation(blocks), np.full((len(need), width), -1, np.int64), 0
    for i, n in enumerate(need):
        out[i, :n] = perm[at:at + n]
        at += n
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("bs,hkv,index", [(16, 1, "int32"), (16, 8, "int64"), (64, 3, "int32"), (256, 2, "int32"), (48, 2, "int64"), (512, 1, "int32"), (8, 5, "int32")])
def test_store_in_several_steps(kind, dtype, bs, hkv, index):
    """Prompts, then chunks and single rows that join blocks and raise their scales."""
    rng = np.random.default_rng(bs + hkv)
    seqs = 5
    need = [6] * seqs
    blocks = sum(need) + 2
    c = Both(blocks, bs, hkv, kind)
    tables = _tables(rng, need, 6, blocks)
    lens = np.zeros(seqs, np.int64)
    for step in range(7):
        one = step >= 4
        new = np.ones(seqs, np.int64) if one else rng.integers(0, bs + 5, seqs)
        if step == 0:
            new[:] = [0, 1, bs, bs + 1, 2 * bs + 3]
        lens = np.minimum(lens + new, 6 * bs)
        new = np.minimum(new, lens)
        cu = np.concatenate([[0], np.cumsum(new)]).tolist()
        x = [_typed(rng.standard_normal((cu[-1], hkv, D)) * 2.0 ** rng.uniform(-2, 1 + step, (cu[-1], 1, 1)), dtype) for _ in range(2)]
        c.store(x, cu, lens.tolist(), tables.tolist(), index, one)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype", [("int8", "bfloat16"), ("int8", "float16"), ("e4m3", "bfloat16"), ("e4m3", "float16")])
@pytest.mark.parametrize("bs,hkv,first,then", [(16, 8, (0, 37, 5000, 16), (5100, 0, 300, 1)), (64, 3, (9000, 700, 1), (63, 10500, 64)), (256, 4, (9000, 255, 1000), (300, 9400, 25)),
                                               (8, 5, (2600,), (2700,)), (48, 1, (31000, 5), (20, 30100))])
def test_store_of_many_rows(kind, dtype, bs, hkv, first, then):
    """More blocks of threads than two to an SM, twice: the second step joins blocks of the first one with larger rows."""
    rng = np.random.default_rng(bs + hkv)
    need = [-(-(a + b) // bs) for a, b in zip(first, then)]
    c, tables, total = Both(sum(need) + 3, bs, hkv, kind), _tables(rng, need, max(need), sum(need) + 3), np.zeros(len(first), np.int64)
    for size, new in ((1.0, first), (5.0, then)):
        cu, total = [0, *np.cumsum(new).tolist()], total + np.array(new)
        c.store([_typed(rng.standard_normal((cu[-1], hkv, D)) * size, dtype) for _ in range(2)], cu, total.tolist(), tables)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_store_of_hard_values(kind, dtype):
    """Zeros, borders between elements and between scales, the largest and the smallest numbers, infinities and NaN, alone and joining a block."""
    rng = np.random.default_rng(9)
    tiny, huge = {"bfloat16": (2.0 ** -133, 3.3895313892515355e38), "float16": (2.0 ** -24, 65504.0)}[dtype]
    top = ref.TOP[kind]
    vectors = [np.zeros(D), np.full(D, -top), np.full(D, top), np.arange(D) - 64.0, (np.arange(D) - 64) * 0.5, np.full(D, 128.0 if kind == "int8" else 464.0),
               np.arange(D) % 7 * tiny, -np.arange(D) * 16 * tiny, np.where(np.arange(D) % 2, huge, -huge), np.arange(D) * huge / 200, np.full(D, 2.0 ** -9),
               np.where(np.arange(D) == 5, np.inf, 1.0), np.where(np.arange(D) == 127, np.nan, 2.0), np.where(np.arange(D) == 0, -np.inf, 0.0), np.full(D, 1.0)]
    n = len(vectors)
    # each pair of vectors, one joining the other in a block of its own, as one call and as two
    pairs = [(a, b) for a in vectors for b in vectors]
    x = np.asarray(pairs).reshape(-1, 1, D)
    blocks = len(pairs)
    tables = np.arange(blocks)[:, None]
    both = [_typed(x, dtype), _typed(x[::-1], dtype)]
    c = Both(blocks, 16, 1, kind)
    c.store(both, list(range(0, 2 * blocks + 1, 2)), [2] * blocks, tables.tolist())
    c = Both(blocks, 16, 1, kind)
    for i in range(2):
        part = [(t.view(blocks, 2, 1, D)[:, i].contiguous(), v.reshape(blocks, 2, 1, D)[:, i]) for t, v in both]
        c.store(part, list(range(blocks + 1)), [i + 1] * blocks, tables.tolist(), one=i == 1)


@pytest.mark.gpu
def test_store_skips_what_has_no_place():
    """Negative positions (a request that waits), blocks outside the cache, rows beyond the table, rows behind the last sequence."""
    rng = np.random.default_rng(10)
    c = Both(6, 16, 2, "int8")
    tables = [[0, 1], [2, 99], [-1, 3], [4, 5]]
    cu, lens = [0, 5, 30, 60, 100], [0, 25, 30, 40]
    x = [_typed(rng.standard_normal((107, 2, D)), "bfloat16") for _ in range(2)]
    c.store(x, cu, lens, tables)
    assert sorted(c.seen) == [2, 3, 4, 5]
    one = [(t[:4], v[:4]) for t, v in x]
    c.store(one, [0, 1, 2, 3, 4], [0, -3, 33, 32], tables, one=True)


@pytest.mark.gpu
def test_store_of_packed_rows_and_on_another_stream():
    import torch
    rng = np.random.default_rng(11)
    hq, hkv, n, bs = 4, 2, 70, 16
    qkv, here = _typed(rng.standard_normal((n, (hq + 2 * hkv) * D)), "bfloat16")
    parts = [((slice(None), slice((hq + i * hkv) * D, (hq + (i + 1) * hkv) * D))) for i in range(2)]
    x = [(qkv[p].unflatten(1, (hkv, D)), here[p].reshape(n, hkv, D)) for p in parts]
    c = Both(8, bs, hkv, "e4m3")
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        c.store(x, [0, n], [n], [list(range(7, 2, -1))])
    one = [(t[-1:], v[-1:]) for t, v in x]
    c.store(one, [0, 1], [n + 1], [list(range(7, 2, -1))], one=True)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("bs,hkv,lens,index", [(16, 2, [40, 0, 1, 16], "int32"), (256, 1, [300], "int64"), (48, 3, [1, 47, 48, 49, 200], "int32")])
def test_gather(kind, dtype, bs, hkv, lens, index):
    import torch
    rng = np.random.default_rng(bs)
    need = [-(-n // bs) for n in lens]
    blocks, width = sum(need) + 1, max(need) + 1
    tables = _tables(rng, need, width, blocks)
    c = Both(blocks, bs, hkv, kind)
    cu = np.concatenate([[0], np.cumsum(lens)]).tolist()
    x = [_typed(rng.standard_normal((cu[-1], hkv, D)) * 2.0 ** rng.uniform(-18, 8, (cu[-1], hkv, 1)), dtype) for _ in range(2)]
    c.store(x, cu, lens, tables.tolist(), index)
    tables[-1, 0] = blocks + 5   # (reads as zeros)
    up = lambda v: torch.as_tensor(np.asarray(v), dtype=getattr(torch, index)).cuda()
    out = [torch.full((cu[-1] + 3, hkv, D), float("nan"), dtype=getattr(torch, dtype), device="cuda") for _ in range(2)]
    nvk().gather_kvcache_blocks8(*c.data, *c.scale, up(cu), up(tables), hkv, D, bs, *out)
    for w in range(2):
        want = np.concatenate([c.ref[w].rows(tables[s], n) for s, n in enumerate(lens)] + [np.zeros((3, hkv, D))])
        assert torch.equal(out[w].cpu().double(), torch.from_numpy(want).to(out[w].dtype).double())


# How far a decode output can be off.  A score: the query's elements (by 2^-25 of the head's largest, int8: 2^-20), 128 products summed in fp32 and 8
# operations more, each addition by 2^-23 of the sum of magnitudes at most (the MMA may cut off instead of rounding).  A weight p by a factor e^(2 score error), its
# exponential by 2^-20; p s to f16: 2^-11 of itself, or, where it is less than 2^-10 of the head's largest, 2^-22 of that; sums over the keys and the merges: 2^-23 for every one of
# some 300 operations of a chain, of the sum of magnitudes.
def _bound(c, table, n, q, scale, dtype):
    """(the output in 64 bits, how far it may be off)"""
    k, v = (r.rows(table, n) for r in c.ref)
    per = q.shape[0] // c.hkv
    kk, vv = (np.repeat(np.abs(x), per, axis=1) for x in (k, v))          # [n, Hq, D]
    score = abs(scale) * (136 * 2.0 ** -23 * np.einsum("hd,nhd->nh", np.abs(q), kk).max(0) + (2.0 ** -25 if c.kind == "e4m3" else 2.0 ** -20) * np.abs(q).max(-1) * kk.sum(-1).max(0))
    s = np.einsum("hd,nhd->hn", q, np.repeat(k, per, axis=1)) * scale
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    want, mags = (np.einsum("hn,nhd->hd", p, x) for x in (np.repeat(v, per, axis=1), vv))
    blocks = np.array([table[i // c.bs] if i // c.bs < len(table) else -1 for i in range(n)])
    steps = np.where(((blocks >= 0) & (blocks < c.blocks))[:, None], c.ref[1].scale[np.clip(blocks, 0, c.blocks - 1)], 0.0)   # [n, Hkv]
    part = p * np.repeat(steps, per, axis=1).T                               # [Hq, n]
    most = part.max(-1, keepdims=True)
    numbers = np.repeat(np.divide(np.abs(v), steps[..., None], out=np.zeros_like(v), where=steps[..., None] > 0), per, axis=1)
    tail = np.einsum("hn,nhd->hd", np.where(part < most * 2.0 ** -10, most * 2.0 ** -22, 0.0), numbers)
    weight = 2 * score + 2.0 ** -11 + 2.0 ** -20 + 300 * 2.0 ** -23
    return want, weight[:, None] * mags * 1.01 + tail + np.abs(want) * ref.HALF_STEP[dtype] + TINY[dtype]


def _decode(c, q, lens, tables, index="int32", workspace=True, scale=0.09):
    import torch
    up = lambda v: torch.as_tensor(np.asarray(v), dtype=getattr(torch, index)).cuda()
    out = torch.full_like(q, float("nan"))
    b, hq = q.shape[:2]
    bt = up(tables)
    size = nvk().decode_attention_workspace_bytes(b, hq, c.hkv, D, bt.shape[1], c.bs)
    ws = torch.full((max(16, size),), 0x7f, dtype=torch.uint8, device="cuda") if workspace else None
    nvk().launch_decode_attention_paged_blocks8(q, *c.data, *c.scale, up(lens), bt, c.hkv, D, c.bs, scale, out, ws)
    return out.double().cpu().numpy()


def _check_decode(c, q, here, lens, tables, dtype, **more):
    scale = more.get("scale", 0.09)
    got = _decode(c, q, lens, tables, **more)
    for s, n in enumerate(lens):
        n = max(0, min(int(n), len(tables[s]) * c.bs))
        if n == 0:
            assert (got[s] == 0).all()
            continue
        want, most = _bound(c, tables[s], n, here[s], scale, dtype)
        assert (np.abs(got[s] - want) <= most).all(), (s, np.abs(got[s] - want).max(), (np.abs(got[s] - want) / most).max())
    return got


def _filled(rng, kind, dtype, bs, hkv, lens, width=None, spread=1.0, std=1.0):
    need = [-(-n // bs) for n in lens]
    blocks = sum(need) + 1
    tables = _tables(rng, need, width or max(max(need), 1), blocks)
    c = Both(blocks, bs, hkv, kind)
    cu = np.concatenate([[0], np.cumsum(lens)]).tolist()
    x = [_typed(rng.standard_normal((cu[-1], hkv, D)) * std * 2.0 ** rng.uniform(-spread, spread, (cu[-1], 1, 1)), dtype) for _ in range(2)]
    c.store(x, cu, lens, tables.tolist())
    return c, tables


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("bs,hq,hkv,lens,width,index", [
    (16, 32, 8, [1], None, "int32"), (256, 32, 8, [300], None, "int64"), (16, 4, 1, [15, 16, 17, 0, 33], 4, "int32"), (64, 14, 2, [700, 5, 64], 40, "int32"),
    (256, 8, 8, [1000, 2049, 1], 16, "int64"), (32, 8, 1, [3000], 128, "int32"), (16, 6, 2, [100] * 40, 9, "int32")])
def test_decode(kind, dtype, bs, hq, hkv, lens, width, index):
    rng = np.random.default_rng(hq * bs + len(lens))
    c, tables = _filled(rng, kind, dtype, bs, hkv, lens, width)
    q, here = _typed(rng.standard_normal((len(lens), hq, D)) * 2.0, dtype)
    a = _check_decode(c, q, here, lens, tables, dtype, index=index)
    _check_decode(c, q, here, lens, tables, dtype, index=index, workspace=False)
    again = _decode(c, q, lens, tables, index=index)
    assert np.array_equal(a, again)
    # one way out of the table: a length beyond it
    long = [n + 10 ** 6 for n in lens[:1]] + lens[1:]
    if len(tables[0]) == -(-lens[0] // bs) and lens[0] % bs == 0:
        assert np.array_equal(_decode(c, q, long, tables, index=index), a)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype", [("int8", "bfloat16"), ("e4m3", "float16")])
@pytest.mark.parametrize("hq,hkv,batch,width,long", [
    (8, 8, 15, 16, [1024, 900]),          # 120 pairs, 1024-key tables: whole contexts, eight warps
    (16, 8, 30, 32, [2048, 1]),           # 240 pairs, 2048 keys: the same, the longest first
    (16, 8, 20, 32, [2048, 1025]),        # 160 pairs: halves of a table row
    (2, 1, 200, 64, [4096, 769, 768]),    # chunks of 768
    (8, 8, 90, 128, [3000, 8192]),        # 720 pairs: of 1024, where the workspace has room for them
    (8, 1, 8, 64, [4096, 4095, 33])])     # clusters of eight
def test_decode_in_all_ways_of_sharing_out(kind, dtype, hq, hkv, batch, width, long):
    """Contexts of which a few fill their tables and the others end in their first blocks, none among them."""
    rng = np.random.default_rng(hq * batch)
    bs = 64
    lens = (long + [0, 1, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129] + [int(x) for x in rng.integers(1, 200, batch)])[:batch]
    rng.shuffle(lens)
    c, tables = _filled(rng, kind, dtype, bs, hkv, lens, width)
    q, here = _typed(rng.standard_normal((batch, hq, D)) * 2.0, dtype)
    got = _check_decode(c, q, here, lens, tables, dtype)
    assert np.array_equal(got, _decode(c, q, lens, tables))
    _check_decode(c, q, here, lens, tables, dtype, workspace=False)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_decode_over_scales_far_apart(kind, dtype):
    """Blocks whose values are 2^16 times the others' must not cost these their bits where hardly any attention goes to them."""
    rng = np.random.default_rng(21)
    lens = [640, 640]
    c, tables = _filled(rng, kind, dtype, 16, 2, lens, spread=0.0)
    import torch
    # values of every fifth block far larger, keys of the same blocks turned away from the query
    q = np.zeros((2, 4, D))
    q[..., 0] = 8.0
    for s in range(2):
        for j, block in enumerate(tables[s]):
            if j % 5 == 2:
                for r, w in ((c.ref[1], 1),):
                    r.scale[block] *= 2.0 ** 14
                    c.scale[w][int(block)] *= 2.0 ** 14
                c.ref[0].data[block, :, :, 0] = -100 if kind == "int8" else -96
                c.data[0].view(torch.uint8)[int(block), :, :, 0] = (256 - 100) if kind == "int8" else int(torch.tensor(-96.0).to(torch.float8_e4m3fn).view(torch.uint8))
    qd, here = _typed(q, dtype)
    _check_decode(c, qd, here, lens, tables, dtype, scale=0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("size", [2.0 ** -20, 2.0 ** -100, 2.0 ** 14, 2.0 ** -60])
def test_decode_with_queries_and_values_of_any_size(dtype, size):
    if dtype == "float16" and size < 2.0 ** -30:
        size = 2.0 ** -22
    rng = np.random.default_rng(22)
    lens = [200, 31]
    c, tables = _filled(rng, "int8", dtype, 16, 2, lens, std=min(size, 2.0 ** 10))
    q, here = _typed(rng.standard_normal((2, 8, D)) * size, dtype)
    k = max(np.abs(r.rows(tables[0], 200)).max() for r in c.ref)
    scale = float(1.0 / (size * k * 8))
    if scale > float(np.finfo(np.float32).max):   # (no number of the call's type)
        with pytest.raises(ValueError, match="finite"):
            _decode(c, q, lens, tables, scale=scale)
        return
    _check_decode(c, q, here, lens, tables, dtype, scale=scale)


@pytest.mark.gpu
def test_decode_with_keys_alike_and_long_contexts():
    """A mean over many keys, whose sums an offset of the elements would swamp."""
    import torch
    rng = np.random.default_rng(23)
    lens, bs = [9000], 256
    c, tables = _filled(rng, "int8", "float16", bs, 1, lens, width=40, spread=0.0)
    q, here = _typed(np.zeros((1, 4, D)), "float16")
    got = _check_decode(c, q, here, lens, tables, "float16")
    mean = c.ref[1].rows(tables[0], 9000)[:, 0].mean(0)
    # weights are 1 / 9000 each: f16 holds 2^-11 of p s; the errors of equal weights are alike, and go into all sums alike
    assert np.abs(got[0] - mean).max() <= np.abs(mean).max() * 2.0 ** -10 + 1e-5


@pytest.mark.gpu
def test_a_block_of_nan_is_one_sequences_and_heads_own():
    rng = np.random.default_rng(24)
    lens = [100, 100, 100]
    c, tables = _filled(rng, "int8", "bfloat16", 16, 2, lens)
    x = np.ones((3, 2, D))
    x[1, 1, 7] = np.nan
    xs = _typed(x, "bfloat16")
    c.store([xs, xs], [0, 1, 2, 3], [101] * 3, tables.tolist() if tables.shape[1] > 6 else np.pad(tables, ((0, 0), (0, 1))).tolist(), one=True)
    q, here = _typed(rng.standard_normal((3, 8, D)), "bfloat16")
    got = _decode(c, q, [101] * 3, tables if tables.shape[1] > 6 else np.pad(tables, ((0, 0), (0, 1))))
    bad = np.isnan(got)
    assert bad[1, 4:].all() and not bad[1, :4].any() and not bad[0].any() and not bad[2].any()


@pytest.mark.gpu
def test_blocks_outside_the_cache_read_as_zeros():
    rng = np.random.default_rng(25)
    lens = [64]
    c, tables = _filled(rng, "e4m3", "bfloat16", 16, 1, lens)
    tables[0, 1], tables[0, 2] = -1, 1 << 20
    q, here = _typed(rng.standard_normal((1, 4, D)), "bfloat16")
    _check_decode(c, q, here, lens, tables, "bfloat16")


@pytest.mark.gpu
@pytest.mark.parametrize("change,word", [
    (dict(k_cache="bfloat16"), "both be int8"), (dict(v_cache="uint8"), "both be int8"), (dict(k_scale="float16"), "float32"), (dict(scale_shape=(3, 2)), "every cache block"),
    (dict(ctx=3), "every context length"), (dict(value=(2, 2, 64)), "same shape"), (dict(key_dim=2), "must be \\[rows")])
def test_the_binding_refuses(change, word):
    import torch
    dt = lambda n, d: getattr(torch, change.get(n, d))
    kc, vc = torch.zeros(4, 16, 2, D, dtype=dt("k_cache", "int8"), device="cuda"), torch.zeros(4, 16, 2, D, dtype=dt("v_cache", "int8"), device="cuda")
    ks, vs = torch.zeros(change.get("scale_shape", (4, 2)), dtype=dt("k_scale", "float32"), device="cuda"), torch.zeros(4, 2, device="cuda")
    key = torch.zeros((2, 2, D) if "key_dim" not in change else (2, 2 * D), dtype=torch.bfloat16, device="cuda")
    value = torch.zeros(change.get("value", key.shape), dtype=torch.bfloat16, device="cuda")
    ctx = torch.zeros(change.get("ctx", 2), dtype=torch.int32, device="cuda")
    bt = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match=word):
        nvk().store_kvcache_blocks8(key, value, kc, vc, ks, vs, None, ctx, bt)


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [(16, 1 << 62, 1 << 10), (1 << 40, 1 << 20, 1 << 10), (1 << 32, 2, D), (16, (1 << 32) + 2, D), (16, 2, (1 << 32) + D)])
def test_the_binding_refuses_sizes_beyond_the_cache(sizes):
    import torch
    bs, hkv, d = sizes
    kc, ks = torch.zeros(4, 16, 2, D, dtype=torch.int8, device="cuda"), torch.zeros(4, 2, device="cuda")
    key, cu, bt = torch.zeros(4, 2, D, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        nvk().gather_kvcache_blocks8(kc, kc, ks, ks, cu, bt, hkv, d, bs, key, key.clone())
    with pytest.raises((ValueError, ZeroDivisionError)):   # (as the other decode calls have it)
        nvk().launch_decode_attention_paged_blocks8(key[:1].contiguous(), kc, kc, ks, ks, cu[:1], bt, hkv, d, bs, 1.0, key[:1].clone())


# ---- together ------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype", [("int8", "bfloat16"), ("e4m3", "float16")])
def test_two_streams_and_two_graphs_of_one_workspace(kind, dtype):
    """Store, gather and decode on two streams at the same time, with a workspace each; then two captured decodes that share one, replayed one after the other."""
    import torch
    rng = np.random.default_rng(41)
    hq, hkv, bs, scale, batch, width = 8, 2, 64, D ** -0.5, 3, 150
    lens = [[9000, 0, 700], [1, 5000, 64]]
    streams, work = [torch.cuda.Stream() for _ in range(2)], []
    for n in lens:
        c = Both(160, bs, hkv, kind)
        tables = _tables(rng, [-(-x // bs) for x in n], width, 160)
        cu = np.concatenate([[0], np.cumsum(n)])
        rows = [_typed(rng.standard_normal((cu[-1], hkv, D)), dtype) for _ in range(2)]
        q, q64 = _typed(rng.standard_normal((batch, hq, D)), dtype)
        for w in range(2):
            c.ref[w].store(rows[w][1], cu, n, tables)
        up = lambda v: torch.as_tensor(np.asarray(v), dtype=torch.int32).cuda()
        ws = torch.empty(max(16, nvk().decode_attention_workspace_bytes(batch, hq, hkv, D, width, bs)), dtype=torch.uint8, device="cuda")
        work.append(dict(c=c, tables=tables, rows=rows, q=q, q64=q64, cu=up(cu), n=up(n), bt=up(tables), ws=ws, out=torch.full_like(q, float("nan")),
                         dense=[torch.full_like(r[0], float("nan")) for r in rows]))

    def decode(x, ws):
        nvk().launch_decode_attention_paged_blocks8(x["q"], *x["c"].data, *x["c"].scale, x["n"], x["bt"], hkv, D, bs, scale, x["out"], ws)

    torch.cuda.synchronize()
    for s, x in zip(streams, work):
        with torch.cuda.stream(s):
            nvk().store_kvcache_blocks8(x["rows"][0][0], x["rows"][1][0], *x["c"].data, *x["c"].scale, x["cu"], x["n"], x["bt"])
            nvk().gather_kvcache_blocks8(*x["c"].data, *x["c"].scale, x["cu"], x["bt"], hkv, D, bs, *x["dense"])
            decode(x, x["ws"])
    torch.cuda.synchronize()

    def check():
        for n, x in zip(lens, work):
            for s in range(batch):
                o = x["out"][s].double().cpu().numpy()
                if n[s] == 0:
                    assert (o == 0).all()
                else:
                    w, most = _bound(x["c"], x["tables"][s], n[s], x["q64"][s], scale, dtype)
                    assert (np.abs(o - w) <= most).all()

    check()
    for x, n in zip(work, lens):
        at = 0
        for s in range(batch):
            for w in range(2):   # (what the block stands for, rounded to the type: a power of two times 8 bits, exact in both)
                assert np.array_equal(x["dense"][w][at:at + n[s]].double().cpu().numpy(), x["c"].ref[w].rows(x["tables"][s], n[s]))
            at += n[s]
    graphs, stream = [], torch.cuda.Stream()
    for x in work:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            decode(x, work[0]["ws"])
        graphs.append(g)
    for x in work:
        x["out"].fill_(float("nan"))
    torch.cuda.synchronize()
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    check()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_a_run_of_steps_from_lengths_to_outputs(kind):
    """Metadata, rotary positions, store, attention: a prefill step, then decode steps replayed as a graph, then a request that ends and one that takes its blocks."""
    import torch
    rng = np.random.default_rng(31)
    hq, hkv, bs, dtype, width, pool = 8, 2, 16, "bfloat16", 8, 40
    scale = D ** -0.5
    f = nvk().rotary_inv_freq(64, 10000.0, "yarn", 4.0, 64.0)
    freq = torch.tensor(f[0], device="cuda")
    lens, held = torch.zeros(6, dtype=torch.int32, device="cuda"), torch.full((6, width), -1, dtype=torch.int32, device="cuda")
    free, count = torch.from_numpy(rng.permutation(pool)).int().cuda(), torch.tensor([pool], dtype=torch.int32, device="cuda")
    c = Both(pool, bs, hkv, kind)
    book = ref.Requests([0] * 6, held.tolist(), free.tolist(), pool, bs)

    def metadata(batch, tokens):
        i = lambda *s: torch.full(s, -9, dtype=torch.int32, device="cuda")
        return i(batch, width), i(batch), i(batch + 1), i(batch + 1), i(tokens), i(tokens)

    def enqueue(new, rows, meta, qkv, q, k):
        nvk().step_metadata(new, rows, lens, held, free, count, bs, pool, *meta)
        parts = [qkv[:, a * D:b * D].unflatten(1, (b - a, D)) for a, b in ((0, hq), (hq, hq + hkv), (hq + hkv, hq + 2 * hkv))]
        nvk().rotary_embedding(parts[0], parts[1], meta[4], freq, False, f[1], q, k)
        return parts[2]

    def here(qkv, positions):
        x = qkv.double().cpu().numpy().reshape(len(qkv), -1, D)
        turned = ref.rotary(x[:, :hq + hkv], positions, freq.double().tolist(), False, f[1])
        return torch.from_numpy(turned).to(torch.bfloat16).double().numpy(), x[:, hq + hkv:]

    # prefill: 20, 0 and 37 tokens, two rows more than there are
    new, rows = [20, 0, 37], [4, 0, 2]
    meta = metadata(3, 59)
    qkv = torch.from_numpy(rng.standard_normal((59, (hq + 2 * hkv) * D))).to(torch.bfloat16).cuda()
    q, k = (torch.empty(59, h, D, dtype=torch.bfloat16, device="cuda") for h in (hq, hkv))
    v = enqueue(torch.tensor(new, dtype=torch.int32, device="cuda"), torch.tensor(rows, dtype=torch.int32, device="cuda"), meta, qkv, q, k)
    want = book.step(new, rows, width, 59, pool)
    assert [m.tolist() for m in meta] == list(want)
    both, v64 = here(qkv, want[4])
    # (within a step of the type, as other arithmetic may round the other way; what is stored is what the kernel made)
    assert (np.abs(torch.cat([q, k], 1).double().cpu().numpy() - both) <= np.abs(both) * 2.0 ** -7 + 2.0 ** -16).all()
    c.store([(k, k.double().cpu().numpy()), (v, v64)], want[2], want[1], want[0])
    dense = [torch.empty(57, hkv, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    nvk().gather_kvcache_blocks8(*c.data, *c.scale, meta[3], meta[0], hkv, D, bs, *dense)
    out = torch.zeros(57, hq, D, dtype=torch.bfloat16, device="cuda")
    nvk().launch_prefill_attention_dense(q[:57].contiguous(), meta[2], *dense, meta[3], hkv, D, scale, out)
    for s, (a, b) in enumerate(((0, 20), (20, 57))):
        kk, vv = (r.rows(want[0][2 * s], b - a) for r in c.ref)
        q64 = q.double().cpu().numpy()
        for i in range(a, b, 7):
            w, w_abs = ref.attend(q64[i], kk[:i - a + 1], vv[:i - a + 1], scale)
            assert np.abs(out[i].double().cpu().numpy() - w).max() <= 2.0 ** -7 * np.max(w_abs) + 2.0 ** -8 * np.abs(w).max()

    # decode steps of the two, and padding, as one graph
    rows = [2, -1, 4]
    meta = metadata(3, 3)
    new_t, rows_t = torch.ones(3, dtype=torch.int32, device="cuda"), torch.tensor(rows, dtype=torch.int32, device="cuda")
    qkv = torch.zeros(3, (hq + 2 * hkv) * D, dtype=torch.bfloat16, device="cuda")
    q, k = (torch.empty(3, h, D, dtype=torch.bfloat16, device="cuda") for h in (hq, hkv))
    out = torch.empty_like(q)
    ws = torch.empty(max(16, nvk().decode_attention_workspace_bytes(3, hq, hkv, D, width, bs)), dtype=torch.uint8, device="cuda")

    def step():
        v = enqueue(new_t, rows_t, meta, qkv, q, k)
        nvk().store_kvcache_blocks8(k, v, *c.data, *c.scale, None, meta[1], meta[0])
        nvk().launch_decode_attention_paged_blocks8(q, *c.data, *c.scale, meta[1], meta[0], hkv, D, bs, scale, out, ws)

    def follow():
        want = book.step([1, 1, 1], rows, width, 3, pool)
        assert [m.tolist() for m in meta] == list(want) and count.item() == book.count
        for w, x in ((0, k), (1, qkv[:, (hq + hkv) * D:].reshape(3, hkv, D))):
            c.ref[w].store(x.double().cpu().numpy(), [0, 1, 2, 3], want[1], want[0])
        q64 = q.double().cpu().numpy()
        for s, n in enumerate(want[1]):
            o = out[s].double().cpu().numpy()
            if n == 0:
                assert (o == 0).all()
                continue
            w, most = _bound(c, want[0][s], n, q64[s], scale, dtype)
            assert (np.abs(o - w) <= most).all()

    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    follow()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for i in range(20):
        qkv.copy_(torch.from_numpy(rng.standard_normal(qkv.shape) * 2.0 ** (i / 6)))
        graph.replay()
        torch.cuda.synchronize()
        follow()

    nvk().release_blocks(torch.tensor([2], dtype=torch.int32, device="cuda"), None, lens, held, free, count, bs)
    book.release([2], None)
    assert free.tolist()[:book.count] == book.free[:book.count] and lens.tolist() == book.lens and count.item() == book.count


# ---- values that are not finite, and scales far apart ---------------------------------------------------------------------------
# Every way of sharing a context out: (Hq, Hkv, sequences, table entries of 64 keys, lengths among them).
WAYS = {"clusters of eight": (8, 1, 6, 64, [4096, 700, 33]), "clusters, few keys": (8, 2, 4, 5, [300, 1, 20]), "eight warps": (8, 8, 15, 16, [1024, 900, 1]),
        "eight warps, longest first": (16, 8, 30, 32, [2048, 100, 17]), "halves": (16, 8, 20, 32, [2048, 1025, 31]), "chunks of 768": (2, 1, 200, 64, [4096, 769, 5]),
        "chunks of 1024": (8, 8, 90, 128, [3000, 1025, 64])}


@pytest.mark.gpu
@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("which", ["K", "V"])
def test_a_block_of_nan_reads_as_nan_wherever_it_lies(way, kind, dtype, which):
    """A scale of NaN, of K alone or of V alone, in a context's first, some or last block: NaN for the sequence and KV head whose it is, and not a bit of the others changes."""
    rng = np.random.default_rng(len(way))
    hq, hkv, batch, width, long = WAYS[way]
    bs, per = 64, hq // hkv
    lens = (long + [int(x) for x in rng.integers(1, 100, batch)])[:batch]
    c, tables = _filled(rng, kind, dtype, bs, hkv, lens, width)
    q, _ = _typed(rng.standard_normal((batch, hq, D)), dtype)
    before = _decode(c, q, lens, tables)
    assert np.isfinite(before).all()
    scale = c.scale["KV".index(which)]
    for s in range(len(long)):
        used = -(-lens[s] // bs)
        for blk in sorted({0, int(rng.integers(0, used)), used - 1}):
            head = int(rng.integers(0, hkv))
            block = int(tables[s][blk])
            was = scale[block, head].clone()
            scale[block, head] = float("nan")
            for workspace in (True, False):
                got = _decode(c, q, lens, tables, workspace=workspace)
                theirs = np.zeros((batch, hq), bool)
                theirs[s, head * per:(head + 1) * per] = True
                assert np.isnan(got[theirs]).all(), (s, blk, head)
                assert not np.isnan(got[~theirs]).any()
                if workspace:
                    assert np.array_equal(got[~theirs], before[~theirs])
            scale[block, head] = was
    assert np.array_equal(_decode(c, q, lens, tables), before)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("leader", ["zeros", "outside", "tiny"])
@pytest.mark.parametrize("lead", [100.0, 131.0, 200.0])
@pytest.mark.parametrize("at", [0, 1, 6, 39])
def test_decode_where_all_attention_goes_to_values_of_nothing(kind, dtype, leader, lead, at):
    """A block whose keys lead all others by 2^lead, with values of zero (a scale of 2^-126), of next to nothing, or outside the cache (a scale of 0): the others' values, of
    scales that are larger by any factor, come with weights of zero and have to leave nothing behind."""
    rng = np.random.default_rng(int(lead) + at)
    bs, hq, hkv, n = 16, 4, 2, 640
    tables = rng.permutation(42)[:40][None]
    c = Both(42, bs, hkv, kind)
    k, v = rng.standard_normal((2, n, hkv, D))
    mine = slice(at * bs, (at + 1) * bs)
    k[..., 0] = -16.0
    k[mine] = 0.0
    v *= 4000.0
    v[mine] = 0.0 if leader != "tiny" else 2.0 ** -24 if dtype == "float16" else 2.0 ** -100
    x = [_typed(k, dtype), _typed(v, dtype)]
    c.store(x, [0, n], [n], tables.tolist())
    if leader == "outside":
        tables[0, at] = -1
    q = np.zeros((1, hq, D))
    q[..., 0] = 1.0
    qd, here = _typed(q, dtype)
    scale = lead * np.log(2.0) / 16.0
    want, most = _bound(c, tables[0], n, here[0], scale, dtype)
    # A weight below 2^-126 of the largest is no number that the exponential gives: it is zero, which takes at most 2^-126 of the sum of magnitudes.  (2^-131 of 4000, as for the lead in between,
    # is a number of BF16.)
    most = most + 2.0 ** -126 * np.repeat(np.abs(c.ref[1].rows(tables[0], n)).sum(0), hq // hkv, axis=0)
    for workspace in (True, False):
        got = _decode(c, qd, [n], tables, scale=scale, workspace=workspace)[0]
        assert np.isfinite(got).all()
        assert (np.abs(got - want) <= most).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype", [("int8", "bfloat16"), ("e4m3", "float16")])
@pytest.mark.parametrize("hq,hkv,batch,width", [(4, 1, 296, 16), (2, 1, 320, 20), (16, 8, 38, 18)])
def test_whole_contexts_with_and_without_a_workspace(kind, dtype, hq, hkv, batch, width):
    """Two pairs to an SM and more, tables of 1024 to 1280 keys: whole contexts, in the same order of sums whether a workspace is there or not (contexts of more than 64 keys: shorter ones are
    dealt to the warps otherwise in clusters)."""
    rng = np.random.default_rng(batch)
    bs = 64
    lens = [int(x) for x in rng.integers(65, 300, batch)]
    lens[:2] = [width * bs, width * bs - 5]
    c, tables = _filled(rng, kind, dtype, bs, hkv, lens, width)
    q, here = _typed(rng.standard_normal((batch, hq, D)) * 2.0, dtype)
    full = _check_decode(c, q, here, lens, tables, dtype)
    assert np.array_equal(full, _decode(c, q, lens, tables, workspace=False))


# ---- tensors of a call that overlap, on the CPU -----------------------------------------------------------------------------------
AT = {name: ctypes.c_void_p((i + 1) << 40) for i, name in enumerate(("key", "value", "k_cache", "v_cache", "k_scale", "v_scale", "cu", "ctx", "bt", "q", "out", "ws"))}   # (nothing is read there)


def _apart(args, **change):
    """The call's arguments with every tensor at a place of its own, then the change."""
    a = dict(args)
    a.update({n: p for n, p in AT.items() if n in a and a[n] is not None})
    a.update(change)
    return a.values()


def _named(build, names):
    return dict(zip(names, build()))


STORE = "key value ks vs k_cache v_cache k_scale v_scale kind cu cu_dtype ctx ctx_dtype bt bt_dtype seqs total max_blocks blocks hkv d bs dtype stream".split()
GATHER = "k_cache v_cache k_scale v_scale kind cu cu_dtype bt bt_dtype seqs total max_blocks blocks hkv d bs key value dtype stream".split()
DECODE = "q k_cache v_cache k_scale v_scale kind ctx ctx_dtype bt bt_dtype batch max_blocks blocks hq hkv d bs scale out dtype ws ws_bytes stream".split()


def _by(name, more=0):
    return ctypes.c_void_p(AT[name].value + more)


@pytest.mark.parametrize("change", [
    dict(v_cache=_by("k_cache")), dict(v_cache=_by("k_cache", 4 * 16 * 256 - 16)), dict(v_scale=_by("k_scale", 28)), dict(k_scale=_by("k_cache", 64)), dict(key=_by("v_cache", 32)),
    dict(value=_by("k_cache", 4 * 16 * 256 - 16)), dict(cu=_by("k_scale", 4)), dict(ctx=_by("v_scale")), dict(bt=_by("k_cache", 8)), dict(k_cache=_by("key", 4 * 512 + 496)),
    dict(ks=L(1024), k_cache=_by("key", 4 * 2048))])
def test_store_refuses_caches_over_other_tensors(built, change):
    rc, said = _call(built, "nvk_store_kvcache_blocks8", *_apart(_named(_store_args, STORE), **change))
    assert rc == 1 and "overlap" in said, said


@pytest.mark.parametrize("change", [
    dict(value=_by("key")), dict(value=_by("key", 10 * 512 - 16)), dict(key=_by("k_cache", 16)), dict(value=_by("v_scale")), dict(cu=_by("key", 4)), dict(bt=_by("value", 10 * 512 - 8))])
def test_gather_refuses_rows_over_other_tensors(built, change):
    rc, said = _call(built, "nvk_gather_kvcache_blocks8", *_apart(_named(_gather_args, GATHER), **change))
    assert rc == 1 and "overlap" in said, said


@pytest.mark.parametrize("change", [
    dict(out=_by("k_cache", 256)), dict(out=_by("q", 8)), dict(out=_by("v_scale", 8)), dict(ctx=_by("out", 4)), dict(bt=_by("out")), dict(ws=AT["ws"], ws_bytes=ctypes.c_size_t(1 << 41)),
    dict(ws=AT["ws"], ws_bytes=ctypes.c_size_t(1 << 30), q=_by("ws", 1024)), dict(ws=AT["ws"], ws_bytes=ctypes.c_size_t(1 << 30), out=_by("ws", 1024), bt=_by("ws", 1 << 31))])
def test_decode_refuses_outputs_over_other_tensors(built, change):
    change = dict(change)
    if change.get("ws_bytes") is not None and change["ws_bytes"].value == 1 << 41:   # (a workspace that reaches to the tables)
        change["bt"] = _by("ws", (1 << 40) + 64)
    rc, said = _call(built, "nvk_decode_attention_paged_blocks8", *_apart(_named(_decode_args, DECODE), **change))
    assert rc == 1 and "overlap" in said, said


@pytest.mark.parametrize("call,change", [
    ("nvk_store_kvcache_blocks8", dict(blocks=L(1 << 50))), ("nvk_store_kvcache_blocks8", dict(ks=L(1 << 60))), ("nvk_store_kvcache_blocks8", dict(seqs=L(1 << 29), max_blocks=L(1 << 30), bs=I(1))),
    ("nvk_gather_kvcache_blocks8", dict(blocks=L(1 << 50))), ("nvk_gather_kvcache_blocks8", dict(seqs=L(1 << 40), max_blocks=L(1 << 26)))])
def test_sizes_beyond_memory_are_refused(built, call, change):
    names, build = (STORE, _store_args) if "store" in call else (GATHER, _gather_args)
    rc, said = _call(built, call, *_apart(_named(build, names), **change))
    assert rc == 3 and "too many" in said, said


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype", [("int8", "bfloat16"), ("e4m3", "float16")])
@pytest.mark.parametrize("way", WAYS)
def test_decode_into_the_query(way, kind, dtype):
    """The output may be the query itself, however contexts are shared out."""
    import torch
    rng = np.random.default_rng(len(way))
    hq, hkv, batch, width, long = WAYS[way]
    lens = (long + [int(x) for x in rng.integers(0, 100, batch)])[:batch]
    c, tables = _filled(rng, kind, dtype, 64, hkv, lens, width)
    q, _ = _typed(rng.standard_normal((batch, hq, D)), dtype)
    want = _decode(c, q, lens, tables)
    up = lambda v: torch.as_tensor(np.asarray(v), dtype=torch.int32).cuda()
    ws = torch.empty(max(16, nvk().decode_attention_workspace_bytes(batch, hq, hkv, D, width, 64)), dtype=torch.uint8, device="cuda")
    n, bt = up(lens), up(tables)
    for _ in range(20):
        x = q.clone()
        nvk().launch_decode_attention_paged_blocks8(x, *c.data, *c.scale, n, bt, hkv, D, 64, 0.09, x, ws)
        assert np.array_equal(x.double().cpu().numpy(), want)
