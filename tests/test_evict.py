"""Decode attention that adds up the weights of the keys (nvk_decode_attention_paged_weights) and the eviction that goes by them (nvk_evict_kvcache),
over 16-bit and 4-bit caches, against 64-bit restatements of their definitions (ref_int4.py)."""
import ctypes

import numpy as np
import pytest

import ref_int4 as ref
from test_int4_kv import D, I, L, ODD, P, _cache, _call, _dev, _typed, built  # noqa: F401  (`built` is a fixture)
from util import nvk, to_dev


# ---- on the CPU --------------------------------------------------------------------------------------------------------------
def test_who_stays_by_hand():
    w = np.array([0.1, 5.0, 2.0, np.nan, 2.0, -1.0, 2.0, np.inf, 0.0, 9.0])
    assert ref.keep(w, 10, 10, 1, 1).tolist() == list(range(10))
    assert ref.keep(w, 10, 5, 1, 1).tolist() == [0, 1, 2, 7, 9]               # of the three 2.0 the first
    assert ref.keep(w, 10, 9, 1, 1).tolist() == [0, 1, 2, 4, 5, 6, 7, 8, 9]   # NaN goes first
    assert ref.keep(w, 10, 3, 2, 1).tolist() == [0, 1, 9]
    assert ref.keep(w, 10, 1, 0, 0).tolist() == [7]


def _weights_args(**change):
    a = dict(q=P, k_cache=P, v_cache=P, k_params=None, v_params=None, ctx=P, ctx_dtype=I(3), bt=P, bt_dtype=I(3), batch=L(2), max_blocks=L(4), blocks=L(4), hq=I(8),
             hkv=I(2), d=I(128), bs=I(256), scale=ctypes.c_float(1.0), old=None, rows=None, rows_dtype=I(3), num_rows=L(2), row_keys=L(1024), new=P, out=P,
             dtype=I(1), ws=P, ws_bytes=ctypes.c_size_t(1 << 30), stream=None)
    a.update(change)
    return a.values()


@pytest.mark.parametrize("change,code,word", [
    (dict(new=None), 1, "requires"), (dict(out=None), 1, "requires"), (dict(k_params=P), 1, "together"), (dict(rows=P, rows_dtype=I(1)), 1, "int32 or int64"),
    (dict(hq=I(7)), 1, "divisible"), (dict(row_keys=L(1023)), 1, "max_blocks"), (dict(num_rows=L(0)), 1, "hold"), (dict(num_rows=L(1)), 1, "every sequence"),
    (dict(num_rows=L(1), rows=P, ws=None), 1, "workspace"), (dict(ws_bytes=ctypes.c_size_t(100)), 1, "workspace"), (dict(ws=ODD), 1, "workspace"),
    (dict(d=I(64)), 3, "head_dim"), (dict(dtype=I(2)), 3, "F16"), (dict(hq=I(18)), 3, "8 query heads"), (dict(bs=I(24)), 3, "multiple"),
    (dict(new=ctypes.c_void_p(258)), 1, "aligned"), (dict(k_params=P, v_params=P, q=ODD), 3, "aligned"), (dict(batch=L(0)), 0, "")])
def test_weights_refuse(built, change, code, word):   # noqa: F811
    rc, said = _call(built, "nvk_decode_attention_paged_weights", *_weights_args(**change))
    assert rc == code and (rc == 0 or word in said), said


def _evict_args(**change):
    a = dict(k_cache=P, v_cache=P, k_params=None, v_params=None, old=P, rows=None, rows_dtype=I(3), num_rows=L(2), row_keys=L(64), ctx=P, ctx_dtype=I(3), bt=P,
             bt_dtype=I(3), batch=L(2), max_blocks=L(4), blocks=L(9), new=P, new_bt=P, new_bt_dtype=I(4), new_max_blocks=L(2), new_ctx=ctypes.c_void_p(512), hkv=I(2),
             d=I(128), bs=I(16), budget=L(32), sinks=L(4), recent=L(8), dtype=I(1), stream=None)
    a.update(change)
    return a.values()


@pytest.mark.parametrize("change,code,word", [
    (dict(old=None), 1, "defined"), (dict(new_ctx=None), 1, "defined"), (dict(v_params=P), 1, "together"), (dict(new_bt_dtype=I(2)), 1, "int32 or int64"),
    (dict(dtype=I(2)), 3, "F16 or BF16"), (dict(d=I(64)), 3, "128"), (dict(budget=L(0)), 1, "budget"), (dict(sinks=L(-1)), 1, "budget"), (dict(recent=L(-1)), 1, "budget"),
    (dict(sinks=L(25)), 1, "budget"), (dict(sinks=L(1 << 62), recent=L(1 << 62)), 1, "budget"), (dict(row_keys=L(63)), 1, "max_blocks"),
    (dict(num_rows=L(1)), 1, "every sequence"), (dict(new_max_blocks=L(1)), 1, "hold the budget"), (dict(k_cache=ODD), 1, "aligned"),
    (dict(new=ctypes.c_void_p(258)), 1, "aligned"), (dict(new_ctx=P), 1, "must not be"), (dict(new_ctx=ctypes.c_void_p(260)), 1, "must not be"),
    (dict(batch=L(0)), 0, "")])
def test_evict_refuses(built, change, code, word):   # noqa: F811
    rc, said = _call(built, "nvk_evict_kvcache", *_evict_args(**change))
    assert rc == code and (rc == 0 or word in said), said


@pytest.mark.parametrize("shift", [4, 64, -64])
def test_weights_that_overlap_in_part_are_refused(built, shift):   # noqa: F811
    """The same memory is in place, other memory is other memory; anything between would be read by one block after another has written it."""
    base = 1 << 20
    for name, args, new in (("nvk_decode_attention_paged_weights", _weights_args, "new"), ("nvk_evict_kvcache", _evict_args, "new")):
        rc, said = _call(built, name, *args(old=ctypes.c_void_p(base), **{new: ctypes.c_void_p(base + shift)}))
        assert rc == 1 and "overlap" in said, (name, said)


def test_a_workspace_covers_fewer_sequences_and_narrower_tables(built):   # noqa: F811
    rng = np.random.default_rng(1)
    size = built.decode_attention_weights_workspace_bytes
    for _ in range(3000):
        hkv = int(rng.choice([1, 2, 8]))
        hq, bs = hkv * int(rng.integers(1, 9)), int(rng.choice([16, 48, 256]))
        b, w = int(2 ** rng.uniform(0, 9)), int(2 ** rng.uniform(0, 10))
        b2, w2 = int(rng.integers(1, b + 1)), int(rng.integers(1, w + 1))
        assert size(b2, hq, hkv, D, w2, bs) <= size(b, hq, hkv, D, w, bs)
    assert size(0, 8, 8, D, 4, 16) == 0


# ---- on the GPU --------------------------------------------------------------------------------------------------------------
def _tables(rng, lens, bs, blocks, width=0, taken=()):
    need = [-(-n // bs) for n in lens]
    free = [i for i in rng.permutation(blocks) if i not in taken]
    out = np.zeros((len(lens), max(1, width, max(need))), np.int64)
    for i, n in enumerate(need):
        for j in range(n):
            out[i, j] = free.pop()
    return out


def _any_cache(rng, rows, hkv, dtype, kv):
    """(k, v, k_params, v_params on the device, values of K and V, what the rounding of p' touches)"""
    if kv == "int4":
        (kc, kp, k, _), (vc, vp, v, spread) = _cache(rng, rows, hkv, dtype)
        return [kc, vc, kp, vp], k, v, spread
    k, v = _typed(rng, (rows, hkv, D), dtype), _typed(rng, (rows, hkv, D), dtype, 0.7)
    return [_dev(k, dtype), _dev(v, dtype), None, None], k, v, np.abs(v)


@pytest.mark.gpu
@pytest.mark.parametrize("kv,dtype,hq,hkv,bs,lens,index,rows", [
    ("same", "bfloat16", 32, 8, 256, [300], "int32", None),
    ("int4", "bfloat16", 32, 8, 256, [300], "int64", None),
    ("same", "float16", 4, 1, 16, [0, 1, 16, 17, 40], "int64", [4, 7, 0, 2, 6]),
    ("int4", "float16", 6, 2, 48, [1, 47, 48, 49, 700], "int32", [0, -1, 5, 9, 1]),
    ("same", "bfloat16", 14, 2, 256, [5000, 260, 1], "int32", None),
    ("int4", "bfloat16", 8, 1, 256, [9000, 3000], "int32", [1, 0]),
    ("same", "bfloat16", 8, 8, 256, [100 + 61 * i for i in range(30)], "int32", None),
    ("int4", "bfloat16", 16, 8, 256, [100 + 61 * i for i in range(40)], "int32", None),
])
def test_weights_are_added_up(kv, dtype, hq, hkv, bs, lens, index, rows):
    import torch
    rng = np.random.default_rng(hq + 7 * len(lens))
    blocks = sum(-(-n // bs) for n in lens) + 3
    cache, k_all, v_all, spread = _any_cache(rng, blocks * bs, hkv, dtype, kv)
    tables = _tables(rng, lens, bs, blocks, max(-(-n // bs) for n in lens) + 1)
    b, width, lib, dt = len(lens), tables.shape[1], nvk(), getattr(torch, index)
    num_rows, keys = 8 if rows is not None else b, width * bs + 5
    old = np.float32(np.exp(2 * rng.standard_normal((num_rows, hkv, keys))) * hq / hkv / max(lens)).astype(np.float64)
    q, scale = _typed(rng, (b, hq, D), dtype), 1.0 / np.sqrt(D)
    dev = to_dev(old.astype(np.float32))
    new, out = torch.full_like(dev, 7.0), torch.full((b, hq, D), float("nan"), dtype=getattr(torch, dtype), device="cuda")
    ws = torch.empty(lib.decode_attention_weights_workspace_bytes(b, hq, hkv, D, width, bs), dtype=torch.uint8, device="cuda").fill_(255)
    ctx, bt, qd = to_dev(np.array(lens), dt), to_dev(tables, dt), _dev(q, dtype)
    rd = to_dev(np.array(rows), dt) if rows is not None else None

    def call(old_weights, new_weights, to):
        lib.launch_decode_attention_paged_weights(qd, *cache, ctx, bt, hkv, D, bs, scale, old_weights, rd, new_weights, to, ws)

    call(dev, new, out)
    torch.cuda.synchronize()
    got, got_out, u = new.double().cpu().numpy(), out.double().cpu().numpy(), ref.HALF_STEP[dtype]
    want = np.full_like(old, 7.0)
    tol = np.zeros_like(old)
    for i, n in enumerate(lens):
        at = ref.places(tables[i], n, bs, blocks)
        k, v = ref.context(k_all, at), ref.context(v_all, at)
        res, p = ref.attend(q[i], k, v, scale)
        around = np.einsum("jgn,njd->jgd", p.reshape(hkv, hq // hkv, n), ref.context(spread, at)).reshape(hq, D)
        e = ref.score_error(q[i], np.abs(k_all).max() + (31 * 0.5 if kv == "int4" else 0.0), scale) + 2.0 ** -20
        assert (np.abs(got_out[i] - res) <= u * around + u * np.abs(res) + 2 * e * (np.abs(v_all).max() + 1)).all(), i
        r = i if rows is None else rows[i]
        if 0 <= r < num_rows:
            add = p.reshape(hkv, hq // hkv, n).sum(1)
            want[r, :, :n] = old[r, :, :n] + add
            # a score off by e moves p by 2e; then the group's sum and the sum with what was there, in fp32
            tol[r, :, :n] = 2 * e * add + 2.0 ** -24 * (2 * hq // hkv * add + want[r, :, :n])
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / np.maximum(want, 1e-30)).max())
    # the output is that of the call without weights, bit for bit; so are the weights in place, and of a second run
    plain = torch.full_like(out, 3.0)
    ws2 = torch.empty(max(16, lib.decode_attention_workspace_bytes(b, hq, hkv, D, width, bs)), dtype=torch.uint8, device="cuda")
    if kv == "int4":
        lib.launch_decode_attention_paged_int4(qd, *cache, ctx, bt, hkv, D, bs, scale, plain, ws2)
    else:
        lib.launch_decode_attention_paged(qd, *cache[:2], ctx, bt, hkv, D, bs, scale, plain, ws2)
    place, again = dev.clone(), torch.full_like(out, 1.0)
    call(place, place, again)
    zero = torch.full_like(dev, 7.0)
    call(None, zero, again)
    torch.cuda.synchronize()
    assert torch.equal(plain, out) and torch.equal(again, out)
    touched = torch.from_numpy(tol > 0).cuda()
    assert torch.equal(place, torch.where(touched, new, dev))
    assert torch.equal(torch.where(touched, dev + zero, new), new) and bool((zero[~touched] == 7.0).all())


def _evict_reference(cache, tables, new_tables, lens, weights, rows, bs, blocks, budget, sinks, recent):
    """numpy arrays in, [moved caches], new weights, new lengths out; in place where the tables are the same."""
    moved, new_w, new_lens = [c.copy() for c in cache], weights.copy(), []
    hkv = weights.shape[1]
    for i, n in enumerate(lens):
        r = rows[i]
        if not 0 <= r < len(weights):
            new_lens.append(n)
            continue
        new_lens.append(min(n, budget))
        at, to = ref.places(tables[i], n, bs, blocks), ref.places(new_tables[i], min(n, budget), bs, blocks)
        for j in range(hkv):
            stay = ref.keep(weights[r, j], n, budget, sinks, recent)
            new_w[r, j] = 0
            new_w[r, j, :len(stay)] = weights[r, j, stay]
            src, good = at[stay], to >= 0
            for was, now in zip(cache, moved):
                rows_in = np.where((src >= 0).reshape(-1, *[1] * (was.ndim - 2)), was[np.maximum(src, 0), j], 0)
                now[to[good], j] = rows_in[good]
    return moved, new_w, np.array(new_lens)


def _np(t):
    import torch
    return t.cpu().numpy() if t.dtype == torch.uint8 else t.cpu().view(torch.int16).numpy()


@pytest.mark.gpu
@pytest.mark.parametrize("kv,dtype,hkv,bs,lens,index,budget,sinks,recent,place", [
    ("same", "bfloat16", 2, 16, [100, 37, 0, 1, 64, 65], "int32", 37, 4, 8, "other"),
    ("same", "float16", 3, 48, [1500, 100, 2049, 1025], "int64", 700, 0, 0, "same"),
    ("int4", "bfloat16", 8, 256, [3000, 513, 512, 511], "int32", 512, 4, 128, "same"),
    ("int4", "float16", 1, 16, [500, 20, 333], "int64", 33, 16, 17, "other"),      # nothing goes by its weight
    ("same", "bfloat16", 1, 256, [5000], "int32", 1, 0, 0, "same"),
    ("same", "bfloat16", 4, 64, [2600, 900], "int32", 899, 1, 0, "same"),          # one key goes
    ("int4", "bfloat16", 2, 256, [70000], "int32", 65001, 0, 5000, "other"),
    ("same", "bfloat16", 8, 256, [1000 + 97 * i for i in range(20)], "int32", 1024, 4, 256, "other"),
])
def test_evict(kv, dtype, hkv, bs, lens, index, budget, sinks, recent, place):
    import torch
    rng = np.random.default_rng(budget)
    b, dt = len(lens), getattr(torch, index)
    kept = [min(n, budget) for n in lens]
    blocks = sum(-(-n // bs) for n in lens) + (sum(-(-n // bs) for n in kept) if place == "other" else 0) + 2
    # whatever bytes: eviction moves them as they are
    shape = (blocks * bs, hkv)
    if kv == "int4":
        cache = [torch.randint(0, 256, (*shape, 64), dtype=torch.uint8, device="cuda") for _ in range(2)]
        cache += [torch.randint(-2 ** 15, 2 ** 15, (*shape, 2), dtype=torch.int16, device="cuda").view(getattr(torch, dtype)) for _ in range(2)]
    else:
        cache = [torch.randint(-2 ** 15, 2 ** 15, (*shape, D), dtype=torch.int16, device="cuda").view(getattr(torch, dtype)) for _ in range(2)]
    tables = _tables(rng, lens, bs, blocks)
    new_tables = _tables(rng, kept, bs, blocks, taken=set(tables.ravel()) if b > 1 or lens[0] else ()) if place == "other" else tables
    if b == 6:
        tables[0, 2], new_tables[4, 0] = -1, blocks + 9                  # outside the cache: zeros, and not written
    rows = rng.permutation(b + 2)[:b]
    if b == 4:
        rows[1] = -1
    keys = tables.shape[1] * bs + 3
    w = np.float32(np.exp(2 * rng.standard_normal((b + 2, hkv, keys))))
    # many equal ones, and such as are hard to order
    w[:, :, 5::7] = np.float32(0.25)
    w[0, :, 9::11], w[1, :, 3::5] = np.float32(np.nan), np.float32(0.0)
    w[1, :, 4::5], w[0, 0, 10::50], w[0, 0, 20::50], w[1, 0, 8::9] = np.float32(-0.0), np.float32(np.inf), np.float32(-np.inf), np.float32(1e-42)
    before = [_np(c) for c in cache]
    want, want_w, want_lens = _evict_reference(before, tables, new_tables, lens, w, rows, bs, blocks, budget, sinks, recent)
    weights = to_dev(w)
    new_w = weights if place == "same" else weights.clone()
    new_lens = torch.full((b,), -5, dtype=dt, device="cuda")
    args = cache if kv == "int4" else [*cache, None, None]
    bt = to_dev(tables, dt)
    nvk().evict_kvcache(*args, weights, to_dev(rows, dt), to_dev(np.array(lens), dt), bt, new_w, bt if place == "same" else to_dev(new_tables, dt), new_lens, hkv, D, bs,
                        budget, sinks, recent)
    torch.cuda.synchronize()
    assert new_lens.tolist() == want_lens.tolist()
    for i, r in enumerate(rows):
        if 0 <= r:
            assert np.array_equal(new_w[r].cpu().numpy(), want_w[r], equal_nan=True), i
    others = [r for r in range(b + 2) if r not in rows]
    assert np.array_equal(new_w.cpu().numpy()[others], w[others], equal_nan=True)
    for got, exp, was in zip(cache, want, before):
        got = _np(got)
        if place == "same":       # what lies behind the kept keys is left as it was
            assert np.array_equal(got, exp)
        else:
            assert np.array_equal(got, exp)
            taken = np.unique(tables[(tables >= 0) & (tables < blocks)])
            old = (taken[:, None] * bs + np.arange(bs)).ravel()
            old = np.setdiff1d(old, (np.unique(new_tables[(new_tables >= 0) & (new_tables < blocks)])[:, None] * bs + np.arange(bs)).ravel())
            assert np.array_equal(got[old], was[old])


def _step(lib, s, cache, kv, q, k, v, old, new, ws, out):
    """One decode step: the token's K and V into the cache, attention, the weights added up."""
    if kv == "int4":
        lib.store_kvcache_int4(k, v, *cache, s["slots"])
    else:
        lib.store_kvcache(k, v, *cache[:2], s["slots"])
    lib.launch_decode_attention_paged_weights(q, *cache, s["ctx"], s["bt"], s["hkv"], D, s["bs"], s["scale"], old, None, new, out, ws)


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["same", "int4"])
def test_steps_eviction_and_steps_again(kv):
    """A prompt into the cache, decode steps that add up the weights, an eviction in place, and a step over what is left, all against 64 bits; then
    the same as one captured graph, replayed twice, bit for bit."""
    import torch
    rng = np.random.default_rng(31)
    hq, hkv, bs, dtype, budget, sinks, recent = 8, 2, 16, "bfloat16", 40, 2, 6
    prompts, steps, scale = [70, 33, 12], 5, 0.088
    b, width = len(prompts), 6
    blocks = b * width
    lib, dt, bf = nvk(), torch.int32, torch.bfloat16
    tables = rng.permutation(blocks).reshape(b, width)
    bt = to_dev(tables, dt)
    if kv == "int4":
        cache = [torch.zeros((blocks * bs, hkv, 64), dtype=torch.uint8, device="cuda") for _ in range(2)] + [torch.zeros((blocks * bs, hkv, 2), dtype=bf, device="cuda") for _ in range(2)]
    else:
        cache = [torch.zeros((blocks * bs, hkv, D), dtype=bf, device="cuda") for _ in range(2)] + [None, None]

    def kept_as(x):
        return ref.values(*ref.quantise(x, dtype)) if kv == "int4" else x

    total = [n + steps for n in prompts]
    keys, vals = [[_typed(rng, (n, hkv, D), dtype) for n in total] for _ in range(2)]
    pslots = np.concatenate([ref.places(tables[i], n, bs, blocks) for i, n in enumerate(prompts)])
    pk, pv = (_dev(np.concatenate([x[i][:n] for i, n in enumerate(prompts)]), dtype) for x in (keys, vals))
    qs = [_typed(rng, (b, hq, D), dtype) for _ in range(steps + 1)]
    last_k, last_v = (_typed(rng, (b, hkv, D), dtype) for _ in range(2))
    plans = []
    for t in range(steps):
        ctx = np.array(prompts) + t + 1
        plans.append(dict(ctx=to_dev(ctx, dt), slots=to_dev(np.array([ref.places(tables[i], n, bs, blocks)[-1] for i, n in enumerate(ctx)]), dt), bt=bt, hkv=hkv, bs=bs,
                          scale=scale))
    ws = torch.empty(lib.decode_attention_weights_workspace_bytes(b, hq, hkv, D, width, bs), dtype=torch.uint8, device="cuda")
    weights, new_lens = torch.zeros((b, hkv, width * bs), device="cuda"), torch.zeros(b, dtype=dt, device="cuda")
    after = [min(n, budget) + 1 for n in total]
    last = dict(ctx=to_dev(np.array(after), dt), bt=bt, hkv=hkv, bs=bs, scale=scale,
                slots=to_dev(np.array([ref.places(tables[i], n, bs, blocks)[-1] for i, n in enumerate(after)]), dt))
    dq = [_dev(q, dtype) for q in qs]
    dk, dv = ([_dev(np.stack([x[i][n + t] for i, n in enumerate(prompts)]), dtype) for t in range(steps)] for x in (keys, vals))
    dlk, dlv, slots = _dev(last_k, dtype), _dev(last_v, dtype), to_dev(pslots, dt)
    outs = torch.empty((steps + 1, b, hq, D), dtype=bf, device="cuda")

    def everything():
        weights.zero_()
        if kv == "int4":
            lib.store_kvcache_int4(pk, pv, *cache, slots)
        else:
            lib.store_kvcache(pk, pv, *cache[:2], slots)
        for t in range(steps):
            _step(lib, plans[t], cache, kv, dq[t], dk[t], dv[t], weights, weights, ws, outs[t])
        lib.evict_kvcache(*cache, weights, None, plans[-1]["ctx"], bt, weights, bt, new_lens, hkv, D, bs, budget, sinks, recent)
        _step(lib, last, cache, kv, dq[steps], dlk, dlv, weights, weights, ws, outs[steps])

    everything()
    torch.cuda.synchronize()
    first, first_w = outs.clone(), weights.clone()
    assert new_lens.tolist() == [n - 1 for n in after]
    u = ref.HALF_STEP[dtype]
    for i, n in enumerate(total):
        k, v = kept_as(keys[i]), kept_as(vals[i])
        w = np.zeros((hkv, n))
        for t in range(steps):
            m = prompts[i] + t + 1
            _, p = ref.attend(qs[t][i], k[:m], v[:m], scale)
            w[:, :m] += p.reshape(hkv, -1, m).sum(1)
        for j in range(hkv):
            stay = ref.keep(w[j], n, budget, sinks, recent)
            gone = np.setdiff1d(np.arange(n), stay)
            if len(gone):   # (no key that stays by its weight is so near to one that goes that fp32 sums could order them otherwise)
                by_weight = stay[(stay >= sinks) & (stay < n - recent)]
                assert w[j, by_weight].min() > w[j, gone].max() * (1 + 1e-4)
            kk = np.concatenate([k[stay, j], kept_as(last_k)[i:i + 1, j]])
            vv = np.concatenate([v[stay, j], kept_as(last_v)[i:i + 1, j]])
            g = hq // hkv
            want, p = ref.attend(qs[steps][i].reshape(hkv, g, D)[j], kk[:, None], vv[:, None], scale)
            got = first[steps, i].double().cpu().numpy().reshape(hkv, g, D)[j]
            e = ref.score_error(qs[steps][i], np.abs(kk).max() + 16, scale) + 2.0 ** -20
            touched = p @ (np.abs(vv) + 4)                      # (a 4-bit value and the middle of its range are 7.5 steps, at most 4, apart)
            assert (np.abs(got - want) <= u * touched + u * np.abs(want) + 2 * e * 6).all()
            new = np.concatenate([w[j, stay], [0.0]]) + p.sum(0)
            assert np.abs(first_w[i, j, :len(new)].double().cpu().numpy() - new).max() <= 1e-3 * new.max()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        everything()
    for _ in range(2):
        outs.zero_()
        new_lens.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs, first) and torch.equal(weights, first_w) and new_lens.tolist() == [n - 1 for n in after]


@pytest.mark.gpu
def test_a_chunked_prefill_over_the_4_bit_cache():
    """A prompt in two chunks: store, gather of the whole context, dense prefill over it; against 64 bits."""
    import torch
    rng = np.random.default_rng(8)
    hq, hkv, bs, dtype, scale = 8, 2, 256, "bfloat16", 0.088
    lens, first = [300, 41], [256, 0]
    lib, dt = nvk(), torch.int32
    blocks = 4
    tables = np.array([[2, 0], [3, 0]])
    cache = [torch.zeros((blocks * bs, hkv, 64), dtype=torch.uint8, device="cuda") for _ in range(2)]
    cache += [torch.zeros((blocks * bs, hkv, 2), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    keys, vals, qs = ([_typed(rng, (n, h, D), dtype) for n in lens] for h in (hkv, hkv, hq))
    for begin, end in ((lambda i: 0, lambda i: first[i]), (lambda i: first[i], lambda i: lens[i])):
        seqs = [i for i in range(2) if end(i) > begin(i)]
        slots = np.concatenate([ref.places(tables[i], end(i), bs, blocks)[begin(i):] for i in seqs])
        k, v, q = (_dev(np.concatenate([x[i][begin(i):end(i)] for i in seqs]), dtype) for x in (keys, vals, qs))
        lib.store_kvcache_int4(k, v, *cache, to_dev(slots, dt))
        cu_q = np.concatenate([[0], np.cumsum([end(i) - begin(i) for i in seqs])])
        cu_k = np.concatenate([[0], np.cumsum([end(i) for i in seqs])])
        dense_k, dense_v = (torch.empty((cu_k[-1] + 100, hkv, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        lib.gather_kvcache_int4(*cache, to_dev(cu_k, dt), to_dev(tables[seqs], dt), hkv, D, bs, dense_k, dense_v)
        out = torch.empty_like(q)
        lib.launch_prefill_attention_dense(q, to_dev(cu_q, dt), dense_k, dense_v, to_dev(cu_k, dt), hkv, D, scale, out)
        torch.cuda.synchronize()
        assert lib.prefill_status() == 0
        for j, i in enumerate(seqs):
            kk, vv = (ref.to_type(ref.values(*ref.quantise(x[i][:end(i)], dtype)), dtype) for x in (keys, vals))
            got = out[cu_q[j]:cu_q[j + 1]].double().cpu().numpy()
            for r in range(begin(i), end(i), 13):
                want, p = ref.attend(qs[i][r], kk[:r + 1], vv[:r + 1], scale)
                e = ref.score_error(qs[i][r], np.abs(kk).max(), scale) + 2.0 ** -18
                bound = 2.0 ** -8 * (np.einsum("jgn,njd->jgd", p.reshape(hkv, -1, r + 1), np.abs(vv[:r + 1])).reshape(hq, D) + np.abs(want)) + 2 * e * np.abs(vv).max()
                assert (np.abs(got[r - begin(i)] - want) <= bound).all()


@pytest.mark.gpu
def test_wrong_tensors_are_refused_here_too():
    import torch
    lib, bf = nvk(), torch.bfloat16
    kc, q = torch.zeros((64, 2, D), dtype=bf, device="cuda"), torch.zeros((1, 8, D), dtype=bf, device="cuda")
    ctx, bt = torch.ones(1, dtype=torch.int32, device="cuda"), torch.zeros((1, 2), dtype=torch.int32, device="cuda")
    w, ws = torch.zeros((1, 2, 32), device="cuda"), torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    kp = torch.zeros((64, 2, 2), dtype=bf, device="cuda")
    for bad in (dict(kp=kp), dict(kc=kc.half()), dict(old=w[..., :16].contiguous()), dict(old=w.double()), dict(new=w[:, :1].contiguous()), dict(rows=ctx.float()),
                dict(rows=torch.zeros(2, dtype=torch.int32, device="cuda")), dict(ws=ws[:100]), dict(ws=None), dict(q=q.float()), dict(bs=8), dict(vc=kc[:32])):
        a = dict(q=q, kc=kc, vc=kc, kp=None, vp=None, ctx=ctx, bt=bt, hkv=2, d=D, bs=16, scale=1.0, old=w, rows=None, new=w.clone(), out=torch.empty_like(q), ws=ws)
        a.update(bad)
        with pytest.raises(ValueError):
            lib.launch_decode_attention_paged_weights(*a.values())
    for bad in (dict(new_ctx=ctx), dict(new_ctx=ctx.long().clone()), dict(budget=0), dict(recent=5), dict(bt=bt[0]), dict(new_bt=bt[:0]), dict(new=w[..., :31].contiguous()),
                dict(kp=kp), dict(bs=0), dict(d=64), dict(vc=kc[:32]), dict(old=w.half()), dict(new_bt=torch.zeros((1, 1), dtype=torch.int32, device="cuda"), budget=17)):
        a = dict(kc=kc, vc=kc, kp=None, vp=None, old=w, rows=None, ctx=ctx, bt=bt, new=w.clone(), new_bt=bt, new_ctx=ctx.clone(), hkv=2, d=D, bs=16, budget=6, sinks=2,
                 recent=1)
        a.update(bad)
        with pytest.raises(ValueError):
            lib.evict_kvcache(*a.values())
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,batch,longest,place", [("bfloat16", 160, 2048, True), ("float16", 120, 1700, False)])
def test_weights_of_whole_contexts_by_blocks_of_eight_warps(dtype, batch, longest, place):
    """Enough pairs beyond the clusters of four, tables of 1537 to 2048 keys: every context is one block's of eight warps, which adds the weights itself."""
    import torch
    rng = np.random.default_rng(batch)
    hq, hkv, bs, blocks, width = 4, 1, 16, 130, -(-longest // 16)
    (kc, kp, k_all, _), (vc, vp, v_all, spread) = _cache(rng, blocks * bs, hkv, dtype)
    lens = [1 + (i * 7919) % longest for i in range(batch)]
    lens[0], lens[1], lens[batch // 2] = 0, 1, longest
    tables = np.stack([rng.permutation(blocks)[:width] for _ in range(batch)])
    keys, scale, u = width * bs, 0.088, ref.HALF_STEP[dtype]
    old = np.float32(np.exp(rng.standard_normal((batch, hkv, keys)))) / 100
    q = _typed(rng, (batch, hq, D), dtype)
    lib, dev = nvk(), to_dev(old)
    new = dev if place else torch.full_like(dev, 7.0)
    out = torch.full((batch, hq, D), float("nan"), dtype=getattr(torch, dtype), device="cuda")
    ws = torch.empty(lib.decode_attention_weights_workspace_bytes(batch, hq, hkv, D, width, bs), dtype=torch.uint8, device="cuda").fill_(255)
    lib.launch_decode_attention_paged_weights(_dev(q, dtype), kc, vc, kp, vp, to_dev(np.array(lens), torch.int32), to_dev(tables, torch.int32), hkv, D, bs, scale,
                                              dev, None, new, out, ws)
    torch.cuda.synchronize()
    got, got_out = new.double().cpu().numpy(), out.double().cpu().numpy()
    for i in sorted({0, 1, batch // 2, *range(0, batch, 13)}):
        n = lens[i]
        at = ref.places(tables[i], n, bs, blocks)
        k, v = ref.context(k_all, at), ref.context(v_all, at)
        want, p = ref.attend(q[i], k, v, scale)
        e = ref.score_error(q[i], np.abs(k_all).max() + 15.5, scale) + 2.0 ** -20
        around = p @ ref.context(spread, at)[:, 0]
        assert (np.abs(got_out[i] - want) <= u * around + u * np.abs(want) + 2 * e * (np.abs(v_all).max() + 1)).all(), i
        # a probability is off by 2 e of itself, and by 2^-18 (the sum: 32 additions in a lane and at most 16 that merge lanes and warps, 48 2^-24; exp2 and
        # 1 / the sum: 2^-21 together); what is added up by an addition for each head
        add = p.sum(0)
        assert (np.abs(got[i, 0, :n] - (old[i, 0, :n] + add)) <= (2 * e + 2.0 ** -18) * add + 4 * 2.0 ** -24 * (old[i, 0, :n] + add) + 1e-30).all(), i
        assert np.array_equal(got[i, 0, n:], old[i, 0, n:] if place else np.full(keys - n, 7.0))


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["same", "int4"])
def test_cache_rows_beyond_32_bits_of_offset(kv):
    """Caches of more than 4 GiB: what a context reads, stores and keeps in its last blocks is what it would in its first ones."""
    import torch
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("24 GB of device memory")
    rng = np.random.default_rng(5)
    hkv, hq, bs, dtype, n = 8, 32, 256, "bfloat16", 700
    row_bytes = hkv * (64 if kv == "int4" else 2 * D)
    blocks = (1 << 32) // (row_bytes * bs) + 8
    lib, dt, bf = nvk(), torch.int32, torch.bfloat16
    k, v = (_dev(_typed(rng, (n, hkv, D), dtype), dtype) for _ in range(2))
    q = _dev(_typed(rng, (1, hq, D), dtype), dtype)
    results = []
    for count in (8, blocks):
        width = 64 if kv == "int4" else D
        cache = [torch.empty((count * bs, hkv, width), dtype=torch.uint8 if kv == "int4" else bf, device="cuda") for _ in range(2)]
        cache += [torch.empty((count * bs, hkv, 2), dtype=bf, device="cuda") for _ in range(2)] if kv == "int4" else [None, None]
        table, fresh = [count - 1, count - 4, count - 2], [count - 6, count - 3, count - 5]
        slots, bt, nt = to_dev(ref.places(table, n, bs, count), torch.int64), to_dev(np.array([table]), dt), to_dev(np.array([fresh]), dt)
        if kv == "int4":
            lib.store_kvcache_int4(k, v, *cache, slots)
        else:
            lib.store_kvcache(k, v, *cache[:2], slots)
        ctx, lens = torch.full((1,), n, dtype=dt, device="cuda"), torch.zeros(1, dtype=dt, device="cuda")
        w, nw = torch.zeros((1, hkv, 3 * bs), device="cuda"), torch.zeros((1, hkv, 3 * bs), device="cuda")
        ws = torch.empty(lib.decode_attention_weights_workspace_bytes(1, hq, hkv, D, 3, bs), dtype=torch.uint8, device="cuda")
        first, second = torch.empty_like(q), torch.empty_like(q)
        lib.launch_decode_attention_paged_weights(q, *cache, ctx, bt, hkv, D, bs, 0.088, None, None, w, first, ws)
        lib.evict_kvcache(*cache, w, None, ctx, bt, nw, nt, lens, hkv, D, bs, 300, 4, 32)
        lib.launch_decode_attention_paged_weights(q, *cache, lens, nt, hkv, D, bs, 0.088, None, None, w, second, ws)
        got = [first, second, w, nw, lens]
        if kv == "int4":
            dense = [torch.empty((300, hkv, D), dtype=bf, device="cuda") for _ in range(2)]
            lib.gather_kvcache_int4(*cache, to_dev(np.array([0, 300]), dt), nt, hkv, D, bs, *dense)
            got += dense
        torch.cuda.synchronize()
        results.append([x.clone() for x in got])
        del cache
    assert all(torch.equal(a, b) for a, b in zip(*results)) and not torch.isnan(results[0][1]).any()


@pytest.mark.gpu
def test_calls_on_two_streams_at_once_do_not_touch_each_other():
    """Two streams, each with its own cache, weights and workspace: forty rounds of steps and evictions in place give what they give one after the other."""
    import torch
    rng = np.random.default_rng(9)
    hq, hkv, bs, dtype, width, b = 8, 2, 16, "bfloat16", 40, 12
    lib, dt, bf = nvk(), torch.int32, torch.bfloat16

    def state(seed):
        r = np.random.default_rng(seed)
        blocks = b * width
        (kc, kp, _, _), (vc, vp, _, _) = _cache(r, blocks * bs, hkv, dtype)
        tables = to_dev(r.permutation(blocks).reshape(b, width), dt)
        q = _dev(_typed(r, (b, hq, D), dtype), dtype)
        return dict(cache=[kc, vc, kp, vp], bt=tables, q=q, ctx=to_dev(np.array([600 - 40 * i for i in range(b)]), dt), out=torch.empty((40, b, hq, D), dtype=bf, device="cuda"),
                    w=torch.zeros((b, hkv, width * bs), device="cuda"), lens=torch.zeros(b, dtype=dt, device="cuda"),
                    ws=torch.empty(lib.decode_attention_weights_workspace_bytes(b, hq, hkv, D, width, bs), dtype=torch.uint8, device="cuda"))

    def round_of(s, i):
        lib.launch_decode_attention_paged_weights(s["q"], *s["cache"], s["ctx"], s["bt"], hkv, D, bs, 0.088, s["w"], None, s["w"], s["out"][i], s["ws"])
        lib.evict_kvcache(*s["cache"], s["w"], None, s["ctx"], s["bt"], s["w"], s["bt"], s["lens"], hkv, D, bs, 590 - 10 * i, 4, 32)
        s["ctx"].copy_(s["lens"])

    alone, at_once = [state(1), state(2)], [state(1), state(2)]
    for s in alone:
        for i in range(40):
            round_of(s, i)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(40):
        for s, stream in zip(at_once, streams):
            with torch.cuda.stream(stream):
                round_of(s, i)
    torch.cuda.synchronize()
    for x, y in zip(alone, at_once):
        assert torch.equal(x["out"], y["out"]) and torch.equal(x["w"], y["w"]) and torch.equal(x["ctx"], y["ctx"])
        assert all(torch.equal(a, c) for a, c in zip(x["cache"], y["cache"])) and not torch.isnan(x["out"]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("kv,dtype,hkv,bs,lens,budget,sinks,recent,tables_are,weights_are", [
    ("same", "bfloat16", 2, 256, [46500], 20000, 4, 256, "same", "same"),                  # more keys than orders are kept of, alone on an SM
    ("int4", "float16", 1, 16, [45057, 46000], 45056, 0, 0, "same", "same"),
    ("int4", "bfloat16", 25, 256, [16385, 17000, 16700], 9000, 4, 1000, "same", "same"),   # and by two blocks to an SM
    ("int4", "bfloat16", 1, 256, [140000], 66000, 4, 128, "other", "other"),               # several tiles counted together
    ("same", "float16", 1, 256, [133000], 131080, 0, 1, "other", "same"),
    ("int4", "bfloat16", 2, 256, [140000], 139990, 100, 100, "same", "same"),
    ("same", "bfloat16", 2, 16, [700, 90, 1, 333], 100, 2, 30, "same", "other"),
    ("int4", "bfloat16", 2, 16, [700, 90, 1, 333], 100, 2, 30, "other", "same"),
    ("same", "float16", 2, 16, [700, 90, 1, 333], 100, 2, 30, "first", "same"),            # the first blocks of the old ones, as a narrower table
    ("int4", "bfloat16", 8, 48, [3000, 2000], 3000, 0, 0, "same", "same"),                 # nothing to do
])
def test_evict_in_place_and_of_long_contexts(kv, dtype, hkv, bs, lens, budget, sinks, recent, tables_are, weights_are):
    import torch
    rng = np.random.default_rng(budget + hkv)
    b = len(lens)
    kept = [min(n, budget) for n in lens]
    blocks = sum(-(-n // bs) for n in lens) + (sum(-(-n // bs) for n in kept) if tables_are == "other" else 0) + 2
    shape = (blocks * bs, hkv)
    if kv == "int4":
        cache = [torch.randint(0, 256, (*shape, 64), dtype=torch.uint8, device="cuda") for _ in range(2)]
        cache += [torch.randint(-2 ** 15, 2 ** 15, (*shape, 2), dtype=torch.int16, device="cuda").view(getattr(torch, dtype)) for _ in range(2)]
    else:
        cache = [torch.randint(-2 ** 15, 2 ** 15, (*shape, D), dtype=torch.int16, device="cuda").view(getattr(torch, dtype)) for _ in range(2)]
    tables = _tables(rng, lens, bs, blocks)
    new_tables = tables if tables_are == "same" else tables[:, :-(-max(kept) // bs)] if tables_are == "first" else _tables(rng, kept, bs, blocks, taken=set(tables.ravel()))
    w = np.float32(np.exp(2 * rng.standard_normal((b, hkv, tables.shape[1] * bs))))
    w[:, :, 5::7] = np.float32(0.25)
    before = [_np(c) for c in cache]
    want, want_w, want_lens = _evict_reference(before, tables, new_tables, lens, w, list(range(b)), bs, blocks, budget, sinks, recent)
    weights, bt = to_dev(w), to_dev(tables, torch.int32)
    new_w, new_lens = weights if weights_are == "same" else torch.full_like(weights, 7.0), torch.full((b,), -5, dtype=torch.int32, device="cuda")
    nvk().evict_kvcache(*(cache if kv == "int4" else [*cache, None, None]), weights, None, to_dev(np.array(lens), torch.int32), bt, new_w,
                        bt if tables_are == "same" else to_dev(np.ascontiguousarray(new_tables), torch.int32), new_lens, hkv, D, bs, budget, sinks, recent)
    torch.cuda.synchronize()
    assert new_lens.tolist() == want_lens.tolist() and np.array_equal(new_w.cpu().numpy(), want_w)
    assert weights_are == "same" or np.array_equal(weights.cpu().numpy(), w)
    assert all(np.array_equal(_np(got), exp) for got, exp in zip(cache, want))
