"""4-bit paged KV cache: nvk_store_kvcache_int4, nvk_gather_kvcache_int4, nvk_decode_attention_paged_int4.

The reference has no such cache, so the format is pinned by the 64-bit restatement of its definition in ref_int4.py (checked by hand on the CPU): the
store and the gather bit for bit, the decode within what its roundings allow."""
import ctypes

import numpy as np
import pytest

import ref_int4 as ref
from util import entry, nvk, to_dev

D = 128


@pytest.fixture(scope="module")
def built():
    entry.build()
    return nvk()


# ---- on the CPU --------------------------------------------------------------------------------------------------------------
def test_the_format_by_hand():
    x = np.zeros((5, D))
    x[0] = np.arange(D) % 16                                  # low 0, step 1: the numbers themselves
    x[1] = 2.5                                                # no range
    x[2, :4] = [-7.5, 7.5, 0.0, -7.0]                         # low -7.5, step 1: 7.5 between 7 and 8 goes up to 8, 0.5 to 1
    x[3, 5] = np.inf
    x[4, 6] = np.nan
    data, params = ref.quantise(x, "bfloat16")
    assert ref.numbers(data)[0].tolist() == x[0].tolist() and params[0].tolist() == [1.0, 0.0]
    assert (data[1] == 0).all() and params[1].tolist() == [0.0, 2.5]
    assert ref.numbers(data)[2][:5].tolist() == [0, 15, 8, 1, 8] and params[2].tolist() == [1.0, -7.5]
    assert data[0][0] == 0x10 and data[0][1] == 0x32          # element 2i in the low half
    assert np.isnan(params[3:]).all() and (data[3:] == 0).all()
    assert np.abs(ref.values(data, params)[:3] - x[:3]).max() <= 0.5


def test_half_a_step_is_the_most_that_an_element_is_off():
    rng = np.random.default_rng(5)
    for dtype in ("bfloat16", "float16"):
        x = ref.to_type(rng.standard_normal((200, D)) * 3.0, dtype)
        data, params = ref.quantise(x, dtype)
        # 15 steps are the range but for the rounding of the step
        most = params[..., :1] * 0.5 + 15 * params[..., :1] * ref.HALF_STEP[dtype]
        assert (np.abs(ref.values(data, params) - x) <= most).all()


def _call(lib, name, *args):
    rc = getattr(lib.lib(), name)(*args)
    return rc, lib.lib().nvk_last_error().decode()


L, I = ctypes.c_int64, ctypes.c_int
P, ODD = ctypes.c_void_p(256), ctypes.c_void_p(260)


def _store_args(**change):
    a = dict(key=P, value=P, k_cache=P, v_cache=P, k_params=P, v_params=P, slots=P, slot_dtype=I(3), tokens=L(4), hkv=I(2), d=I(128), rows=L(64), dtype=I(1),
             stream=None)
    a.update(change)
    return a.values()


def _gather_args(**change):
    a = dict(k_cache=P, v_cache=P, k_params=P, v_params=P, cu=P, cu_dtype=I(3), bt=P, bt_dtype=I(4), seqs=L(2), total=L(10), max_blocks=L(2), blocks=L(4),
             hkv=I(2), d=I(128), bs=I(16), key=P, value=P, dtype=I(0), stream=None)
    a.update(change)
    return a.values()


def _decode_args(**change):
    a = dict(q=P, k_cache=P, v_cache=P, k_params=P, v_params=P, ctx=P, ctx_dtype=I(3), bt=P, bt_dtype=I(3), batch=L(2), max_blocks=L(40), blocks=L(4), hq=I(8),
             hkv=I(2), d=I(128), bs=I(256), scale=ctypes.c_float(1.0), out=P, dtype=I(1), ws=None, ws_bytes=ctypes.c_size_t(0), stream=None)
    a.update(change)
    return a.values()


@pytest.mark.parametrize("change,code,word", [
    (dict(k_params=None), 1, "defined"), (dict(value=None), 1, "defined"), (dict(slots=None), 1, "defined"), (dict(dtype=I(2)), 3, "F16 or BF16"),
    (dict(d=I(64)), 3, "128"), (dict(d=I(0)), 1, "positive"), (dict(hkv=I(0)), 1, "positive"), (dict(slot_dtype=I(2)), 1, "int32 or int64"),
    (dict(tokens=L(-1)), 1, "positive"), (dict(rows=L(0)), 1, "positive"), (dict(key=ODD), 1, "aligned"), (dict(v_cache=ODD), 1, "aligned"),
    (dict(k_params=ctypes.c_void_p(258)), 1, "aligned"), (dict(tokens=L(1 << 31)), 1, "too many"), (dict(tokens=L(0)), 0, "")])
def test_store_refuses(built, change, code, word):
    rc, said = _call(built, "nvk_store_kvcache_int4", *_store_args(**change))
    assert rc == code and (rc == 0 or word in said), said


@pytest.mark.parametrize("change,code,word", [
    (dict(cu=None), 1, "defined"), (dict(key=None), 1, "defined"), (dict(dtype=I(2)), 3, "F16 or BF16"), (dict(d=I(256)), 3, "128"),
    (dict(cu_dtype=I(0)), 1, "int32 or int64"), (dict(seqs=L(0)), 1, "positive"), (dict(total=L(-1)), 1, "positive"), (dict(max_blocks=L(0)), 1, "positive"),
    (dict(blocks=L(0)), 1, "positive"), (dict(bs=I(0)), 1, "positive"), (dict(value=ODD), 1, "aligned"), (dict(total=L(0)), 0, ""),
    (dict(total=L(1 << 40)), 3, "too many")])
def test_gather_refuses(built, change, code, word):
    rc, said = _call(built, "nvk_gather_kvcache_int4", *_gather_args(**change))
    assert rc == code and (rc == 0 or word in said), said


@pytest.mark.parametrize("change,code,word", [
    (dict(q=None), 1, "requires"), (dict(v_params=None), 1, "requires"), (dict(ctx_dtype=I(1)), 1, "int32 or int64"), (dict(batch=L(-1)), 1, "positive"),
    (dict(hq=I(7)), 1, "divisible"), (dict(dtype=I(2)), 3, "F16 / BF16"), (dict(d=I(64)), 3, "head_dim"), (dict(hq=I(18)), 3, "8 query heads"),
    (dict(bs=I(24)), 3, "multiple"), (dict(q=ODD), 3, "aligned"), (dict(ws=P, ws_bytes=ctypes.c_size_t(64)), 1, "workspace"),
    (dict(ws=ODD, ws_bytes=ctypes.c_size_t(1 << 30)), 1, "aligned"), (dict(batch=L(0)), 0, "")])
def test_decode_refuses(built, change, code, word):
    rc, said = _call(built, "nvk_decode_attention_paged_int4", *_decode_args(**change))
    assert rc == code and (rc == 0 or word in said), said


# ---- on the GPU --------------------------------------------------------------------------------------------------------------
def _typed(rng, shape, dtype, std=1.0, mean=0.0):
    return ref.to_type(rng.standard_normal(shape) * std + mean, dtype)


def _dev(x, dtype):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x)).to(getattr(torch, dtype)).cuda()


def _cache(rng, rows, hkv, dtype):
    """A cache of stored normal vectors: device tensors, and their values in 64 bits."""
    import torch
    out = []
    for std in (1.0, 0.7):
        data, params = ref.quantise(_typed(rng, (rows, hkv, D), dtype, std), dtype)
        out.append((torch.from_numpy(data).cuda(), _dev(params, dtype), ref.values(data, params), np.abs(ref.numbers(data) - 7.5) * params[..., :1]))
    return out


def _bits(t):
    import torch
    return t.detach().cpu().view(torch.int16).numpy()


def _hard_vectors(dtype):
    """Vectors on which a quantiser goes wrong: constant, zero, on the borders between numbers, tiny, huge, not finite."""
    tiny = {"bfloat16": 2.0 ** -133, "float16": 2.0 ** -24}[dtype]
    huge = {"bfloat16": 3.0e38, "float16": 65504.0}[dtype]
    steps = np.arange(D) % 31 * 0.5                                      # every border of a range of 15
    x = [np.zeros(D), np.full(D, -3.25), steps, -steps, steps * 2.0 ** -12, steps - 7.5, np.arange(D) % 2 * tiny, np.arange(D) % 24 * tiny, np.arange(D) % 11 * tiny,
         np.arange(D) % 90 * tiny, np.where(np.arange(D) % 2, huge / 4, -huge / 4), np.where(np.arange(D) % 2, huge, -huge),
         np.where(np.arange(D) == 127, np.inf, 1.0), np.where(np.arange(D) == 3, -np.inf, 1.0), np.where(np.arange(D) == 64, np.nan, 1.0), np.full(D, np.nan),
         np.where(np.arange(D) == 9, 1.0, -0.0), np.where(np.arange(D) == 0, 100.0, 2.0 ** -10 * np.arange(D)), np.full(D, huge)]
    return ref.to_type(np.stack(x), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tokens,hkv,index", [("bfloat16", 1, 1, "int32"), ("bfloat16", 97, 8, "int64"), ("float16", 70, 3, "int32"), ("float16", 2, 8, "int64"),
                                                    ("bfloat16", 1111, 5, "int32")])
def test_store_is_bit_identical_to_the_definition(dtype, tokens, hkv, index):
    import torch
    rng = np.random.default_rng(tokens)
    rows = tokens + 40
    key, val = _typed(rng, (tokens, hkv, D), dtype, 1.3, 0.4), _typed(rng, (tokens, hkv, D), dtype, 0.02)
    hard = _hard_vectors(dtype)
    if tokens > 40:
        key[3:3 + len(hard), 0], val[20:20 + len(hard), hkv - 1] = hard, hard[::-1]
    # values on a coarse grid: many lie exactly between two numbers
    key[-1], val[-1] = np.round(key[-1] * 2) / 2, np.round(val[-1] * 64) / 64
    slots = rng.permutation(rows)[:tokens]
    if tokens > 40:
        slots[::9], slots[4] = -1, rows + 3
    kc, vc = (torch.full((rows, hkv, D // 2), 0x5a, dtype=torch.uint8, device="cuda") for _ in range(2))
    kp, vp = (torch.full((rows, hkv, 2), -2.0, dtype=getattr(torch, dtype), device="cuda") for _ in range(2))
    nvk().store_kvcache_int4(_dev(key, dtype), _dev(val, dtype), kc, vc, kp, vp, to_dev(slots, getattr(torch, index)))
    torch.cuda.synchronize()
    for x, data, params in ((key, kc, kp), (val, vc, vp)):
        want_data, want_params = np.full((rows, hkv, D // 2), 0x5a, np.uint8), np.full((rows, hkv, 2), -2.0)
        good = (slots >= 0) & (slots < rows)
        want_data[slots[good]], want_params[slots[good]] = (y[good] for y in ref.quantise(x, dtype))
        got = params.double().cpu().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(want_params)) and np.array_equal(np.nan_to_num(got), np.nan_to_num(want_params))
        assert np.array_equal(data.cpu().numpy(), want_data)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hkv,bs,lens,index", [("bfloat16", 8, 256, [589], "int32"), ("float16", 1, 16, [1, 0, 33, 16, 0], "int64"),
                                                     ("bfloat16", 3, 48, [100, 7, 300, 1, 48, 95], "int32"), ("float16", 2, 5, [3, 5, 6, 11], "int32")])
def test_gather_brings_the_values_rounded_once_more(dtype, hkv, bs, lens, index):
    import torch
    rng = np.random.default_rng(len(lens))
    need = [-(-n // bs) for n in lens]
    blocks, width = sum(need) + 2, max(need)
    (kc, kp, kv, _), (vc, vp, vv, _) = _cache(rng, blocks * bs, hkv, dtype)
    tables = np.full((len(lens), width), 77777)                       # (entries behind a sequence's end are never used)
    perm, at = rng.permutation(blocks), 0
    for i, n in enumerate(need):
        tables[i, :n] = perm[at:at + n]
        at += n
    if len(lens) == 6:
        tables[2, 1], tables[0, 0] = -3, blocks                       # outside the cache: zeros
    cu = np.concatenate([[0], np.cumsum(lens)])
    total = int(cu[-1]) + 9
    key, value = (torch.full((total, hkv, D), float("nan"), dtype=getattr(torch, dtype), device="cuda") for _ in range(2))
    dt = getattr(torch, index)
    nvk().gather_kvcache_int4(kc, vc, kp, vp, to_dev(cu, dt), to_dev(tables, dt), hkv, D, bs, key, value)
    torch.cuda.synchronize()
    at = np.concatenate([ref.places(tables[i], n, bs, blocks) for i, n in enumerate(lens)] + [np.full(9, -1)])
    for got, x in ((key, kv), (value, vv)):
        assert np.array_equal(got.double().cpu().numpy(), ref.to_type(ref.context(x, at), dtype))
    # a total that cuts the last sequences off
    short = max(1, total - 9 - lens[-1] // 2 - 1)
    key2, value2 = torch.full_like(key[:short], 5.0), torch.full_like(value[:short], 5.0)
    nvk().gather_kvcache_int4(kc, vc, kp, vp, to_dev(cu, dt), to_dev(tables, dt), hkv, D, bs, key2, value2)
    assert torch.equal(key2, key[:short]) and torch.equal(value2, value[:short])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hq,hkv,bs,lens,index,use_ws", [
    ("bfloat16", 32, 8, 256, [300], "int32", True),
    ("bfloat16", 32, 8, 256, [0, 1, 15, 16, 17, 255, 256, 257, 700], "int64", True),
    ("float16", 4, 1, 64, [1000, 3, 64, 65, 129], "int32", False),
    ("bfloat16", 8, 8, 16, [31, 47, 500], "int32", True),
    ("float16", 14, 2, 48, [1000, 1, 2000], "int32", True),
    ("bfloat16", 8, 1, 256, [4000, 9000, 100], "int64", True),
    ("float16", 6, 2, 256, [3000] * 3 + [1], "int32", True),
    ("bfloat16", 16, 8, 256, [200 + 37 * i for i in range(40)], "int32", True),
])
def test_decode_matches_64_bits(dtype, hq, hkv, bs, lens, index, use_ws):
    import torch
    rng = np.random.default_rng(hq * 100 + len(lens))
    need = [-(-n // bs) for n in lens]
    blocks, width = sum(need) + 1, max(need) + 1
    (kc, kp, kv, _), (vc, vp, vv, spread) = _cache(rng, blocks * bs, hkv, dtype)
    spare = rng.permutation(blocks)[-1]
    kp[spare * bs:(spare + 1) * bs], vp[spare * bs:(spare + 1) * bs] = float("nan"), float("nan")     # a block of no context
    free = [i for i in rng.permutation(blocks) if i != spare]
    tables = np.full((len(lens), width), spare)
    for i, n in enumerate(need):
        for j in range(n):
            tables[i, j] = free.pop()
        # rows behind the end of the last block hold NaN
        if lens[i] % bs:
            row = tables[i, n - 1] * bs + lens[i] % bs
            kp[row:(tables[i, n - 1] + 1) * bs], vp[row:(tables[i, n - 1] + 1) * bs] = float("nan"), float("nan")
    if len(lens) == 3 and bs == 48:
        tables[2, 3] = blocks + 5                                     # outside the cache: zeros
    ctx = np.array(lens)
    if len(lens) == 9:
        ctx[0] = -4                                                   # an empty context
    q, scale = _typed(rng, (len(lens), hq, D), dtype), 1.0 / np.sqrt(D)
    lib, dt = nvk(), getattr(torch, index)
    out = torch.full((len(lens), hq, D), float("nan"), dtype=getattr(torch, dtype), device="cuda")
    ws = torch.empty(max(16, lib.decode_attention_workspace_bytes(len(lens), hq, hkv, D, width, bs)), dtype=torch.uint8, device="cuda") if use_ws else None
    lib.launch_decode_attention_paged_int4(_dev(q, dtype), kc, vc, kp, vp, to_dev(ctx, dt), to_dev(tables, dt), hkv, D, bs, scale, out, ws)
    torch.cuda.synchronize()
    got, u = out.double().cpu().numpy(), ref.HALF_STEP[dtype]
    for i, n in enumerate(lens):
        at = ref.places(tables[i], n, bs, blocks)
        k, v = ref.context(kv, at), ref.context(vv, at)
        want, p = ref.attend(q[i], k, v, scale)
        if n == 0:
            assert (got[i] == 0).all()
            continue
        # p' and the result are rounded to the type; a score off by e moves p by 2e, and the result by 2e times the largest value
        around = np.einsum("jgn,njd->jgd", p.reshape(hkv, hq // hkv, n), ref.context(spread, at)).reshape(hq, D)
        e = ref.score_error(q[i], np.abs(k).max() + 31 * 0.5, scale) + 2.0 ** -20
        assert (np.abs(got[i] - want) <= u * around + u * np.abs(want) + 2 * e * (np.abs(v).max() + 1)).all(), (i, np.abs(got[i] - want).max())


@pytest.mark.gpu
def test_a_context_beyond_the_table_is_cut_off_and_one_key_is_its_value():
    import torch
    rng = np.random.default_rng(2)
    hq, hkv, bs = 8, 2, 16
    (kc, kp, kv, _), (vc, vp, vv, _) = _cache(rng, 4 * bs, hkv, "bfloat16")
    q = _dev(_typed(rng, (2, hq, D), "bfloat16"), "bfloat16")
    tables = to_dev(np.array([[3, 1], [2, 0]]), torch.int64)
    out, cut = torch.empty_like(q), torch.empty_like(q)
    for lens, to in (([1 << 40, 1], out), ([32, 1], cut)):
        nvk().launch_decode_attention_paged_int4(q, kc, vc, kp, vp, to_dev(np.array(lens), torch.int64), tables, hkv, D, bs, 0.1, to)
    torch.cuda.synchronize()
    assert torch.equal(out, cut)
    want = np.repeat(vv[2 * bs], hq // hkv, 0)
    # p' = step exactly; one rounding of the result, and fp32's of the sum's terms, of up to 23.5 steps
    assert (np.abs(out[1].double().cpu().numpy() - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -18).all()


@pytest.mark.gpu
def test_values_far_from_one_and_vectors_that_are_not_finite():
    import torch
    rng = np.random.default_rng(9)
    hq, hkv, bs, n = 4, 1, 64, 150
    for dtype, size in (("bfloat16", 1e30), ("bfloat16", 1e-30), ("float16", 300.0), ("float16", 0.05)):
        key, val = _typed(rng, (192, hkv, D), dtype), _typed(rng, (192, hkv, D), dtype, size)
        (kd, kpar), (vd, vpar) = ref.quantise(key, dtype), ref.quantise(val, dtype)
        q = _typed(rng, (1, hq, D), dtype)
        out = torch.empty((1, hq, D), dtype=getattr(torch, dtype), device="cuda")
        kp, vp = _dev(kpar, dtype), _dev(vpar, dtype)
        args = torch.from_numpy(kd).cuda(), torch.from_numpy(vd).cuda(), kp, vp, to_dev(np.array([n]), torch.int32), to_dev(np.array([[0, 1, 2]]), torch.int32)
        nvk().launch_decode_attention_paged_int4(_dev(q, dtype), *args, hkv, D, bs, 0.088, out)
        torch.cuda.synchronize()
        v = ref.values(vd, vpar)
        want, p = ref.attend(q[0], ref.values(kd, kpar)[:n], v[:n], 0.088)
        u = ref.HALF_STEP[dtype]
        around = p @ (np.abs(ref.numbers(vd) - 7.5) * vpar[..., :1])[:n, 0]
        e = ref.score_error(q[0], 20.0, 0.088) + 2.0 ** -20
        assert (np.abs(out[0].double().cpu().numpy() - want) <= u * around + u * np.abs(want) + 2 * e * np.abs(v).max()).all(), (dtype, size)
        vp[7] = float("nan")                                          # one value that was not finite: every head's result is NaN, as with a 16-bit cache
        nvk().launch_decode_attention_paged_int4(_dev(q, dtype), *args, hkv, D, bs, 0.088, out)
        assert torch.isnan(out).all()


@pytest.mark.gpu
def test_wrong_tensors_are_refused():
    import torch
    lib, bf = nvk(), torch.bfloat16
    kc, kp = torch.zeros((32, 2, 64), dtype=torch.uint8, device="cuda"), torch.zeros((32, 2, 2), dtype=bf, device="cuda")
    x, slots = torch.zeros((3, 2, D), dtype=bf, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    for bad in (dict(key=x.half()), dict(key=x[:2]), dict(key=x.view(6, D)), dict(kc=kc.to(torch.int16)), dict(kp=kp.half()), dict(kp=kp[:16]), dict(slots=slots[:2]),
                dict(slots=slots.float()), dict(kc=kc.transpose(0, 1)), dict(kc=kc.cpu()), dict(vc=kc[:16])):
        a = dict(key=x, value=x, kc=kc, vc=kc, kp=kp, vp=kp, slots=slots)
        a.update(bad)
        with pytest.raises(ValueError):
            lib.store_kvcache_int4(*a.values())
    lib.store_kvcache_int4(x[:0], x[:0], kc, kc, kp, kp, slots[:0])   # nothing to do
    cu, bt = to_dev(np.array([0, 5]), torch.int32), to_dev(np.array([[0, 1]]), torch.int32)
    rows = torch.zeros((5, 2, D), dtype=bf, device="cuda")
    for bad in (dict(key=rows[:4]), dict(key=rows.half()), dict(cu=cu[:1]), dict(bt=bt[0]), dict(bs=0), dict(d=64), dict(vp=kp[:1])):
        a = dict(kc=kc, vc=kc, kp=kp, vp=kp, cu=cu, bt=bt, hkv=2, d=D, bs=16, key=rows, value=rows)
        a.update(bad)
        with pytest.raises(ValueError):
            lib.gather_kvcache_int4(*a.values())
    q, ctx = torch.zeros((1, 8, D), dtype=bf, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    for bad in (dict(q=q.float()), dict(q=q.half()), dict(ctx=torch.ones(2, dtype=torch.int32, device="cuda")), dict(out=q[..., :64].contiguous()), dict(kp=kp.half()),
                dict(bs=8), dict(bt=bt[:0]), dict(q=q.view(1, 16, 64))):
        a = dict(q=q, kc=kc, vc=kc, kp=kp, vp=kp, ctx=ctx, bt=bt, hkv=2, d=D, bs=16, scale=1.0, out=torch.empty_like(q))
        a.update(bad)
        with pytest.raises(ValueError):
            lib.launch_decode_attention_paged_int4(*a.values())
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("batch,longest", [(120, 2000), (200, 2048), (300, 1700), (460, 900), (60, 8000)])
def test_decode_of_many_contexts_however_they_are_shared_out(batch, longest):
    """Blocks of four and of eight warps, whole contexts in order of length, long chunks: what comes out is within the roundings of what single calls give, and
    the same in a second run."""
    import torch
    rng = np.random.default_rng(batch)
    bs, dtype = 256, "bfloat16"
    hkv = 8 if longest > 4096 else 1
    hq = 4 * hkv
    lens = [1 + (i * 7919) % longest for i in range(batch)]
    lens[batch // 2] = longest
    width = -(-longest // bs)
    blocks = 40
    (kc, kp, _, _), (vc, vp, vv, spread) = _cache(rng, blocks * bs, hkv, dtype)
    tables = np.stack([rng.permutation(blocks)[:width] for _ in range(batch)])         # (contexts may share blocks)
    q = _dev(_typed(rng, (batch, hq, D), dtype), dtype)
    lib, dt = nvk(), torch.int32
    ctx, bt = to_dev(np.array(lens), dt), to_dev(tables, dt)
    ws = torch.empty(max(16, lib.decode_attention_workspace_bytes(batch, hq, hkv, D, width, bs)), dtype=torch.uint8, device="cuda")
    out, again, single = (torch.full_like(q, float("nan")) for _ in range(3))
    for to in (out, again):
        lib.launch_decode_attention_paged_int4(q, kc, vc, kp, vp, ctx, bt, hkv, D, bs, 0.088, to, ws)
    for i in range(0, batch, 37):
        lib.launch_decode_attention_paged_int4(q[i:i + 1], kc, vc, kp, vp, ctx[i:i + 1], bt[i:i + 1], hkv, D, bs, 0.088, single[i:i + 1])
    torch.cuda.synchronize()
    assert torch.equal(out, again) and not torch.isnan(out).any()
    # both round p' to f16 (2^-11 of at most 15 steps each way) and the result to bf16 (half a step each)
    most = 2 * 2.0 ** -11 * 15 * float(spread.max()) / 7.5 + 2 * 2.0 ** -8 * float(np.abs(vv).max())
    assert (single[::37].float() - out[::37].float()).abs().max().item() <= most


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,power", [("bfloat16", 16), ("bfloat16", 20), ("bfloat16", 60), ("float16", 17)])
@pytest.mark.parametrize("place", [0, 40, 289])
def test_a_value_of_a_large_range_without_weight_leaves_the_others_alone(dtype, power, place):
    """One key whose value spans 2^power times what the others do, and that hardly any of the attention goes to: before, among and after the others."""
    import torch
    rng = np.random.default_rng(power)
    hq, hkv, bs, n, scale = 4, 1, 64, 290, 0.088
    key, val = _typed(rng, (320, hkv, D), dtype, 0.25), _typed(rng, (320, hkv, D), dtype, 2.0 ** -4)
    q = _typed(rng, (1, hq, D), dtype)
    away = -q[0].sum(0)
    key[place, 0] = ref.to_type(away * (80.0 + power) / scale / np.abs(q[0] @ away).min(), dtype)
    val[place] = ref.to_type(val[place] * 2.0 ** power, dtype)
    (kd, kpar), (vd, vpar) = ref.quantise(key, dtype), ref.quantise(val, dtype)
    k, v = ref.values(kd, kpar)[:n], ref.values(vd, vpar)[:n]
    want, p = ref.attend(q[0], k, v, scale)
    assert p[:, place].max() * 2.0 ** power < 2.0 ** -24                  # what the key itself adds
    out = torch.empty((1, hq, D), dtype=getattr(torch, dtype), device="cuda")
    nvk().launch_decode_attention_paged_int4(_dev(q, dtype), torch.from_numpy(kd).cuda(), torch.from_numpy(vd).cuda(), _dev(kpar, dtype), _dev(vpar, dtype),
                                             to_dev(np.array([n]), torch.int32), to_dev(np.arange(5)[None], torch.int32), hkv, D, bs, scale, out)
    # p' is rounded to f16 (2^-11 of it, or 2^-22 of the largest p step) and multiplied by up to 15, the result is rounded to the type; a score off by e moves
    # p by 2e of itself.  What a key without weight can do to the sums in fp32 goes by its p step as well.
    u, step = ref.HALF_STEP[dtype], vpar[:n, 0, 0]
    e = ref.score_error(q[0], np.abs(np.delete(k, place, 0)).max() + 31 * 0.25, scale) + 2.0 ** -20
    most = 15 * (2.0 ** -11 * (p @ step) + 2.0 ** -22 * n * (p * step).max(-1))[:, None] + u * np.abs(want) + 2 * e * (p @ np.abs(v[:, 0]) + np.abs(want)) + 2.0 ** -20
    assert (np.abs(out[0].double().cpu().numpy() - want) <= most).all(), (np.abs(out[0].double().cpu().numpy() - want) / most).max()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,other", [("bfloat16", "infinite"), ("bfloat16", "large"), ("float16", "infinite"), ("float16", "large")])
def test_a_query_head_of_other_magnitude_leaves_the_others_alone(dtype, other):
    """Of a group of four heads one holds an infinity, and another (BF16) elements beyond f16's range; or one is 2^28 (F16: 2^15) times the others."""
    import torch
    rng = np.random.default_rng(3)
    hq, hkv, bs, n, scale = 4, 1, 16, 150, 0.088
    small = 2.0 ** -12 if dtype == "float16" else 1.0
    q = _typed(rng, (1, hq, D), dtype, small)
    key_std = 1.0 / small
    if other == "infinite":
        q[0, 2, 77] = np.inf
        if dtype == "bfloat16":
            q[0, 0] *= 2.0 ** 18
            key_std = 2.0 ** -18
    else:
        q[0, 2] *= 2.0 ** (15 if dtype == "float16" else 28)
    key, val = _typed(rng, (160, hkv, D), dtype, key_std), _typed(rng, (160, hkv, D), dtype)
    (kd, kpar), (vd, vpar) = ref.quantise(key, dtype), ref.quantise(val, dtype)
    k, v = ref.values(kd, kpar)[:n], ref.values(vd, vpar)[:n]
    out = torch.empty((1, hq, D), dtype=getattr(torch, dtype), device="cuda")
    nvk().launch_decode_attention_paged_int4(_dev(q, dtype), torch.from_numpy(kd).cuda(), torch.from_numpy(vd).cuda(), _dev(kpar, dtype), _dev(vpar, dtype),
                                             to_dev(np.array([n]), torch.int32), to_dev(np.arange(10)[None], torch.int32), hkv, D, bs, scale, out)
    got, u, step = out[0].double().cpu().numpy(), ref.HALF_STEP[dtype], vpar[:n, 0, 0]
    for h in range(hq):
        if h == 2 and other == "infinite":
            assert np.isnan(got[h]).all()
            continue
        want, p = (x[0] for x in ref.attend(q[0, h:h + 1], k, v, scale))
        # (as above: p' rounded to f16, the result rounded, scores off by e); the large head gives one key everything, by far more than its e
        e = ref.score_error(q[0, h:h + 1], np.abs(k).max() + 31 * 0.5 * key_std, scale) + 2.0 ** -20
        if h == 2:
            top = np.sort(q[0, h] @ k[:, 0].T * scale)
            assert top[-1] - top[-2] > 4 * e + 200
            e = 2.0 ** -20
        assert (np.abs(got[h] - want) <= 15 * 2.0 ** -11 * (p @ step) + u * np.abs(want) + 2 * e * (p @ np.abs(v[:, 0]) + np.abs(want)) + 2.0 ** -20).all(), h
