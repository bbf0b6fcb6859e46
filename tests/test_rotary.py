"""nvk_rotary_embedding against the formula in 64 bits and more, and nvk_rotary_inv_freq."""
import ctypes
import math

import numpy as np
import pytest

import ref_blocks8 as ref
from util import entry, nvk


@pytest.fixture(scope="module")
def built():
    entry.build()
    return nvk()


# ---- on the CPU --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rot", [2, 10, 64, 128])
@pytest.mark.parametrize("scaling,factor,original,low,high", [("plain", 1.0, 0.0, 0.0, 0.0), ("linear", 4.0, 0.0, 0.0, 0.0), ("base", 8.0, 0.0, 0.0, 0.0),
                                                              ("parts", 8.0, 8192.0, 1.0, 4.0), ("yarn", 32.0, 32768.0, 1.0, 32.0)])
def test_frequencies(built, rot, scaling, factor, original, low, high):
    if scaling == "base" and rot == 2:
        with pytest.raises(ValueError, match="more than one pair"):
            built.rotary_inv_freq(rot, 10000.0, scaling, factor)
        return
    got, m = built.rotary_inv_freq(rot, 500000.0, scaling, factor, original, low, high)
    want, factor_ = ref.inv_freq(rot, 500000.0, scaling, factor, original, low, high)
    assert np.allclose(got, want, rtol=2.0 ** -23, atol=0) and math.isclose(m, factor_, rel_tol=2.0 ** -23)
    if scaling == "base" and rot > 2:
        assert math.isclose(got[-1], 500000.0 ** (-(rot - 2) / rot) / factor, rel_tol=1e-6)   # the slowest pair as by linear scaling


@pytest.mark.parametrize("change,word", [(dict(rotary_dim=7), "even"), (dict(rotary_dim=0), "even"), (dict(base=0.0), "base"), (dict(scaling="linear", factor=0.5), "factor"),
                                         (dict(scaling="yarn", factor=2.0), "original"), (dict(scaling="slow"), "scaling must be"),
                                         (dict(scaling="parts", factor=2.0, original_positions=10.0, low_turns=4.0, high_turns=4.0), "high_turns")])
def test_frequencies_refuse(built, change, word):
    with pytest.raises(ValueError, match=word):
        built.rotary_inv_freq(**{**dict(rotary_dim=64), **change})


L, I = ctypes.c_int64, ctypes.c_int
P, Q = ctypes.c_void_p(1 << 20), ctypes.c_void_p(1 << 24)


@pytest.mark.parametrize("change,code,word", [
    (dict(q=None), 1, "defined"), (dict(f=None), 1, "defined"), (dict(k=None), 1, "together"), (dict(dtype=I(3)), 1, "float16"), (dict(pos_dtype=I(2)), 1, "int32 or int64"),
    (dict(rows=L(-1)), 1, "positive"), (dict(hkv=I(0)), 1, "positive"), (dict(rot=I(63)), 1, "even"), (dict(rot=I(130)), 1, "at most head_dim"), (dict(rot=I(0)), 1, "positive"),
    (dict(d=I(1026), rot=I(2), q_stride=L(1 << 16), k_stride=L(1 << 16), qo_stride=L(1 << 16), ko_stride=L(1 << 16)), 3, "1024"), (dict(q_stride=L(1000)), 1, "less than a row"),
    (dict(qo=ctypes.c_void_p((1 << 20) + 64)), 1, "overlap"), (dict(qo=P, qo_stride=L(2048)), 1, "overlap"), (dict(q=ctypes.c_void_p((1 << 20) + 1)), 1, "misaligned"),
    (dict(f=ctypes.c_void_p(2)), 1, "misaligned"), (dict(rows=L(0)), 0, ""),
    (dict(hq=I((1 << 19) + 1), q_stride=L(1 << 40), qo_stride=L(1 << 40)), 3, "too many heads"), (dict(hkv=I((1 << 31) - 1), k_stride=L(1 << 40), ko_stride=L(1 << 40)), 3, "too many heads")])
def test_refuses(built, change, code, word):
    a = dict(q=P, k=ctypes.c_void_p(1 << 22), pos=P, pos_dtype=I(3), f=P, factor=ctypes.c_float(1.0), rows=L(4), hq=I(8), hkv=I(2), d=I(128), rot=I(128), pairs=I(0),
             q_stride=L(1024), k_stride=L(256), qo=Q, ko=ctypes.c_void_p(1 << 25), qo_stride=L(1024), ko_stride=L(256), dtype=I(1), stream=None)
    a.update(change)
    rc = built.lib().nvk_rotary_embedding(*a.values())
    said = built.lib().nvk_last_error().decode()
    assert rc == code and (rc == 0 or word in said), said


# ---- on the GPU --------------------------------------------------------------------------------------------------------------
# With |a|, |b| <= A: cosine and sine are off by 2^-53 of the turns (none to speak of below 2^27 turns), 2^-25 of a turn in the fraction (2 pi 2^-25 = 2^-22.3), sincospi's own
# few ulp (2^-23) and half a unit for the factor, 2^-24: together below 2^-21.  Two products and a sum: 2 A factor (2^-21 + 2^-24 + 2^-24), then the rounding to the type.
def _tolerance(want, top, factor, dtype):
    tiny = {"bfloat16": 2.0 ** -134, "float16": 2.0 ** -25, "float32": 2.0 ** -150}[dtype]
    return np.abs(want) * ref.HALF_STEP[dtype] + 2 * top * factor * (2.0 ** -21 + 2.0 ** -23) * 1.01 + tiny


def _inputs(rng, rows, heads, d, dtype, packed):
    """Rows as a part of wider ones, or by themselves; in 64 bits too."""
    import torch
    x = torch.from_numpy(rng.standard_normal((rows, heads * d + (packed if packed else 0)))).to(getattr(torch, dtype)).cuda()
    part = x[:, packed // 2:packed // 2 + heads * d] if packed else x
    return part.unflatten(1, (heads, d))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("rows,hq,hkv,d,rot", [(1, 32, 8, 128, 128), (7, 16, 8, 128, 64), (300, 4, 1, 64, 64), (2, 3, 1, 80, 20), (5, 14, 2, 96, 24), (3, 1, 1, 2, 2),
                                               (9, 6, 2, 192, 48), (2500, 4, 2, 64, 32), (4, 2, 1, 256, 256), (3, 5, 3, 33, 6), (2, 2, 2, 1024, 1000)])
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("packed", [0, 256, 6])
def test_against_the_formula(dtype, rows, hq, hkv, d, rot, pairs, packed):
    import torch
    rng = np.random.default_rng(rows + d + rot)
    q, k = (_inputs(rng, rows, h, d, dtype, packed) for h in (hq, hkv))
    wide = rows % 2 == 1
    positions = rng.integers(-5, 1 << 20, rows)
    positions[:1] = 0
    f = torch.tensor(nvk().rotary_inv_freq(rot, 10000.0)[0], dtype=torch.float32, device="cuda")
    factor = 1.25 if pairs else 1.0
    pos = torch.from_numpy(positions).to(torch.int64 if wide else torch.int32).cuda()
    before = [q.clone(), k.clone()]
    out = [torch.full_like(x.contiguous(), float("nan")) for x in (q, k)]
    nvk().rotary_embedding(q, k, pos, f, pairs, factor, *out)
    for x, y, was in zip((q, k), out, before):
        assert torch.equal(x, was)
        want = ref.rotary(was.double().cpu().numpy(), positions, f.double().tolist(), pairs, factor)
        top = np.abs(was.double().cpu().numpy()).max()
        got = y.double().cpu().numpy()
        assert (np.abs(got - want) <= _tolerance(want, top, factor, dtype)).all()
        assert torch.equal(y[..., rot:], was[..., rot:])
    assert torch.equal(out[0][0, :, :rot], before[0][0, :, :rot] if factor == 1.0 else (before[0][0, :, :rot].float() * factor).to(q.dtype))   # position 0
    # in place, inside the packed rows: the same bits, and nothing else is touched
    holder = [x._base if x._base is not None else x for x in (q, k)]
    kept = [h.clone() for h in holder]
    nvk().rotary_embedding(q, k, pos, f, pairs, factor)
    for x, y, h, was in zip((q, k), out, holder, kept):
        assert torch.equal(x, y)
        n = x.shape[1] * x.shape[2]
        flat, old = h.reshape(rows, -1), was.reshape(rows, -1)
        assert torch.equal(flat[:, :packed // 2], old[:, :packed // 2]) and torch.equal(flat[:, packed // 2 + n:], old[:, packed // 2 + n:])


@pytest.mark.gpu
@pytest.mark.parametrize("position", [2 ** 24 + 1, 2 ** 31 - 1, 2 ** 40 + 12345, -(2 ** 33) - 7])
def test_far_positions(position):
    """2^40 radians are 2^37.3 turns, in 64 bits off by 2^-14 of a turn: below 2^-11 radians."""
    import torch
    rng = np.random.default_rng(1)
    x = torch.from_numpy(rng.standard_normal((1, 2, 64))).float().cuda()
    f = [1.0, 0.5, 2.0 ** -7, 0.1] * 8
    fd = torch.tensor(f, dtype=torch.float32, device="cuda")
    out = torch.empty_like(x)
    nvk().rotary_embedding(x, None, torch.tensor([position], device="cuda"), fd, query_out=out)
    # the angle with 80 digits
    import decimal
    decimal.getcontext().prec = 80
    pi = decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")
    angle = [float((decimal.Decimal(position) * decimal.Decimal(v)).remainder_near(2 * pi)) for v in fd.double().tolist()]
    c, s = np.cos(angle), np.sin(angle)
    y = x.double().cpu().numpy()
    want = np.concatenate([y[..., :32] * c - y[..., 32:] * s, y[..., 32:] * c + y[..., :32] * s], -1)
    off = 2 * math.pi * abs(position) / (2 * math.pi) * 2.0 ** -52     # two roundings of the turns, in radians
    assert np.abs(out.double().cpu().numpy() - want).max() <= 2 * np.abs(y).max() * (off + 2.0 ** -21 + 2.0 ** -23) + 2.0 ** -23


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("rows,heads,d,rot", [(14300, 1, 1024, 1024), (2400, 2, 1024, 1024), (19000, 1, 128, 128), (3000, 1, 1024, 8)])
@pytest.mark.parametrize("pairs", [False, True])
def test_many_rows_of_few_heads(dtype, rows, heads, d, rot, pairs):
    """As many rows to a block, and as many angles, as there can be; queries alone, and another call of them on a second stream at the same time."""
    import torch
    rng = np.random.default_rng(rows)
    sets, streams = [], [torch.cuda.Stream() for _ in range(2)]
    f = torch.tensor(nvk().rotary_inv_freq(rot, 10000.0)[0], dtype=torch.float32, device="cuda")
    for _ in streams:
        x = torch.from_numpy(rng.standard_normal((rows, heads, d))).to(getattr(torch, dtype)).cuda()
        sets.append((x, torch.from_numpy(rng.integers(0, 1 << 17, rows)).cuda(), torch.full_like(x, float("nan"))))
    torch.cuda.synchronize()
    for s, (x, pos, out) in zip(streams, sets):
        with torch.cuda.stream(s):
            nvk().rotary_embedding(x, None, pos, f, pairs, query_out=out)
    torch.cuda.synchronize()
    for x, pos, out in sets:
        y = x.double().cpu().numpy()
        want = ref.rotary(y, pos.tolist(), f.double().tolist(), pairs, 1.0)
        assert (np.abs(out.double().cpu().numpy() - want) <= _tolerance(want, np.abs(y).max(), 1.0, dtype)).all()
        assert torch.equal(out[..., rot:], x[..., rot:])


@pytest.mark.gpu
def test_the_prologue_rotates_alike():
    """Half of a head against the other half by the table of the fused prologue: the same pairs, the same signs."""
    import torch
    rng = np.random.default_rng(2)
    rows, hq, hkv, d = 40, 8, 2, 128
    qkv = torch.from_numpy(rng.standard_normal((rows, (hq + 2 * hkv) * d))).to(torch.bfloat16).cuda()
    f, _ = nvk().rotary_inv_freq(d, 10000.0)
    angle = torch.arange(64, device="cuda").double()[:, None] * torch.tensor(f, device="cuda", dtype=torch.float64)
    table = torch.cat([angle.cos(), angle.sin()], -1).float()
    pos = torch.from_numpy(rng.integers(0, 64, rows)).int().cuda()
    q_out, k_out, v_out = (torch.empty(rows, h, d, dtype=qkv.dtype, device="cuda") for h in (hq, hkv, hkv))
    nvk().fused_split_norm_rope_store(qkv, pos, None, None, 1e-6, table, None, k_out, v_out, hq, hkv, d, q_out)
    q, k = qkv[:, :hq * d].unflatten(1, (hq, d)), qkv[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
    mine = torch.empty_like(q_out), torch.empty_like(k_out)
    nvk().rotary_embedding(q, k, pos, torch.tensor(f, device="cuda"), query_out=mine[0], key_out=mine[1])
    for a, b in zip(mine, (q_out, k_out)):   # (each within half a step of the true value, and the step doubles where it crosses a power of two)
        assert ((a.double() - b.double()).abs() <= b.double().abs() * 2 * 2.0 ** -8 + 8 * 2.0 ** -20).all()


@pytest.mark.gpu
def test_infinities_and_nan_stay_in_their_pairs():
    import torch
    x = torch.ones(1, 1, 8, device="cuda")
    x[0, 0, 1], x[0, 0, 2] = float("inf"), float("nan")
    out = torch.empty_like(x)
    nvk().rotary_embedding(x, None, torch.tensor([3], device="cuda"), torch.tensor([1.0, 1.0, 1.0, 1.0], device="cuda"), query_out=out)
    bad = (~torch.isfinite(out[0, 0])).tolist()
    assert bad == [False, True, True, False, False, True, True, False]


@pytest.mark.gpu
@pytest.mark.parametrize("change,word", [
    (dict(key=(3, 2, 64), key_out=(3, 2, 64)), "key must have the rows"), (dict(q_out=(4, 2, 64)), "shapes"), (dict(pos=(5,)), "element for every row"), (dict(f="float64"), "float32"),
    (dict(pos="float32"), "int32 or int64"), (dict(q=(4, 4)), "must be \\[rows"), (dict(key_out=None), "together"), (dict(f=(33,)), "at most head_dim")])
def test_the_binding_refuses(change, word):
    import torch
    shapes = dict(q=(4, 4, 64), key=(4, 2, 64), pos=(4,), f=(32,), q_out=(4, 4, 64), key_out=(4, 2, 64))
    kinds = dict(pos=torch.int32)
    for name, v in change.items():
        if isinstance(v, str):
            kinds[name] = getattr(torch, v)
        else:
            shapes[name] = v
    x = {n: None if s is None else torch.zeros(s, dtype=kinds.get(n, torch.float32), device="cuda") for n, s in shapes.items()}
    if x["key_out"] is None:
        with pytest.raises(ValueError, match=word):
            nvk()._load_binding().rotary_embedding(x["q"], x["key"], x["pos"], x["f"], False, 1.0, x["q_out"], None)
        return
    with pytest.raises(ValueError, match=word):
        nvk().rotary_embedding(x["q"], x["key"], x["pos"], x["f"], query_out=x["q_out"], key_out=x["key_out"])
    with pytest.raises(ValueError, match="contiguous rows"):
        nvk().rotary_embedding(torch.zeros(4, 64, 4, device="cuda").transpose(1, 2), None, torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(32, device="cuda"))


# ---- tensors of a call that overlap ----------------------------------------------------------------------------------------------
def _at(n):
    return ctypes.c_void_p(n)


@pytest.mark.parametrize("change", [
    dict(qo=_at(1 << 22)), dict(qo=_at((1 << 22) + 512)), dict(ko=_at(1 << 20)), dict(ko=_at(1 << 24)), dict(ko=_at((1 << 24) + 6 * 1024)), dict(qo=_at(1 << 26)), dict(ko=_at((1 << 26) - 512)),
    dict(qo=_at(1 << 27)), dict(ko=_at((1 << 27) - 1024)), dict(q=_at(1 << 25), qo=_at(1 << 25)),
    # columns of one packed row: queries 0 .. 1023, keys 1024 .. 1279, of 1536
    dict(q=_at(1 << 20), k=_at((1 << 20) + 2048), qo=_at((1 << 20) + 2048), ko=_at((1 << 20) + 2048), packed=True),
    dict(q=_at(1 << 20), k=_at((1 << 20) + 2048), qo=_at(1 << 20), ko=_at((1 << 20) + 2040), packed=True),
    dict(q=_at(1 << 20), k=_at((1 << 20) + 2048), qo=_at((1 << 20) + 1040), ko=_at((1 << 20) + 2048), packed=True),
    dict(q=_at((1 << 20) + 3072), k=_at((1 << 20) + 3072 + 2048), qo=_at((1 << 20) + 3072), ko=_at((1 << 20) + 2560 + 256), packed=True)])
def test_refuses_outputs_over_other_tensors(built, change):
    """Queries' output over the keys, keys' output over the queries or their output, either over positions or frequencies, in whole or in part."""
    a = dict(q=_at(1 << 20), k=_at(1 << 22), pos=_at(1 << 26), pos_dtype=I(3), f=_at(1 << 27), factor=ctypes.c_float(1.0), rows=L(4), hq=I(8), hkv=I(2), d=I(128), rot=I(128), pairs=I(0),
             q_stride=L(1024), k_stride=L(256), qo=Q, ko=_at(1 << 25), qo_stride=L(1024), ko_stride=L(256), dtype=I(1), stream=None)
    change = dict(change)
    if change.pop("packed", False):
        a.update(dict.fromkeys(("q_stride", "k_stride", "qo_stride", "ko_stride"), L(1536)))
    a.update(change)
    rc = built.lib().nvk_rotary_embedding(*a.values())
    said = built.lib().nvk_last_error().decode()
    assert rc == 1 and "overlap" in said, said


@pytest.mark.parametrize("change", [dict(rows=L(1 << 50)), dict(q_stride=L(1 << 41)), dict(ko_stride=L(1 << 60))])
def test_refuses_rows_beyond_memory(built, change):
    a = dict(q=_at(1 << 20), k=_at(1 << 22), pos=_at(1 << 26), pos_dtype=I(3), f=_at(1 << 27), factor=ctypes.c_float(1.0), rows=L(4), hq=I(8), hkv=I(2), d=I(128), rot=I(128), pairs=I(0),
             q_stride=L(1024), k_stride=L(256), qo=Q, ko=_at(1 << 25), qo_stride=L(1024), ko_stride=L(256), dtype=I(1), stream=None)
    a.update(change)
    assert built.lib().nvk_rotary_embedding(*a.values()) == 3 and "too many rows" in built.lib().nvk_last_error().decode()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 37])
def test_outputs_beside_their_inputs_in_packed_rows(rows):
    """Other columns of the same packed rows are no overlap; nor is the queries' output in place with the keys' elsewhere."""
    import torch
    rng = np.random.default_rng(rows)
    hq, hkv, d = 4, 2, 64
    n = (hq + hkv) * d
    base = torch.from_numpy(rng.standard_normal((rows, 2 * n + 16))).to(torch.bfloat16).cuda()
    part = lambda a, heads: base[:, a:a + heads * d].unflatten(1, (heads, d))
    q, k, qo, ko = part(0, hq), part(hq * d, hkv), part(n + 8, hq), part(n + 8 + hq * d, hkv)
    pos = torch.from_numpy(rng.integers(0, 1 << 16, rows)).cuda()
    f = torch.tensor(nvk().rotary_inv_freq(d, 10000.0)[0], device="cuda")
    apart = torch.empty_like(q.contiguous()), torch.empty_like(k.contiguous())
    nvk().rotary_embedding(q, k, pos, f, query_out=apart[0], key_out=apart[1])
    kept = base.clone()
    nvk().rotary_embedding(q, k, pos, f, query_out=qo, key_out=ko)
    assert torch.equal(qo, apart[0]) and torch.equal(ko, apart[1])
    assert torch.equal(base[:, :n + 8], kept[:, :n + 8]) and torch.equal(base[:, 2 * n + 8:], kept[:, 2 * n + 8:])
    nvk().rotary_embedding(q, k, pos, f, key_out=ko)
    assert torch.equal(q, apart[0]) and torch.equal(ko, apart[1]) and torch.equal(k, kept[:, hq * d:n].unflatten(1, (hkv, d)))
    with pytest.raises(ValueError, match="overlap"):
        nvk().rotary_embedding(q, k, pos, f, query_out=q, key_out=q[:, 1:1 + hkv])


@pytest.mark.gpu
@pytest.mark.parametrize("position", [1, 2 ** 24 + 1, 2 ** 31 - 1, 2 ** 40 + 12345, -(2 ** 33) - 7, 2 ** 52 + 1, -(2 ** 53) + 1])
@pytest.mark.parametrize("pairs", [False, True])
def test_angles_far_out_are_as_exact_as_near(position, pairs):
    """The same bound at every position up to 2^53, the one of the tests above: 2^-26 of a turn for the fraction in 32 bits and what sincospi and the products add; nothing that grows with
    the position (2^53 turns to 2^-104 of themselves are off by 2^-51)."""
    import decimal

    import torch
    rng = np.random.default_rng(3)
    x = torch.from_numpy(rng.standard_normal((1, 3, 64))).float().cuda()
    f = [1.0, 0.5, 2.0 ** -7, 0.1, 1 / 3, 0.7071, 1.2345e-4, 0.9999] * 4
    fd = torch.tensor(f, dtype=torch.float32, device="cuda")
    out = torch.empty_like(x)
    nvk().rotary_embedding(x, None, torch.tensor([position], device="cuda"), fd, pairs, query_out=out)
    with decimal.localcontext() as ctx:
        ctx.prec = 100
        turn = 2 * decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")
        angle = np.array([float((decimal.Decimal(position) * decimal.Decimal(v)).remainder_near(turn)) for v in fd.double().tolist()])
    c, s = np.cos(angle), np.sin(angle)
    y = x.double().cpu().numpy()
    a, b = (y[..., 0::2], y[..., 1::2]) if pairs else (y[..., :32], y[..., 32:])
    first, second = a * c - b * s, b * c + a * s
    want = np.stack([first, second], -1).reshape(y.shape) if pairs else np.concatenate([first, second], -1)
    assert (np.abs(out.double().cpu().numpy() - want) <= _tolerance(want, np.abs(y).max(), 1.0, "float32")).all()
