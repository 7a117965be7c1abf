"""The 4-bit pool and the rotation by axes without a GPU: the oracle's codes and angles, what
the C ABI, the pool and the rotary refuse before any device work."""

from __future__ import annotations

import math

import pytest
import torch

from infrared_amd import _lib, kernels, Quant4PagedKVPool, rotary, RotaryAxes
from oracle import quant4

P = 256  # an aligned address that is never used


def test_oracle_rounds_to_the_nearest_code_and_ties_to_the_even_one():
    y = torch.tensor([0.25, 0.26, 0.75, 0.74, 1.25, 1.75, 2.5, 2.51, 3.5, 5.0, 5.01, 7.0, 0.0]).double()
    want = torch.tensor([0.0, 0.5, 1.0, 0.5, 1.0, 2.0, 2.0, 3.0, 4.0, 4.0, 6.0, 6.0, 0.0]).double()
    assert torch.equal(quant4.round_code(y), want) and torch.equal(quant4.round_code(-y), -want)


def test_scale_is_the_least_that_holds_the_largest_magnitude():
    for amax, k in ((7.0, 0), (7.0000005, 1), (3.5, -1), (3.51, 0), (1.0, -2), (0.0, -100)):
        assert quant4.scale_exponent(amax, torch.float32) == k, amax
        x = torch.zeros(1, 64).double()
        x[0, 40] = -amax
        assert quant4.exponents(x, torch.float32).tolist() == [[-100, k]]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_every_value_is_a_number_of_the_dtype_and_is_held_as_it_is(dtype):
    lo, hi = quant4.BOUNDS[dtype]
    codes = torch.tensor(quant4.CODES).double().repeat(4)
    for k in range(lo, hi + 1):
        v = codes * 2.0**k
        assert torch.equal(v.to(dtype).double(), v), k
        assert torch.equal(quant4.quantise(v, dtype), v), k


def test_oracle_angles_are_those_of_far_positions():
    for p, f in ((3, 0.7), (10**6, 1.0), (-(10**6), 0.1), (2**40, 1e-3)):
        a = quant4._angle(p, f)
        # (a double's product is off by up to 2^-53 of it, and so is its reduction)
        assert abs(a) <= math.pi and abs(math.remainder(p * f - a, 2 * math.pi)) <= 2.0**-51 * abs(p * f) + 1e-15


def test_steps_are_the_frequencies_turns():
    assert abs(float(rotary._TWO_PI) - 2 * math.pi) <= 2.0**-51
    for f in (1.0, 1e-6, 0.37, 100.0, -0.5, 0.0):
        step = rotary._step(f)
        assert 0 <= step < 2**64
        for p in (1, 12345, -7, 10**9):
            turn = (p * step) % 2**64 / 2**64
            off = (turn * 2 * math.pi - quant4._angle(p, f)) % (2 * math.pi)
            assert min(off, 2 * math.pi - off) <= 2 * math.pi * abs(p) * 2.0**-64 + 1e-14, (f, p)


def test_pool_refuses_what_it_has_no_kernel_for():
    for bs in (0, 8, 24, 2048):
        with pytest.raises(ValueError, match="4-bit pool's block size"):
            Quant4PagedKVPool(1, 4, bs, 2, 64, torch.bfloat16)
    with pytest.raises(ValueError, match="head_dim"):
        Quant4PagedKVPool(1, 4, 16, 2, 96, torch.bfloat16)
    with pytest.raises(ValueError, match="2\\^31"):
        Quant4PagedKVPool(1, 1 << 27, 16, 2, 64, torch.bfloat16)
    with pytest.raises(RuntimeError, match="dtype"):
        Quant4PagedKVPool(1, 4, 16, 2, 64, torch.int8)
    with pytest.raises(RuntimeError, match="ROCm device"):
        Quant4PagedKVPool(1, 4, 16, 2, 64, torch.bfloat16, device="cpu")


@pytest.mark.parametrize("freq, axis, text", [
    ([], [], "one of each"), ([1.0] * 8, [0] * 7, "one of each"), ([1.0] * 5, [0] * 5, "multiple of 16"),
    ([1.0] * 136, [0] * 136, "up to 256"), ([1.0] * 7 + [float("nan")], [0] * 8, "finite"),
    ([1.0] * 8, [0] * 7 + [8], "axes must be"), ([1.0] * 8, [-1] * 8, "axes must be"),
])
def test_rotary_refusals(freq, axis, text):
    with pytest.raises(ValueError, match=text):
        RotaryAxes(freq, axis)


def test_rotary_arrangements_refuse_what_does_not_fit():
    with pytest.raises(ValueError, match="finite"):
        RotaryAxes([1.0] * 8, [0] * 8, scaling=float("inf"))
    with pytest.raises(ValueError, match="sections"):
        RotaryAxes.sections(128, (16, 24, 25))
    with pytest.raises(ValueError, match="share"):
        RotaryAxes.grid(64, 3)
    with pytest.raises(RuntimeError, match="ROCm device"):
        RotaryAxes([1.0] * 8, [0] * 8, device="cpu")


def _scatter(**kw):
    a = dict(k=P, kt=256, kh=128, v=P, vt=256, vh=128, kc=P, vc=P, sc=P, nb=4, bs=16, slots=P, n=3, h=2, d=128, dt=2)
    a.update(kw)
    return _lib.lib().ir_kv_scatter_q4(*a.values(), None, None)


@pytest.mark.parametrize("kw, code, text", [
    ({"dt": 4}, -1, b"dtype"), ({"n": -1}, -1, b"bad sizes"), ({"bs": 24}, -1, b"block size"),
    ({"bs": 2048}, -1, b"block size"), ({"bs": 0}, -1, b"block size"), ({"d": 96}, -2, b"head_dim"),
    ({"nb": 1 << 28}, -1, b"2^31"), ({"nb": 1 << 60}, -1, b"2^31"), ({"sc": None}, -1, b"null"),
    ({"k": None}, -1, b"null"), ({"slots": None}, -1, b"null"), ({"k": P + 8}, -1, b"aligned"),
    ({"kc": P + 8}, -1, b"aligned"), ({"sc": P + 8}, -1, b"aligned"), ({"kt": 257}, -1, b"strides"),
    ({"h": 0}, -1, b"bad sizes"), ({"n": 1 << 31}, -1, b"too many"),
])
def test_scatter_refusals(kw, code, text):
    assert _scatter(**kw) == code
    assert text in _lib.lib().ir_last_error()


def test_scatter_of_nothing():
    assert _scatter(n=0, k=None, slots=None) == 0


def _rope(**kw):
    a = dict(q=P, qt=512, qh=128, qo=P, qot=512, qoh=128, k=P, kt=256, kh=128, v=P, vt=256, vh=128, wq=P, wk=P,
             eps=1e-6, cos=P, sin=P, cs=128, kc=P, vc=P, sc=P, nb=4, bs=16, slots=P, n=3, hq=4, h=2, d=128, dt=2, qdt=2)
    a.update(kw)
    return _lib.lib().ir_rope_kv_scatter_q4(*a.values(), None, None)


@pytest.mark.parametrize("kw, code, text", [
    ({"dt": 9}, -1, b"dtype"), ({"qdt": 1}, -1, b"q_out_dtype"), ({"wq": None}, -1, b"norm weight"),
    ({"eps": -1.0}, -1, b"eps"), ({"cos": None}, -1, b"null"), ({"cs": 3}, -1, b"cos/sin"), ({"q": None}, -1, b"null"),
    ({"d": 80}, -2, b"head_dim"), ({"qoh": 129}, -1, b"strides"), ({"wk": P + 4}, -1, b"aligned"),
])
def test_rope_refusals(kw, code, text):
    assert _rope(**kw) == code
    assert text in _lib.lib().ir_last_error()


def _axes(fn, **kw):
    a = dict(q=P, qt=512, qh=128, qo=P, qot=512, qoh=128, k=P, kt=256, kh=128)
    if fn == "rows":
        a |= dict(ko=P, kot=256, koh=128)
    else:
        a |= dict(v=P, vt=256, vh=128)
    a |= dict(wq=P, wk=P, eps=1e-6, pos=P, pt=3, na=3, pairs=P, scaling=1.0)
    if fn == "cache":
        a |= dict(kc=P, vc=P, cst=128, csh=8192, ns=64, slots=P)
    if fn == "q4":
        a |= dict(kc=P, vc=P, sc=P, nb=4, bs=16, slots=P)
    a |= dict(n=3, hq=4, h=2, d=128, dt=2, qdt=2)
    a.update(kw)
    tail = (None,) if fn == "rows" else (None, None)
    name = {"rows": "ir_rope_axes", "cache": "ir_rope_axes_kv_scatter", "q4": "ir_rope_axes_kv_scatter_q4"}[fn]
    return getattr(_lib.lib(), name)(*a.values(), *tail)


@pytest.mark.parametrize("fn", ["rows", "cache", "q4"])
@pytest.mark.parametrize("kw, code, text", [
    ({"dt": 5}, -1, b"dtype"), ({"qdt": 1}, -1, b"q_out_dtype"), ({"na": 0}, -1, b"axes"), ({"na": 9}, -1, b"axes"),
    ({"pos": None}, -1, b"null"), ({"pairs": None}, -1, b"null"), ({"pairs": P + 8}, -1, b"aligned"),
    ({"pos": P + 4}, -1, b"aligned"), ({"scaling": float("inf")}, -1, b"scaling"), ({"wk": None}, -1, b"norm weight"),
    ({"eps": -1.0}, -1, b"eps"), ({"q": None}, -1, b"null"), ({"k": None}, -1, b"null"), ({"d": 40}, -2, b"head_dim"),
    ({"d": 80}, -2, b"head_dim"), ({"qt": 511}, -1, b"strides"), ({"n": -1}, -1, b"bad sizes"),
    ({"q": P + 8}, -1, b"aligned"), ({"n": 1 << 33}, -1, b"too many"),
])
def test_rope_axes_refusals(fn, kw, code, text):
    assert _axes(fn, **kw) == code
    assert text in _lib.lib().ir_last_error()


def test_rope_axes_of_nothing():
    assert _axes("rows", n=0, q=None) == 0 and _axes("cache", n=0, q=None) == 0 and _axes("q4", n=0, q=None) == 0
    assert _axes("rows", hq=0, h=0, q=None, k=None) == 0


@pytest.mark.parametrize("fn, kw, text", [
    ("rows", {"d": 272, "wq": None, "wk": None}, b"head_dim"), ("rows", {"ko": P + 8}, b"k_out"),
    ("rows", {"koh": 4}, b"k_out"), ("cache", {"kc": None}, b"null"), ("cache", {"csh": 4}, b"caches"),
    ("cache", {"slots": None}, b"null"), ("q4", {"sc": None}, b"null"), ("q4", {"bs": 24}, b"block size"),
    ("cache", {"v": None}, b"null"),
])
def test_rope_axes_refusals_of_one_form(fn, kw, text):
    assert _axes(fn, **kw) < 0
    assert text in _lib.lib().ir_last_error()


def _attend(fn, **kw):
    lib = _lib.lib()
    if fn == "decode":
        a = dict(q=P, qs=512, qh=128, kc=P, vc=P, sc=P, nb=4, bs=16, bt=P, bts=4, mb=4, ctx=P, out=P, os=512, oh=128,
                 b=1, hq=4, h=2, d=128, scale=0.1, dt=2, qdt=2, part=0, ctr=P, nctr=64, ws=P, wsb=1 << 20)
        a.update(kw)
        return lib.ir_paged_decode_q4(*a.values(), None, None)
    if fn == "planned":
        a = dict(q=P, qs=512, qh=128, kc=P, vc=P, sc=P, out=P, os=512, oh=128, b=1, hq=4, h=2, d=128, mb=4, bs=16,
                 scale=0.1, dt=2, qdt=2, flags=0, plan=P, ctr=P, nctr=64, ws=P, wsb=1 << 30)
        a.update(kw)
        return lib.ir_paged_decode_planned_q4(*a.values(), None, None)
    a = dict(q=P, qs=512, qh=128, kc=P, vc=P, sc=P, nb=4, bs=16, bt=P, bts=4, mb=4, cu=P, qst=P, b=1, n=3, mq=3, out=P,
             os=512, oh=128, hq=4, h=2, d=128, scale=0.1, dt=2, qdt=2, plan=None, planb=0)
    a.update(kw)
    return lib.ir_paged_prefill_q4(*a.values(), None, None)


@pytest.mark.parametrize("fn", ["decode", "planned", "prefill"])
@pytest.mark.parametrize("kw, text", [
    ({"sc": None}, b"null"), ({"sc": P + 8}, b"aligned"), ({"q": None}, b"null"), ({"dt": 4}, b"dtype"),
    ({"qdt": 1}, b"q_dtype"), ({"d": 96}, b"head_dim"), ({"bs": 24}, b""), ({"kc": P + 8}, b"aligned"),
    ({"qh": 65}, b"strides"), ({"hq": 5}, b""),
])
def test_attention_refusals(fn, kw, text):
    assert _attend(fn, **kw) < 0
    assert text in _lib.lib().ir_last_error()


@pytest.mark.parametrize("fn", ["decode", "planned", "prefill"])
@pytest.mark.parametrize("scale", [float("nan"), float("inf")])
def test_attention_refuses_a_scale_that_is_no_number(fn, scale):
    assert _attend(fn, scale=scale) < 0
    assert b"scale" in _lib.lib().ir_last_error()


def test_tables_of_few_keys_are_not_planned():
    assert not kernels.decode_plan_pays(512, 28, 4, 64, 16, bits=4)


def test_decode_plan_takes_the_4_bit_layers_strides():
    lib = _lib.lib()
    args = dict(bt=P, bts=4, mb=4, ctx=P, b=1, hq=4, h=2, bs=16, nb=4, cs=64, ch=64 * 64, dt=4, flags=0, plan=None,
                pb=0)
    assert lib.ir_paged_decode_plan(*args.values(), None, None) == -1 and b"plan of" in lib.ir_last_error()
    args["dt"] = 5
    assert lib.ir_paged_decode_plan(*args.values(), None, None) == -1 and b"dtype" in lib.ir_last_error()
