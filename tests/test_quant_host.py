"""The 8-bit pool without a GPU: the oracle's codes against torch's e4m3 type, and what
the C ABI and the pool refuse before any device work."""

from __future__ import annotations

import pytest
import torch

from infrared_amd import QuantPagedKVPool, _lib
from oracle import quant

P = 256  # an aligned address that is never used


def test_oracle_rounds_as_the_e4m3_type_does():
    """Every fp16 number within the codes' range, at scale 1, and the codes themselves."""
    x = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(torch.float16)
    x = x[torch.isfinite(x) & (x.abs() <= 448)]
    want = x.float().to(torch.float8_e4m3fn).double()
    assert torch.equal(quant.round_code(x.double(), 0, torch.bfloat16), want)
    assert torch.equal(quant.round_code(want * 2.0**-30, -30, torch.bfloat16), want * 2.0**-30)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_every_value_is_a_number_of_the_dtype(dtype):
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    codes = codes[torch.isfinite(codes)]
    lo, hi, most = quant.BOUNDS[dtype]
    for k in range(lo, hi + 1):
        v = codes * 2.0**k
        v = v[v.abs() <= most]
        assert torch.equal(v.to(dtype).double(), v), k


def test_scale_is_the_least_that_holds_the_largest_magnitude():
    for amax, k in ((448.0, 0), (449.0, 1), (224.0, -1), (1.75, -8), (1.7500001, -7), (0.0, -100)):
        assert quant.scale_exponent(amax, torch.float32) == k, amax


def test_pool_refuses_what_it_has_no_kernel_for():
    for bs in (0, 8, 24, 2048):
        with pytest.raises(ValueError, match="block size"):
            QuantPagedKVPool(1, 4, bs, 2, 64, torch.bfloat16)
    with pytest.raises(ValueError, match="head_dim"):
        QuantPagedKVPool(1, 4, 16, 2, 96, torch.bfloat16)
    with pytest.raises(ValueError, match="2\\^31"):
        QuantPagedKVPool(1, 1 << 27, 16, 2, 64, torch.bfloat16)
    with pytest.raises(RuntimeError, match="dtype"):
        QuantPagedKVPool(1, 4, 16, 2, 64, torch.int8)
    with pytest.raises(RuntimeError, match="ROCm device"):
        QuantPagedKVPool(1, 4, 16, 2, 64, torch.bfloat16, device="cpu")


def _scatter(**kw):
    a = dict(k=P, kt=256, kh=128, v=P, vt=256, vh=128, kc=P, vc=P, sc=P, nb=4, bs=16, slots=P, n=3, h=2, d=128, dt=2)
    a.update(kw)
    return _lib.lib().ir_kv_scatter_q8(*a.values(), None, None)


@pytest.mark.parametrize("kw, code, text", [
    ({"dt": 3}, -1, b"dtype"), ({"n": -1}, -1, b"bad sizes"), ({"bs": 24}, -1, b"block size"),
    ({"bs": 2048}, -1, b"block size"), ({"bs": 0}, -1, b"block size"), ({"d": 96}, -2, b"head_dim"),
    ({"nb": 1 << 28}, -1, b"2^31"), ({"sc": None}, -1, b"null"), ({"k": None}, -1, b"null"),
    ({"slots": None}, -1, b"null"),
    ({"k": P + 8}, -1, b"aligned"), ({"kc": P + 8}, -1, b"aligned"), ({"sc": P + 4}, -1, b"aligned"),
    ({"kt": 257}, -1, b"strides"), ({"h": 0}, -1, b"bad sizes"), ({"n": 1 << 31}, -1, b"too many"),
])
def test_scatter_refusals(kw, code, text):
    assert _scatter(**kw) == code
    assert text in _lib.lib().ir_last_error()


def test_scatter_of_nothing():
    assert _scatter(n=0, k=None, slots=None) == 0


def _rope(fn, q8, **kw):
    a = dict(q=P, qt=512, qh=128, qo=P, qot=512, qoh=128, k=P, kt=256, kh=128, v=P, vt=256, vh=128, wq=P, wk=P,
             eps=1e-6, cos=P, sin=P, cs=128, kc=P, vc=P)
    a.update(dict(sc=P, nb=4, bs=16) if q8 else dict(cst=128, csh=8192, ns=64))
    a.update(slots=P, n=3, hq=4, h=2, d=128, dt=2)
    if q8:
        a.update(qdt=2)
    a.update(kw)
    return getattr(_lib.lib(), fn)(*a.values(), None, None)


@pytest.mark.parametrize("fn, q8", [("ir_qk_norm_rope_kv_scatter", False), ("ir_rope_kv_scatter_q8", True)])
@pytest.mark.parametrize("kw, code, text", [
    ({"dt": 7}, -1, b"dtype"), ({"d": 256}, -2, b"head_dim"), ({"wk": None}, -1, b"weight"),
    ({"wq": P + 8, "wk": P}, -1, b"aligned"), ({"eps": -1.0}, -1, b"eps"), ({"cs": 130}, -1, b"stride"),
    ({"qt": 514}, -1, b"strides"), ({"cos": None}, -1, b"null"), ({"q": None}, -1, b"null"),
    ({"kc": None}, -1, b"null"), ({"n": -1}, -1, b"bad sizes"),
])
def test_norm_rope_refusals(fn, q8, kw, code, text):
    assert _rope(fn, q8, **kw) == code
    assert text in _lib.lib().ir_last_error()


def test_norm_rope_needs_weights_where_it_norms():
    assert _rope("ir_qk_norm_rope_kv_scatter", False, wq=None, wk=None) == -1
    assert b"null" in _lib.lib().ir_last_error()
    assert _rope("ir_qk_norm_rope_kv_scatter", False, n=0) == 0
    assert _rope("ir_rope_kv_scatter_q8", True, n=0) == 0


def test_queries_leave_the_rotation_in_the_dtype_or_fp32():
    assert _rope("ir_rope_kv_scatter_q8", True, qdt=1) == -1
    assert b"q_out_dtype" in _lib.lib().ir_last_error()
    assert _rope("ir_rope_kv_scatter_q8", True, qdt=0, qot=514) == -1  # (fp32's strides)
    assert b"strides" in _lib.lib().ir_last_error()


def test_read_refusals():
    lib = _lib.lib()
    ok = (P, P, P, 4, 16, P, 3, 2, 128, 2, P, P, None, None)
    for at, x, code, text in ((9, 3, -1, b"dtype"), (8, 32, -2, b"head_dim"), (4, 17, -1, b"block size"),
                              (6, -1, -1, b"bad sizes"), (5, None, -1, b"null"), (10, P + 4, -1, b"aligned")):
        assert lib.ir_gather_slots_q8(*ok[:at], x, *ok[at + 1 :]) == code and text in lib.ir_last_error(), at
    assert lib.ir_gather_slots_q8(P, P, P, 4, 16, None, 0, 2, 128, 2, None, None, None, None) == 0
    assert lib.ir_paged_gather_q8(P, P, P, 4, 16, None, 4, 4, None, 2, 64, 2, 128, 2, P, P, None, None) == -1
    assert b"null" in lib.ir_last_error()


def test_attention_refusals():
    lib = _lib.lib()
    # scales missing, a block size that is no multiple of 16, scales off their alignment
    dec = [P, 512, 128, P, P, P, 4, 16, P, 4, 4, P, P, 512, 128, 2, 4, 2, 128, 1.0, 2, 2, 0, P, 64, P, 1 << 30, None,
           None]
    for at, x, text in ((5, None, b"null"), (7, 24, b"block size"), (5, P + 4, b"aligned"), (20, 3, b"dtype"),
                        (21, 1, b"q_dtype"), (0, P + 8, b"aligned")):
        a = dec[:at] + [x] + dec[at + 1 :]
        assert lib.ir_paged_decode_q8(*a) == -1 and text in lib.ir_last_error(), at
    pre = [P, 512, 128, P, P, P, 4, 16, P, 4, 4, P, P, 2, 8, 8, P, 512, 128, 4, 2, 128, 1.0, 2, 2, None, 0, None, None]
    for at, x, text in ((5, None, b"null"), (7, 24, b"block size"), (5, P + 4, b"aligned"), (23, 3, b"dtype"),
                        (24, 1, b"q_dtype"), (1, 514, b"strides")):
        a = pre[:at] + [x] + pre[at + 1 :]
        assert lib.ir_paged_prefill_q8(*a) == -1 and text in lib.ir_last_error(), at
    plan = [P, 512, 128, P, P, P, P, 512, 128, 2, 4, 2, 128, 4, 16, 1.0, 2, 2, 0, P, P, 64, P, 1 << 30, None, None]
    for at, x, text in ((5, None, b"null"), (5, P + 4, b"aligned"), (16, 3, b"dtype"), (14, 24, b"plannable"),
                        (17, 1, b"q_dtype")):
        a = plan[:at] + [x] + plan[at + 1 :]
        assert lib.ir_paged_decode_planned_q8(*a) == -1 and text in lib.ir_last_error(), at
