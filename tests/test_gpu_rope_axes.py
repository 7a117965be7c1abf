"""Rotation by positions with several axes on the GPU against the formula in 64 bits, with
and without norms, of rows and into every kind of pool, alone and as a step uses it."""

from __future__ import annotations

import pytest
import torch

from infrared_amd import (
    PagedKVPool,
    Quant4PagedKVPool,
    QuantPagedKVPool,
    RotaryAxes,
    kernels,
    metadata,
    paged_attention,
    rope_axes_paged_attention,
)
from oracle import quant4
from test_gpu_quant import gen, rows

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
DEV = "cuda"


def positions(g, axes, n, most=70000):
    return torch.randint(0, most, (axes, n), generator=g, device=DEV)


# With m = |a| + |b| over a pair: the angle as an fp32 number of half turns is off by at
# most 2^-24 of it, pi * 2^-24 radians at most; sine and cosine of it by two steps, 2^-23;
# scaling, two products and the sum by half a step each: (pi + 2 + 2.5) 2^-24 m, 8 * 2^-24 m
# with the integer step's 2^-32. A norm before adds (d / 4 + 8) 2^-24 (test_gpu_quant.py has
# its derivation). Then half a step of the dtype.


def tolerance(x, o, dtype, w=None, eps=0.0, scaling=1.0, stored=True):
    x = x.cpu().double()
    d = x.shape[-1]
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.cpu().double()
    a, b = x.abs().chunk(2, dim=-1)
    m = torch.cat([a + b, a + b], -1) * abs(scaling)
    f = torch.finfo(dtype)
    half = torch.maximum(f.eps / 2 * o.abs(), torch.tensor(f.smallest_normal * f.eps / 2, dtype=torch.float64))
    return (8 + (d / 4 + 8 if w is not None else 0)) * 2.0**-24 * m + (half if stored else 0)


def check(got, x, pos, rotary, w=None, eps=0.0, dtype=None):
    o = quant4.turn(x, pos, rotary.inv_freq, rotary.axis_of, w, eps, rotary.scaling)
    tol = tolerance(x, o, dtype or got.dtype, w, eps, rotary.scaling)
    err = (got.double().cpu() - o).abs()
    assert (err <= tol).all(), (err / tol).max()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [16, 48, 64, 80, 96, 128, 240, 256])
@pytest.mark.parametrize("n, hq, h", [(1, 3, 1), (5, 16, 16), (133, 1, 4)])
def test_rows_of_any_width(dtype, d, n, hq, h):
    g = gen(d + n)
    rotary = RotaryAxes.grid(d, 2, 1e4)
    qk = rows(g, n, hq + h, d, dtype)
    q, k = qk.split([hq, h], 1)
    pos = positions(g, 2, n, 300)
    qo, ko = kernels.rope_axes(q, k, pos, rotary)
    check(qo, q, pos, rotary)
    check(ko, k, pos, rotary)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d, sections", [(128, (16, 24, 24)), (64, (8, 12, 12)), (64, (32,)), (128, (1, 30, 32, 1))])
@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("n", [1, 37, 2100])
def test_rows_and_16_bit_pools(dtype, d, sections, normed, n):
    """The three outputs of the fused write, rows of the call without a cache, fp32 queries."""
    hq, h, bs = 6, 2, 16
    g = gen(n + d)
    rotary = RotaryAxes.sections(d, sections, scaling=1.0 if n == 1 else 0.83)
    q, k, v = rows(g, n, hq + 2 * h, d, dtype).split([hq, h, h], 1)
    w = (1 + 0.3 * torch.randn(2, d, generator=g, device=DEV)).to(dtype) if normed else (None, None)
    pos = positions(g, len(sections), n)
    some = slice(0, 60)  # (the oracle's cost)
    for layout in ("head_major", "slot_major"):
        pool = PagedKVPool(1, n // bs + 3, bs, h, d, dtype, layout=layout)
        slots = torch.randperm(pool.num_slots, generator=g, device=DEV)[:n]
        before = pool.k.clone()
        qo = kernels.rope_axes_kv_scatter(q, k, v, pos, rotary, pool.k[0], pool.v[0], slots, *w, 1e-5)
        check(qo[some], q[some], pos[:, some], rotary, w[0], 1e-5)
        check(pool.k[0, slots[some]], k[some], pos[:, some], rotary, w[1], 1e-5)
        assert torch.equal(pool.v[0, slots], v)
        rest = torch.ones(pool.num_slots, dtype=torch.bool, device=DEV)
        rest[slots] = False
        assert torch.equal(pool.k[0][rest], before[0][rest]) and not pool.v[0][rest].any()
        q2, k2 = kernels.rope_axes(q, k, pos, rotary, *w, 1e-5)
        assert torch.equal(q2, qo) and torch.equal(k2, pool.k[0, slots])
        q3, _ = kernels.rope_axes(q, k, pos, rotary, *w, 1e-5, q_out=torch.empty(n, hq, d, device=DEV))
        assert torch.equal(q3.to(dtype), qo)


@pytest.mark.parametrize("d, normed", [(80, False), (64, True)])
def test_in_place_and_strided(d, normed):
    g, n, dtype = gen(3), 50, torch.float16
    rotary = RotaryAxes.grid(d, 2)
    wide = rows(g, n, 20, d, dtype)
    q, k = wide[:, 3:9], wide[:, 11:13]
    w = (1 + 0.3 * torch.randn(2, d, generator=g, device=DEV)).to(dtype) if normed else (None, None)
    pos = torch.randint(-500, 500, (n, 2), generator=g, device=DEV).T  # (columns of a [tokens, axes] tensor)
    want = kernels.rope_axes(q.contiguous(), k.contiguous(), pos.contiguous(), rotary, *w)
    untouched = wide.clone()
    got = kernels.rope_axes(q, k, pos, rotary, *w, q_out=q, k_out=k)
    assert torch.equal(got[0], want[0]) and torch.equal(q, want[0]) and torch.equal(k, want[1])
    for a in (slice(0, 3), slice(9, 11), slice(13, 20)):
        assert torch.equal(wide[:, a], untouched[:, a])


def test_far_positions():
    """Positions whose angle an fp32 product would lose, negative ones, and the largest there are."""
    d, n = 64, 12
    g = gen(4)
    freq = [1.0, 0.999, 0.3, 1e-3, 1e-6, 2.5, -0.7, 0.0] * 4
    rotary = RotaryAxes(freq, [0, 1] * 16)
    x = torch.randn(n, 2, d, generator=g, device=DEV)
    pos = torch.tensor([0, 1, -1, 1000003, -(2**31), 2**31 - 1, 2**40 + 12345, -(2**45), 2**24 + 1, 7, 2**33, 99999],
                       device=DEV)
    pos = torch.stack([pos, pos.flip(0)])
    qo, ko = kernels.rope_axes(x, x[:, :1], pos, rotary)
    o = quant4.turn(x, pos, freq, rotary.axis_of)
    # the integer step: up to position * 2^-65 turns
    most = pos.abs().amax(0).double().cpu()[:, None, None] * 2.0**-64 * 3.15
    a, b = x.cpu().double().abs().chunk(2, -1)
    tol = tolerance(x, o, torch.float32) + most * torch.cat([a + b, a + b], -1)
    assert ((qo.double().cpu() - o).abs() <= tol).all() and torch.equal(ko, qo[:, :1])


def test_one_axis_is_the_usual_rotation():
    """Equal positions: the rotation of ``rope_kv_scatter`` up to its roundings (fp32: its
    products and their sum are rounded, and its cos and sin)."""
    d, n, hq, h = 128, 40, 4, 2
    g = gen(5)
    q, k, v = rows(g, n, hq + 2 * h, d, torch.float32).split([hq, h, h], 1)
    pos = torch.arange(100, 100 + n, device=DEV)
    rotary = RotaryAxes.sections(d, (16, 24, 24))
    pools = [PagedKVPool(1, 4, 16, h, d, torch.float32) for _ in range(3)]
    slots = torch.arange(n, device=DEV)
    angle = pos.double()[:, None] * torch.tensor(rotary.inv_freq, dtype=torch.float64, device=DEV)
    cos, sin = (torch.cat([t, t], 1).float() for t in (angle.cos(), angle.sin()))
    want = kernels.rope_kv_scatter(q, k, v, cos, sin, pools[0].k[0], pools[0].v[0], slots)
    got = kernels.rope_axes_kv_scatter(q, k, v, pos.expand(3, n), rotary, pools[1].k[0], pools[1].v[0], slots)
    one = RotaryAxes.sections(d, (64,))
    flat = kernels.rope_axes_kv_scatter(q, k, v, pos, one, pools[2].k[0], pools[2].v[0], slots)
    assert torch.equal(got, flat) and torch.equal(pools[1].k, pools[2].k)
    tol = 2 * tolerance(q, want.double().cpu(), torch.float32)
    assert ((got - want).double().cpu().abs() <= tol).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d, normed", [(128, True), (64, False), (64, True)])
def test_into_the_4_bit_pool(dtype, d, normed):
    """Keys to the code nearest the number in 64 bits, or the next where that lies within the
    fp32 error of the border; queries as the call without a cache gives them."""
    hq, h, bs, n = 6, 2, 16, 45
    g = gen(6)
    rotary = RotaryAxes.sections(d, (d // 8, d // 8, d // 4))
    q, k, v = rows(g, n, hq + 2 * h, d, dtype).split([hq, h, h], 1)
    w = (1 + 0.3 * torch.randn(2, d, generator=g, device=DEV)).to(dtype) if normed else (None, None)
    pos = positions(g, 3, n)
    pool, want = Quant4PagedKVPool(1, 4, bs, h, d, dtype), quant4.Quant4Cache(4 * bs, h, d, dtype)
    slots = torch.randperm(4 * bs, generator=g, device=DEV)[:n]
    slots[4] = -1
    qo = kernels.rope_axes_kv_scatter(q, k, v, pos, rotary, pool.k[0], pool.v[0], slots, *w, 1e-6,
                                      err_flags=pool.err_flags, kv_scales=pool.kv_scales[0], block_size=bs)
    pool.check_errors()
    assert torch.equal(qo, kernels.rope_axes(q, k, pos, rotary, *w, 1e-6)[0])
    o = quant4.turn(k, pos, rotary.inv_freq, rotary.axis_of, w[1], 1e-6)
    want.write(o, v, slots)
    gk, gv = (t.double().cpu() for t in pool.gather(0, torch.arange(4 * bs, device=DEV)))
    assert torch.equal(gv, want.values[1])
    at = slots.cpu()
    at, o, x = at[at >= 0], o[at >= 0], k.cpu()[at >= 0]
    tol = tolerance(x, o, dtype, w[1], 1e-6, stored=False)
    e = quant4.exponents(o, dtype).double().repeat_interleave(32, -1)
    size = torch.frexp((o.abs() * torch.exp2(-e)).clamp(1.0, 6.0))[1].double() - 1
    assert ((gk[at] - o).abs() <= torch.exp2(e + size - 2) + tol).all()
    assert (gk[at] != want.values[0, at]).double().mean() < 1e-3
    rest = torch.ones(4 * bs, dtype=torch.bool)
    rest[at] = False
    assert not gk[rest].any()


@pytest.mark.parametrize("kind", [PagedKVPool, QuantPagedKVPool, Quant4PagedKVPool])
@pytest.mark.parametrize("normed", [False, True])
def test_seam_rotates_writes_and_attends_as_its_parts_do(kind, normed):
    """A mixed step and a decode step over each kind of pool."""
    hq, h, d, bs, dtype = 8, 2, 64, 16, torch.bfloat16
    g = gen(7)
    rotary = RotaryAxes.sections(d, (8, 12, 12))
    w = (1 + 0.3 * torch.randn(2, d, generator=g, device=DEV)).to(dtype)
    norms = {"q_norm": w[0], "k_norm": w[1], "eps": 1e-5} if normed else {}
    pools = [kind(1, 12, bs, h, d, dtype) for _ in range(2)]
    tables = [[3, 1, 5], [0, 2, 4], [9, 8, 7]]
    for cached, new in (([0, 0, 0], [20, 33, 1]), ([20, 33, 1], [1, 5, 1]), ([21, 38, 2], [1, 1, 1])):
        total = sum(new)
        decode = max(new) == 1
        b, sq = (total, 1) if decode else (1, total)
        q, k, v = rows(g, total, hq + 2 * h, d, dtype).view(b, sq, hq + 2 * h, d).split([hq, h, h], 2)
        pos = positions(g, 3, total).view(3, b, sq)
        got = []
        for pool, whole in zip(pools, (True, False)):
            paged, mask = (metadata.decode_context(pool, tables, cached) if decode
                           else metadata.prefill_context(pool, tables, cached, new))
            if whole:
                got.append(rope_axes_paged_attention(q, k, v, pos, rotary, paged, mask, 0, d**-0.5, hq // h, **norms))
                continue
            args = (q.reshape(-1, hq, d), k.reshape(-1, h, d), pos.view(3, -1), rotary,
                    *((w[0], w[1], 1e-5) if normed else ()))
            if kind is PagedKVPool:
                qr, kr = kernels.rope_axes(*args)
                got.append(paged_attention(qr.view(b, sq, hq, d), kr.view(b, sq, h, d), v, paged, mask, 0, d**-0.5,
                                           hq // h))
                continue
            wide = torch.empty(total, hq, d, device=DEV)
            if kind is QuantPagedKVPool:
                _, kr = kernels.rope_axes(*args, q_out=wide)
                pool.write(0, kr, v.reshape(-1, h, d), paged.write_slots)
            else:
                kernels.rope_axes_kv_scatter(*args[:2], v.reshape(-1, h, d), *args[2:4], pool.k[0], pool.v[0],
                                             paged.write_slots, *args[4:6], eps=1e-5, q_out=wide,
                                             kv_scales=pool.kv_scales[0], block_size=bs)
            from infrared_amd.paged_attention import _attend

            got.append(_attend(wide.view(b, sq, hq, d), paged, mask, 0, d**-0.5))
        assert got[0].dtype == dtype and torch.equal(got[0], got[1])
        pools[0].check_errors()
    for name in ("k", "v", "kv_scales"):
        if hasattr(pools[0], name):
            assert torch.equal(getattr(pools[0], name).view(torch.uint8), getattr(pools[1], name).view(torch.uint8))


def test_replayed_graph_and_another_stream():
    hq, h, d, bs, n, dtype = 6, 2, 128, 16, 33, torch.bfloat16
    g = gen(8)
    rotary = RotaryAxes.sections(d, (16, 24, 24))
    w = torch.ones(d, device=DEV, dtype=dtype)
    slots = torch.arange(n, device=DEV)
    x, pos = rows(g, n, hq + 2 * h, d, dtype), positions(g, 3, n)

    def step(x, pos, plain, four):
        q, k, v = x.split([hq, h, h], 1)
        a = kernels.rope_axes_kv_scatter(q, k, v, pos, rotary, plain.k[0], plain.v[0], slots, w, w)
        b = kernels.rope_axes_kv_scatter(q, k, v, pos, rotary, four.k[0], four.v[0], slots,
                                         kv_scales=four.kv_scales[0], block_size=bs)
        return a, b, *kernels.rope_axes(q, k, pos, rotary), *four.gather(0, slots), plain.k, plain.v

    def pools():
        return PagedKVPool(1, 3, bs, h, d, dtype), Quant4PagedKVPool(1, 3, bs, h, d, dtype)

    mine, other = pools(), pools()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, pos, *mine)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x, pos, *mine)
    for i in range(4):
        x.copy_(rows(g, n, hq + 2 * h, d, dtype))
        pos.copy_(positions(g, 3, n, 10 ** (i + 2)))
        want = [t.clone() for t in step(x, pos, *other)]
        graph.replay()
        if i % 2:
            torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), i


def test_empty_calls_and_bad_slots():
    hq, h, d, bs, dtype = 4, 2, 64, 16, torch.bfloat16
    rotary = RotaryAxes.grid(d, 2)
    pool = PagedKVPool(1, 2, bs, h, d, dtype)
    x = torch.ones(3, hq + 2 * h, d, device=DEV, dtype=dtype)
    q, k, v = x.split([hq, h, h], 1)
    pos = torch.ones(2, 3, dtype=torch.long, device=DEV)
    none = slice(0, 0)
    out = kernels.rope_axes_kv_scatter(q[none], k[none], v[none], pos[:, none], rotary, pool.k[0], pool.v[0],
                                       pos[0, none])
    assert out.shape == (0, hq, d)
    assert kernels.rope_axes(q[none], k[none], pos[:, none], rotary)[1].shape == (0, h, d)
    only_k = kernels.rope_axes(q[:, :0], k, pos, rotary)
    assert only_k[0].shape == (3, 0, d) and torch.equal(only_k[1], kernels.rope_axes(q, k, pos, rotary)[1])
    slots = torch.tensor([1, -1, 32], device=DEV)
    qo = kernels.rope_axes_kv_scatter(q, k, v, pos, rotary, pool.k[0], pool.v[0], slots, err_flags=pool.err_flags)
    with pytest.raises(IndexError, match="write slot"):
        pool.check_errors()
    assert torch.equal(qo[0], qo[2]) and pool.k[0, 1].any() and not pool.k[0, 2:].any() and not pool.k[0, 0].any()


def test_refusals():
    hq, h, d, bs, dtype = 4, 2, 64, 16, torch.bfloat16
    rotary = RotaryAxes.sections(d, (8, 12, 12))
    pool, eight = PagedKVPool(1, 2, bs, h, d, dtype), QuantPagedKVPool(1, 2, bs, h, d, dtype)
    x = torch.ones(3, hq + 2 * h, d, device=DEV, dtype=dtype)
    q, k, v = x.split([hq, h, h], 1)
    pos = torch.ones(3, 3, dtype=torch.long, device=DEV)
    slots = torch.arange(3, device=DEV)
    caches = (pool.k[0], pool.v[0])
    w = torch.ones(d, device=DEV, dtype=dtype)
    for bad in (pos[:2], pos[0], pos[None]):
        with pytest.raises(RuntimeError, match="axes"):
            kernels.rope_axes(q, k, bad, rotary)
    for bad in (pos.int(), pos.float(), pos[:, :2]):
        with pytest.raises(RuntimeError, match="positions must be"):
            kernels.rope_axes(q, k, bad, rotary)
    with pytest.raises(RuntimeError, match="pairs"):
        kernels.rope_axes(q, k, pos, RotaryAxes.sections(128, (16, 24, 24)))
    with pytest.raises(RuntimeError, match="expected"):
        kernels.rope_axes(q, k[:2], pos, rotary)
    with pytest.raises(RuntimeError, match="dtype"):
        kernels.rope_axes(q, k.half(), pos, rotary)
    with pytest.raises(RuntimeError, match="norm weight"):
        kernels.rope_axes(q, k, pos, rotary, w)
    with pytest.raises(RuntimeError, match="q_norm"):
        kernels.rope_axes(q, k, pos, rotary, w.float(), w)
    with pytest.raises(RuntimeError, match="out must be"):
        kernels.rope_axes(q, k, pos, rotary, q_out=q.half())
    with pytest.raises(RuntimeError, match="k_out must be"):
        kernels.rope_axes(q, k, pos, rotary, k_out=k.float())
    with pytest.raises(RuntimeError, match="head_dim 80"):
        r80, x80 = RotaryAxes.grid(80, 2), torch.ones(1, 2, 80, device=DEV, dtype=dtype)
        kernels.rope_axes(x80, x80, pos[:2, :1], r80, w80 := torch.ones(80, device=DEV, dtype=dtype), w80)
    with pytest.raises(RuntimeError, match="ROCm device"):
        kernels.rope_axes(q.cpu(), k.cpu(), pos.cpu(), rotary)
    with pytest.raises(RuntimeError, match="pool"):
        kernels.rope_axes_kv_scatter(q, k, v, pos, rotary, eight.k[0], eight.v[0], slots)
    with pytest.raises(RuntimeError, match="kv_scales|codes"):
        kernels.rope_axes_kv_scatter(q, k, v, pos, rotary, eight.k[0], eight.v[0], slots,
                                     kv_scales=eight.kv_scales[0], block_size=bs)
    with pytest.raises(RuntimeError, match="slots"):
        kernels.rope_axes_kv_scatter(q, k, v, pos, rotary, *caches, slots[:2])
    with pytest.raises(RuntimeError, match="k and v differ"):
        kernels.rope_axes_kv_scatter(q, k, v[:, :1], pos, rotary, *caches, slots)
    paged, mask = metadata.decode_context(pool, [[0], [1], [0]], [1, 1, 3])
    r4 = [t.unsqueeze(1) for t in (q, k, v)]
    with pytest.raises(RuntimeError, match="positions"):
        rope_axes_paged_attention(*r4, pos, rotary, paged, mask, 0, 0.1, 2)
    with pytest.raises(RuntimeError, match="go together"):
        rope_axes_paged_attention(*r4, pos.view(3, 3, 1), rotary, paged, mask, 0, 0.1, 2, q_norm=w)
    with pytest.raises(RuntimeError, match="n_rep"):
        rope_axes_paged_attention(*r4, pos.view(3, 3, 1), rotary, paged, mask, 0, 0.1, 3)
    assert not pool.k.any() and not eight.k.view(torch.uint8).any()
    torch.cuda.synchronize()
