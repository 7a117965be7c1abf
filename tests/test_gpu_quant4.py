"""The 4-bit pool on the GPU against its definition in 64 bits: the quantising write and
reading back exactly, attention within the bounds that the 8-bit pool's tests derive (its
roundings are the same), and all of them together as a step uses them."""

from __future__ import annotations

import pytest
import torch

from infrared_amd import (
    PagedContext,
    PagedKVPool,
    Quant4PagedKVPool,
    QuantPagedKVPool,
    RotaryAxes,
    kernels,
    metadata,
    paged_attention,
    rope_axes_paged_attention,
    rope_paged_attention,
)
from infrared_amd.hip_graph import HipGraphDecoder, build_decode_static_inputs
from infrared_amd.mixed_step import MixedConfig, MixedStep, make_mixed_case
from oracle import quant, quant4
from test_gpu_quant import (
    decode_tolerance,
    device_tables,
    fp32_tolerance,
    gen,
    norm_tolerance,
    prefill_tolerance,
    rotation,
    rows,
    run_decode,
    same,
    step_inputs,
)
from test_gpu_rope_axes import positions
from test_gpu_rope_axes import tolerance as turn_tolerance

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
DEV = "cuda"


def held(pool, layer=0):
    """All values of a layer ``[2, slots, H_kv, D]`` in 64 bits on the CPU."""
    k, v = pool.gather(layer, torch.arange(pool.num_slots, device=DEV))
    assert k.dtype == pool.dtype
    return torch.stack([k, v]).double().cpu()


# ---- writing and reading


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_holds_every_code_at_every_scale(dtype, d):
    """Numbers that are codes times a scale come back as they are."""
    lo, hi = quant4.BOUNDS[dtype]
    n = hi - lo + 1
    codes = torch.tensor(quant4.CODES).double()
    group = torch.cat([codes, -codes, codes.flip(0), -codes])
    x = torch.exp2(torch.arange(lo, hi + 1).double())[:, None, None] * group.repeat(d // 32)
    # (each group at a scale of its own)
    x = x.view(n, 1, d // 32, 32)
    x = torch.cat([x[:, :, :1], x.flip(0)[:, :, 1:]], 2).reshape(n, 1, d)
    pool = Quant4PagedKVPool(1, -(-n // 16), 16, 1, d, dtype)
    slots = torch.randperm(n, generator=torch.Generator().manual_seed(1)).to(DEV)
    pool.write(0, x.to(dtype).to(DEV), x.flip(0).neg().to(dtype).to(DEV), slots)
    got = held(pool)[:, slots.cpu()]
    assert torch.equal(got[0], x) and torch.equal(got[1], -x.flip(0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d, h, bs", [(128, 4, 16), (64, 2, 16), (64, 3, 32), (128, 1, 48), (64, 5, 1024)])
@pytest.mark.parametrize("n", [1, 2, 15, 77])
def test_write_changes_its_slots_alone(dtype, d, h, bs, n):
    """Tokens in any order over a pool that holds others; skipped and bad slots."""
    blocks = -(-200 // bs) + 1
    pool, want = Quant4PagedKVPool(2, blocks, bs, h, d, dtype), quant4.Quant4Cache(blocks * bs, h, d, dtype)
    g = gen(n + d + h)
    total = pool.num_slots
    assert same(held(pool, 1), want.values)
    for i in range(3):
        slots = torch.randperm(total, generator=g, device=DEV)[:n]
        if i == 1:
            slots[0] = -5
        k, v = rows(g, n, h, d, dtype, 2.0), rows(g, n, h, d, dtype)
        pool.write(1, k, v, slots)
        pool.check_errors()
        want.write(k, v, slots)
        assert same(held(pool, 1), want.values)
    assert not held(pool, 0).any()
    slots[n // 2] = total
    pool.write(1, k, v, slots)
    with pytest.raises(IndexError, match="write slot"):
        pool.check_errors()
    want.write(k, v, slots)
    assert same(held(pool, 1), want.values)


@pytest.mark.parametrize("n", [3, 65, 1024])
@pytest.mark.parametrize("d", [64, 128])
def test_the_last_of_rows_given_the_same_slot_is_written(n, d):
    """Also where the rows differ; with rotation and norms too."""
    h, bs, dtype = 3, 16, torch.bfloat16
    g = gen(n)
    k, v = rows(g, n, h, d, dtype, 3.0), rows(g, n, h, d, dtype, 3.0)
    slots = torch.randint(0, max(2, n // 3), (n,), generator=g, device=DEV)
    pool, want = Quant4PagedKVPool(1, 30, bs, h, d, dtype), quant4.Quant4Cache(480, h, d, dtype)
    for _ in range(3):
        pool.write(0, k, v, slots)
        for i in range(n):
            want.write(k[i : i + 1], v[i : i + 1], slots[i : i + 1])
        assert same(held(pool), want.values)
    cos, sin = rotation(g, n, d)
    w = torch.ones(d, dtype=dtype, device=DEV)
    one = Quant4PagedKVPool(1, 30, bs, h, d, dtype)
    last = torch.tensor([int((slots == s).nonzero().max()) for s in slots.unique()], device=DEV)
    for p, at in ((pool, slice(None)), (one, last)):
        p.kv_scales.fill_(27)
        p.k.zero_()
        p.v.zero_()
        kernels.rope_kv_scatter_q4(k[at], k[at], v[at], cos[at], sin[at], p.k[0], p.v[0], p.kv_scales[0], slots[at], bs,
                                   w, w, 1e-6)
    assert torch.equal(pool.k, one.k) and torch.equal(pool.v, one.v) and torch.equal(pool.kv_scales, one.kv_scales)


def test_write_of_long_calls():
    """More tokens than one wavefront each, in order and shuffled."""
    h, d, bs, n, dtype = 3, 128, 16, 5000, torch.bfloat16
    g = gen(3)
    pool, want = Quant4PagedKVPool(1, 320, bs, h, d, dtype), quant4.Quant4Cache(5120, h, d, dtype)
    for slots in (torch.arange(7, 7 + n, device=DEV), torch.randperm(5120, generator=g, device=DEV)[:n]):
        k, v = rows(g, n, h, d, dtype), rows(g, n, h, d, dtype)
        pool.write(0, k, v, slots)
        want.write(k, v, slots)
        assert same(held(pool), want.values)


@pytest.mark.parametrize("dtype", DTYPES)
def test_write_of_extreme_numbers(dtype):
    """Zeros, the type's largest and smallest numbers, NaN and infinities, borders."""
    bs, h, d = 16, 1, 64
    f = torch.finfo(dtype)
    pool, want = Quant4PagedKVPool(1, 8, bs, h, d, dtype), quant4.Quant4Cache(128, h, d, dtype)
    g = gen(5)

    def put(x, slots):
        x = x.to(dtype).view(-1, h, d)
        slots = torch.tensor(slots, device=DEV)
        pool.write(0, x, -x, slots)
        want.write(x, -x, slots)
        assert same(held(pool), want.values)

    put(torch.zeros(3 * d, device=DEV), [0, 1, 2])
    ramp = torch.linspace(-1, 1, d, device=DEV, dtype=torch.float64)
    put(f.max * ramp, [16])
    put(f.max * ramp.flip(0) / 3, [17])
    put(f.smallest_normal * 64 * ramp, [32])
    put(f.smallest_normal * f.eps * (torch.arange(d, device=DEV) % 9), [33])
    odd = torch.randn(d, generator=g, device=DEV)
    odd[3] = float("nan")
    put(odd, [48])  # (the other group of the row is as it was)
    odd[3] = float("inf")
    put(odd, [49])
    odd[3], odd[60] = 0.0, float("-inf")
    put(odd, [48])
    put(torch.full((d,), float("nan"), device=DEV), [64])
    put(odd.nan_to_num(0.0, 0.0, 0.0), [64])
    # both sides of the border where the scale steps, and of ties between codes
    for top in (7.0, 7.0 * (1 + f.eps), 6.5, 3.5, 3.5 * (1 + f.eps)):
        edge = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.2, 0.3, 1.2, 2.6, 3.4, 4.9, 0.0, -0.75, top],
                            device=DEV).repeat(4)
        put(edge, [80])


def test_write_reads_strided_rows_and_runs_on_the_current_stream():
    bs, h, d, n = 16, 4, 128, 37
    pool, want = Quant4PagedKVPool(3, 8, bs, h, d, torch.bfloat16), quant4.Quant4Cache(128, h, d, torch.bfloat16)
    qkv = rows(gen(6), n, 3 * h, d, torch.bfloat16)
    slots = torch.arange(60, 60 + n, device=DEV)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        pool.write(2, qkv[:, h : 2 * h], qkv[:, 2 * h :], torch.stack([slots, slots], 1)[:, 1])
    torch.cuda.current_stream().wait_stream(stream)
    want.write(qkv[:, h : 2 * h], qkv[:, 2 * h :], slots)
    assert same(held(pool, 2), want.values)
    assert not pool.k[:2].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_reads_through_tables_and_flags_bad_slots(dtype, d):
    pool = Quant4PagedKVPool(2, 12, 16, 3, d, dtype)
    g = gen(1)
    slots = torch.arange(pool.num_slots, device=DEV)
    pool.write(1, rows(g, pool.num_slots, 3, d, dtype), rows(g, pool.num_slots, 3, d, dtype), slots)
    k, v = pool.gather(1, slots)
    tables = torch.tensor([[3, 7, 1], [11, 0, 99]], dtype=torch.int32, device=DEV)
    ctx = torch.tensor([40, 17], dtype=torch.int32, device=DEV)
    gk, gv = pool.gather_blocks(1, tables, ctx, 45)
    pool.check_errors()
    for b in range(2):
        for t in range(45):
            s = int(tables[b, min(t // 16, 2)]) * 16 + t % 16
            inside = t < int(ctx[b])
            assert torch.equal(gk[b, t], k[s] if inside else torch.zeros_like(k[0]))
            assert torch.equal(gv[b, t], v[s] if inside else torch.zeros_like(v[0]))
    bad = torch.tensor([[5, -1], [pool.num_slots, 6]], device=DEV)
    gk, _ = pool.gather(1, bad)
    assert torch.equal(gk[0, 0], k[5]) and torch.equal(gk[1, 1], k[6]) and not gk[0, 1].any() and not gk[1, 0].any()
    with pytest.raises(IndexError, match="gather slot"):
        pool.check_errors()
    pool.gather_blocks(1, tables, torch.tensor([1, 40], dtype=torch.int32, device=DEV), 45)
    with pytest.raises(IndexError, match="block id"):
        pool.check_errors()
    pool.gather_blocks(1, tables, torch.tensor([1, 50], dtype=torch.int32, device=DEV), 2)
    with pytest.raises(IndexError, match="context length"):
        pool.check_errors()
    assert pool.gather(1, bad[:0])[0].shape == (0, 2, 3, d)


def test_pool_over_four_gigabytes():
    """Codes whose offsets pass 32 bits: the last blocks of a 4.3 GB layer, and its last head."""
    blocks, bs, h, d = (1 << 18) + 64, 64, 4, 128
    pool = Quant4PagedKVPool(1, blocks, bs, h, d, torch.bfloat16)
    assert pool.k[0].numel() > 1 << 32
    g = gen(7)
    ids = [blocks - 1, 3, blocks - 2]
    n = 150
    slots = torch.tensor([ids[p // bs] * bs + p % bs for p in range(n)], device=DEV)
    k, v = rows(g, n, h, d, torch.bfloat16), rows(g, n, h, d, torch.bfloat16)
    pool.write(0, k, v, slots)
    small = quant4.Quant4Cache(3 * bs, h, d, torch.bfloat16)
    small.write(k, v, torch.arange(n))
    gk, gv = pool.gather(0, slots)
    assert torch.equal(torch.stack([gk, gv]).double().cpu(), small.values[:, :n])
    q = torch.randn(1, 8, d, generator=g, device=DEV).bfloat16()
    tables = torch.tensor([ids], dtype=torch.int32, device=DEV)
    ctx = torch.tensor([n], dtype=torch.int32, device=DEV)
    o, a, reach = quant.attend(q, small.values, [0, 1, 2], bs, n - 1, d**-0.5)
    tol = decode_tolerance(o, a, torch.bfloat16) + fp32_tolerance(o, a, reach, d)
    for planned in (False, True):
        out = run_decode(pool, q, tables, ctx, planned)
        assert ((out.double().cpu() - o).abs() <= tol).all()
    cu = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    out = kernels.paged_prefill(q, pool.k[0], pool.v[0], tables, cu, ctx - 1, 1, bs, d**-0.5,
                                kv_scales=pool.kv_scales[0])
    assert ((out.double().cpu() - o).abs() <= tol + prefill_tolerance(o, a, reach, torch.bfloat16)).all()
    pool.check_errors()


# ---- attention


def filled(seed, dtype, lens, h, d, bs, spare=3):
    """A pool whose sequences of ``lens`` tokens were written, the rest of it NaN."""
    g = gen(seed)
    need = [max(1, -(-n // bs)) for n in lens]
    blocks = sum(need) + spare
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).tolist()
    tables = [[order.pop() for _ in range(n)] for n in need]
    pool = Quant4PagedKVPool(1, blocks, bs, h, d, dtype)
    everything = torch.arange(pool.num_slots, device=DEV)
    nan = torch.full((pool.num_slots, h, d), float("nan"), dtype=dtype, device=DEV)
    pool.write(0, nan, nan, everything)
    slots = torch.tensor([metadata.slot(t, p, bs) for t, n in zip(tables, lens) for p in range(n)],
                         dtype=torch.long, device=DEV)
    total = len(slots)
    k, v = rows(g, total, h, d, dtype, 0.5), rows(g, total, h, d, dtype)
    pool.write(0, k, v, slots)
    return pool, tables, held(pool).nan_to_num(0.0)


# Many values are 0, and an output can consist of small probabilities alone. fp16 ones are held
# 2^7 times larger than their ratio to a running maximum that the largest is not below, and
# below fp16's smallest normal number a rounding is off by up to 2^-25: 2^-32 sum |v| of an
# output, whose divisor is 1 at least (two roundings where a probability is two pieces). In
# the other types a probability below fp32's smallest normal number, 2^-126, may be 0. An output
# that small is rounded by up to half of the type's smallest number, 2^-25 in fp16, or to 0.


def small_probabilities(values, table, n, bs, hq, dtype):
    t = torch.arange(n)
    v = values[1, torch.tensor(table)[t // bs] * bs + t % bs].abs().sum(0)
    p, out = (-32, -25) if dtype == torch.float16 else (-126, -126)
    return 2 * 2.0**p * v.repeat_interleave(hq // v.shape[0], 0) + 2.0**out


def check_decode(out, q, values, tables, lens, bs, dtype):
    d = q.shape[2]
    for i, n in enumerate(lens):
        if n == 0:
            assert not out[i].any()
            continue
        o, a, reach = quant.attend(q[i : i + 1], values, tables[i], bs, n - 1, d**-0.5)
        tol = fp32_tolerance(o, a, reach, d) + small_probabilities(values, tables[i], n, bs, q.shape[1], dtype)
        if dtype != torch.float32:
            tol = tol + decode_tolerance(o, a, dtype)
        err = (out[i : i + 1].double().cpu() - o).abs()
        assert (err <= tol).all(), (i, n, (err / tol).max())


@pytest.mark.parametrize("planned", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq, h, d, bs", [(28, 4, 128, 16), (14, 2, 64, 16), (8, 8, 64, 32), (20, 1, 128, 48),
                                          (3, 3, 128, 128), (33, 1, 64, 16)])
def test_decode(planned, dtype, hq, h, d, bs):
    lens = [1, 2, 15, 16, 17, 33, 300, 1100, 64, 0, 5]
    pool, tables, values = filled(hq + d, dtype, lens, h, d, bs)
    q = torch.randn(len(lens), 2 * hq, d, generator=gen(9), device=DEV).to(dtype)[:, hq:]
    ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = run_decode(pool, q, device_tables(tables), ctx, planned)
    pool.check_errors()
    check_decode(out, q, values, tables, lens, bs, dtype)


@pytest.mark.parametrize("planned", [False, True])
@pytest.mark.parametrize("dtype, d", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 128)])
def test_decode_of_long_contexts_and_shared_prefixes(planned, dtype, d):
    """Contexts cut into parts, pairs of sequences whose tables begin alike."""
    bs, hq, h = 16, 28, 4
    lens = [9000, 700, 4097, 2500]
    pool, tables, values = filled(21, dtype, lens, h, d, bs)
    tables.append(tables[3][:100] + tables[1][:20])
    tables.append(tables[3][:100] + tables[0][:7])
    lens = lens + [1600 + 311, 1600 + 112]
    q = torch.randn(len(lens), hq, d, generator=gen(10), device=DEV).to(dtype)
    ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
    bt = device_tables(tables)
    out = run_decode(pool, q, bt, ctx, planned)
    pool.check_errors()
    check_decode(out, q, values, tables, lens, bs, dtype)
    assert torch.equal(out, run_decode(pool, q, bt, ctx, planned))  # nothing of a call is left for the next


@pytest.mark.parametrize("dtype, hq, h, d, lens", [
    (torch.bfloat16, 28, 4, 128, [20011]), (torch.float16, 14, 2, 64, [9000, 0, 17]),
    (torch.float32, 6, 2, 128, [5000]),
    (torch.bfloat16, 40, 2, 64, [8191, 4000]), (torch.bfloat16, 8, 1, 128, [300, 1, 0]),
])
def test_decode_of_few_sequences_over_many_slices(dtype, hq, h, d, lens):
    """Few units over many slices: groups of more than 16 query heads, an empty sequence, and
    the same with a sequence that shares a prefix."""
    bs = 16
    pool, tables, values = filled(23, dtype, lens, h, d, bs)
    if lens[0] > 1000:
        tables.append(tables[0][:200])
        lens = lens + [200 * bs - 3]
        tables, lens = [tables[0], tables[-1], *tables[1:-1]], [lens[0], lens[-1], *lens[1:-1]]
    q = torch.randn(len(lens), hq, d, generator=gen(10), device=DEV).to(dtype)
    ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
    bt = device_tables(tables)
    for planned in (True, False):
        out = run_decode(pool, q, bt, ctx, planned)
        pool.check_errors()
        check_decode(out, q, values, tables, lens, bs, dtype)
        assert torch.equal(out, run_decode(pool, q, bt, ctx, planned))


def test_decode_of_many_sequences():
    """More sequences than wavefronts, most of them short, several units a wavefront."""
    bs, hq, h, d, dtype = 16, 14, 2, 64, torch.bfloat16
    lens = [(i * 37) % 90 for i in range(300)] + [1200]
    pool, tables, values = filled(24, dtype, lens, h, d, bs)
    q = torch.randn(len(lens), hq, d, generator=gen(25), device=DEV).to(dtype)
    ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
    for planned in (True, False):
        out = run_decode(pool, q, device_tables(tables), ctx, planned)
        pool.check_errors()
        check_decode(out, q, values, tables, lens, bs, dtype)


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("dtype, hq, h, d", [(torch.bfloat16, 28, 4, 128), (torch.float32, 10, 2, 64)])
def test_decode_joins_units_of_several_wavefronts(dtype, hq, h, d, shared):
    """Sequences of about a wavefront's, several wavefronts' and more than a workgroup's share of
    the keys: one to eight units of a workgroup are joined, others cross to the next."""
    bs = 16
    for lens in ([320] * 60 + [17, 700, 2500, 1], [(i * 97) % 400 + 1 for i in range(150)], [1100, 1090, 3, 1300]):
        pool, tables, values = filled(29, dtype, lens, h, d, bs)
        if shared:
            for i in range(0, len(lens) - 1, 3):  # every third sequence begins as the one before it
                n = min(lens[i], lens[i + 1]) // bs
                tables[i + 1][:n] = tables[i][:n]
        q = torch.randn(len(lens), hq, d, generator=gen(30), device=DEV).to(dtype)
        ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
        bt = device_tables(tables)
        out = run_decode(pool, q, bt, ctx, True)
        pool.check_errors()
        check_decode(out, q, values, tables, lens, bs, dtype)
        assert torch.equal(out, run_decode(pool, q, bt, ctx, True))


# (the bounds of check_decode; a negative scale's scores are those of the opposite queries)
@pytest.mark.parametrize("planned", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.0, -0.11, 1e-40, 0.7])
def test_decode_at_any_scale(planned, dtype, scale):
    bs, hq, h, d = 16, 14, 2, 64
    lens = [1, 40, 333, 0]
    pool, tables, values = filled(31, dtype, lens, h, d, bs)
    ctx, bt = torch.tensor(lens, dtype=torch.int32, device=DEV), device_tables(tables)
    for q_dtype in {dtype, torch.float32}:
        q = torch.randn(len(lens), hq, d, generator=gen(32), device=DEV).to(q_dtype)
        kw = {"out": torch.empty(len(lens), hq, d, dtype=dtype, device=DEV), "kv_scales": pool.kv_scales[0]}
        if planned:
            plan = kernels.decode_plan(bt, ctx, hq, pool.k[0], bs)
            out = kernels.paged_decode_planned(q, pool.k[0], pool.v[0], plan, scale, **kw)
        else:
            out = kernels.paged_decode(q, pool.k[0], pool.v[0], bt, ctx, bs, scale, **kw)
        for i, n in enumerate(lens):
            if n == 0:
                assert not out[i].any()
                continue
            sign = -1.0 if scale < 0 else 1.0
            o, a, reach = quant.attend(sign * q[i : i + 1], values, tables[i], bs, n - 1, sign * scale)
            tol = fp32_tolerance(o, a, reach, d) + small_probabilities(values, tables[i], n, bs, hq, dtype)
            if dtype != torch.float32:
                # (an fp32 query in two pieces of the dtype: 2^-18 of an element, as above)
                tol = tol + decode_tolerance(o, a, dtype) + 4 * 2.0**-13 * reach[..., None] * a
            err = (out[i : i + 1].double().cpu() - o).abs()
            assert (err <= tol).all(), (q_dtype, i, n, (err / tol).max())


@pytest.mark.parametrize("planned", [False, True])
def test_decode_masks_bad_blocks_and_lengths(planned):
    bs, hq, h, d = 16, 8, 2, 64
    pool, tables, values = filled(22, torch.bfloat16, [100, 50], h, d, bs)
    bt = device_tables(tables)
    q = torch.randn(2, hq, d, generator=gen(11), device=DEV).bfloat16()
    ctx = torch.tensor([100, 50], dtype=torch.int32, device=DEV)
    want = run_decode(pool, q, bt, ctx, planned)
    for bad in (pool.num_blocks, -1):
        bt[0, 2] = bad
        got = run_decode(pool, q, bt, ctx, planned)
        with pytest.raises(IndexError, match="block id"):
            pool.check_errors()
        assert torch.equal(got[1], want[1]) and got[0].isfinite().all() and not torch.equal(got[0], want[0])
    bt[0, 2] = tables[0][2]
    over = torch.tensor([-3, bt.shape[1] * bs + 1], dtype=torch.int32, device=DEV)
    got = run_decode(pool, q, bt, over, planned)
    with pytest.raises(IndexError, match="context length"):
        pool.check_errors()
    assert not got[0].any()


@pytest.mark.parametrize("path", ["decode", "planned", "prefill"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_a_key_that_is_no_number_spoils_who_sees_it_alone(path, dtype, d):
    """NaN in a group of one key of a head: that head's queries of that sequence. (Of V in a
    prefill also the queries of its chunk that come before it, as over the other pools: a
    tile's products are with all its keys, and zero times NaN is NaN.)"""
    bs, hq, h = 16, 6, 2
    lens, at = [70, 40], 33
    pool, tables, values = filled(26, dtype, lens, h, d, bs)
    slot = torch.tensor([metadata.slot(tables[0], at, bs)], device=DEV)
    k, v = pool.gather(0, slot)
    for which in (0, 1):  # K, then V
        kv = [k.clone(), v.clone()]
        kv[which][0, 1, 3] = float("nan")
        pool.write(0, *kv, slot)
        bt, ctx = device_tables(tables), torch.tensor(lens, dtype=torch.int32, device=DEV)
        if path != "prefill":
            q = torch.randn(2, hq, d, generator=gen(27), device=DEV).to(dtype)
            out = run_decode(pool, q, bt, ctx, path == "planned").float()
            seen = torch.tensor([[False] * 3 + [True] * 3, [False] * 6], device=DEV)
        else:
            n = [50, 40]
            q = torch.randn(sum(n), hq, d, generator=gen(27), device=DEV).to(dtype)
            cu = torch.tensor([0, 50, 90], dtype=torch.int32, device=DEV)
            start = torch.tensor([20, 0], dtype=torch.int32, device=DEV)
            out = kernels.paged_prefill(q, pool.k[0], pool.v[0], bt, cu, start, 50, bs, d**-0.5,
                                        kv_scales=pool.kv_scales[0]).float()
            seen = torch.zeros(90, hq, dtype=torch.bool, device=DEV)
            seen[at - 20 : 50, 3:] = True
        if which:  # the group's 32 channels
            assert out[..., :32][seen].isnan().all() and out[..., 32:].isfinite().all()
            if path == "prefill":
                seen[:50, 3:] = True
        else:
            assert out[seen].isnan().all()
        assert out[~seen].isfinite().all()


@pytest.mark.parametrize("plan", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq, h, d, bs", [(28, 4, 128, 16), (14, 2, 64, 16), (8, 8, 64, 64), (20, 1, 128, 48)])
def test_prefill(plan, dtype, hq, h, d, bs):
    """Chunks of one token to several tiles after prefixes of any length, an empty one."""
    cached, new = [0, 37, 0, 512, 1, 130], [1, 70, 200, 1, 0, 65]
    lens = [c + n for c, n in zip(cached, new)]
    pool, tables, values = filled(hq, dtype, lens, h, d, bs)
    total = sum(new)
    q = torch.randn(total, 2 * hq, d, generator=gen(12), device=DEV).to(dtype)[:, :hq]  # (rows of a wider tensor)
    cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
    start = torch.tensor(cached, dtype=torch.int32, device=DEV)
    bt = device_tables(tables)
    p = kernels.prefill_plan(cu, start, bt, total, max(new), bs, hq, h, d, dtype=dtype) if plan else None
    out = kernels.paged_prefill(q, pool.k[0], pool.v[0], bt, cu, start, max(new), bs, d**-0.5,
                                err_flags=pool.err_flags, plan=p, kv_scales=pool.kv_scales[0])
    pool.check_errors()
    row = 0
    for t, c, n in zip(tables, cached, new):
        if n:
            o, a, reach = quant.attend(q[row : row + n], values, t, bs, c, d**-0.5)
            tol = fp32_tolerance(o, a, reach, d) + small_probabilities(values, t, c + n, bs, hq, dtype)
            if dtype != torch.float32:
                tol = tol + prefill_tolerance(o, a, reach, dtype)
            err = (out[row : row + n].double().cpu() - o).abs()
            assert (err <= tol).all(), (c, n, (err / tol).max())
        row += n


@pytest.mark.parametrize("dtype", DTYPES)
def test_prefill_masks_bad_blocks(dtype):
    """A bad block id is flagged and its keys read as zeros; the other sequence is as it was."""
    bs, hq, h, d = 16, 4, 2, 128
    pool, tables, values = filled(28, dtype, [90, 60], h, d, bs)
    q = torch.randn(50, hq, d, generator=gen(29), device=DEV).to(dtype)
    cu = torch.tensor([0, 30, 50], dtype=torch.int32, device=DEV)
    start = torch.tensor([60, 40], dtype=torch.int32, device=DEV)
    bt = device_tables(tables)
    args = (cu, start, 30, bs, d**-0.5)
    want = kernels.paged_prefill(q, pool.k[0], pool.v[0], bt, *args, kv_scales=pool.kv_scales[0])
    bt[0, 1] = pool.num_blocks + 5
    got = kernels.paged_prefill(q, pool.k[0], pool.v[0], bt, *args, err_flags=pool.err_flags,
                                kv_scales=pool.kv_scales[0])
    with pytest.raises(IndexError, match="block id"):
        pool.check_errors()
    assert torch.equal(got[30:], want[30:]) and got.isfinite().all()
    spare = torch.zeros(2, bs, h, d, dtype=torch.float64)
    o, a, reach = quant.attend(q[:30], torch.cat([values, spare], 1),
                               [tables[0][0], pool.num_blocks, *tables[0][2:]], bs, 60, d**-0.5)
    tol = fp32_tolerance(o, a, reach, d) + small_probabilities(values, tables[0], 90, bs, hq, dtype)
    if dtype != torch.float32:
        tol = tol + prefill_tolerance(o, a, reach, dtype)
    assert ((got[:30].double().cpu() - o).abs() <= tol).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_prefill_of_queries_of_any_size(dtype, d):
    """Queries of zeros, of the type's small numbers, with one element that dwarfs the
    others; infinite and NaN ones spoil their own rows alone."""
    bs, hq, h, n = 16, 4, 2, 40
    pool, tables, values = filled(33, dtype, [60], h, d, bs)
    q = torch.randn(n, hq, d, generator=gen(14), device=DEV)
    q[1] = 0.0
    q[2] *= 1e-4
    q[3, :, 5] *= 3e3
    q[4, :, 5] *= 300.0
    q[5] *= 60.0
    q = q.to(dtype)
    spoiled = torch.zeros(n, hq, dtype=torch.bool)
    for i, x in ((7, float("inf")), (9, float("-inf")), (11, float("nan"))):
        q[i, 1, 3] = x
        spoiled[i, 1] = True
    cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    start = torch.tensor([20], dtype=torch.int32, device=DEV)
    out = kernels.paged_prefill(q, pool.k[0], pool.v[0], device_tables(tables), cu, start, n, bs, d**-0.5,
                                err_flags=pool.err_flags, kv_scales=pool.kv_scales[0])
    o, a, reach = quant.attend(q.nan_to_num(0.0, 0.0, 0.0), values, tables[0], bs, 20, d**-0.5)
    tol = fp32_tolerance(o, a, reach, d) + small_probabilities(values, tables[0], 60, bs, hq, dtype)
    if dtype != torch.float32:
        tol = tol + prefill_tolerance(o, a, reach, dtype)
    out = out.double().cpu()
    assert ((out - o).abs() <= tol)[~spoiled].all()
    assert out[spoiled].isnan().any(-1).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_prefill_over_many_workgroups_and_wide_groups(dtype):
    """More workgroups than the device holds, cut items; 8-wavefront workgroups (more than
    128 query heads a KV head) in bf16."""
    bs, d = 16, 64
    cached, new = [6000, 0, 300], [700, 900, 257]
    lens = [c + n for c, n in zip(cached, new)]
    for hq, h in ((8, 4), (130, 1) if dtype == torch.bfloat16 else (64, 1)):
        pool, tables, values = filled(31, dtype, lens, h, d, bs)
        total = sum(new)
        q = torch.randn(total, hq, d, generator=gen(13), device=DEV).to(dtype)
        cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
        start = torch.tensor(cached, dtype=torch.int32, device=DEV)
        bt = device_tables(tables)
        plan = kernels.prefill_plan(cu, start, bt, total, max(new), bs, hq, h, d, dtype=dtype)
        for p in (plan, None, plan):
            out = kernels.paged_prefill(q, pool.k[0], pool.v[0], bt, cu, start, max(new), bs, d**-0.5, plan=p,
                                        kv_scales=pool.kv_scales[0])
            row = 0
            for t, c, n in zip(tables, cached, new):
                heads = slice(0, hq) if hq <= 8 else slice(hq - 3, hq)  # (the oracle's cost)
                x = q[row : row + n]
                o, a, reach = quant.attend(x[:, heads] if h == 1 else x, values, t, bs, c, d**-0.5)
                tol = fp32_tolerance(o, a, reach, d)
                if dtype != torch.float32:
                    tol = tol + prefill_tolerance(o, a, reach, dtype)
                got = out[row : row + n]
                err = ((got[:, heads] if h == 1 else got).double().cpu() - o).abs()
                assert (err <= tol).all(), (hq, c, n, (err / tol).max())
                row += n


# (the bounds are those of test_gpu_quant.py's test of the same name, but for fp16's small
# probabilities)
@pytest.mark.parametrize("path", ["decode", "planned", "prefill", "prefill_plan"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq, h, d, bs", [(28, 4, 128, 16), (14, 2, 64, 32), (130, 1, 64, 16)])
def test_fp32_queries_of_a_16_bit_pool(path, dtype, hq, h, d, bs):
    lens = [1, 16, 33, 300, 700, 64]
    pool, tables, values = filled(41 + hq, dtype, lens, h, d, bs)
    q = torch.randn(len(lens), 2 * hq, d, generator=gen(42), device=DEV)[:, :hq]
    bt, out = device_tables(tables), torch.empty(len(lens), hq, d, dtype=dtype, device=DEV)
    ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
    common = {"err_flags": pool.err_flags, "kv_scales": pool.kv_scales[0], "out": out}
    if path == "decode":
        kernels.paged_decode(q, pool.k[0], pool.v[0], bt, ctx, bs, 1.0, **common)
    elif path == "planned":
        plan = kernels.decode_plan(bt, ctx, hq, pool.k[0], bs)
        kernels.paged_decode_planned(q, pool.k[0], pool.v[0], plan, 1.0, **common)
    else:
        cu = torch.arange(len(lens) + 1, dtype=torch.int32, device=DEV)
        plan = None
        if path == "prefill_plan":
            plan = kernels.prefill_plan(cu, ctx - 1, bt, len(lens), 1, bs, hq, h, d, dtype=dtype)
        kernels.paged_prefill(q, pool.k[0], pool.v[0], bt, cu, ctx - 1, 1, bs, 1.0, plan=plan, **common)
    pool.check_errors()
    off = rounded = 0.0
    for i, n in enumerate(lens):
        o, a, reach = quant.attend(q[i : i + 1], values, tables[i], bs, n - 1, 1.0)
        tol = fp32_tolerance(o, a, reach, d) + decode_tolerance(o, a, dtype) + 4 * 2.0**-13 * reach[..., None] * a
        tol = tol + small_probabilities(values, tables[i], n, bs, hq, dtype)
        err = (out[i : i + 1].double().cpu() - o).abs()
        assert (err <= tol).all(), (i, n, (err / tol).max())
        off += err.square().sum().item()
        r, _, _ = quant.attend(q[i : i + 1].to(dtype), values, tables[i], bs, n - 1, 1.0)
        rounded += (r - o).square().sum().item()
    assert off < 0.25 * rounded, (off, rounded)


# (bf16 products of three pieces each: the pieces add up to the number, a product of 32 terms is off by
# 2^-22 of their size at most, and a score has d / 32 * 3 of them: within the 4 (d + 8) 2^-24 of fp32_tolerance)
@pytest.mark.parametrize("path", ["decode", "planned", "prefill"])
@pytest.mark.parametrize("d", [64, 128])
def test_fp32_pools_keep_queries_of_unlike_elements(path, d):
    """Elements of a row from 2^-14 to 2^14 times the others, rows of any size."""
    bs, hq, h = 16, 6, 2
    lens = [1, 40, 300, 1500]
    pool, tables, values = filled(45, torch.float32, lens, h, d, bs)
    g = gen(46)
    q = torch.randn(len(lens), hq, d, generator=g, device=DEV)
    q = q * torch.exp2(torch.randint(-14, 15, q.shape, generator=g, device=DEV).float())
    q = q * torch.tensor([1.0, 2.0**-20, 2.0**-10, 2.0**-13], device=DEV)[:, None, None]
    bt, ctx = device_tables(tables), torch.tensor(lens, dtype=torch.int32, device=DEV)
    if path == "prefill":
        cu = torch.arange(len(lens) + 1, dtype=torch.int32, device=DEV)
        out = kernels.paged_prefill(q, pool.k[0], pool.v[0], bt, cu, ctx - 1, 1, bs, d**-0.5,
                                    kv_scales=pool.kv_scales[0])
    else:
        out = run_decode(pool, q, bt, ctx, path == "planned")
    check_decode(out, q, values, tables, lens, bs, torch.float32)


def test_prefill_writes_rows_of_a_wider_output_alone():
    bs, hq, h, d = 48, 21, 3, 64
    cached, new = [0, 5, 1111, 48], [1, 49, 300, 48]
    lens = [c + n for c, n in zip(cached, new)]
    for dtype in DTYPES:
        pool, tables, values = filled(47, dtype, lens, h, d, bs)
        total = sum(new)
        q = torch.randn(total, 2 * hq, d + 8, generator=gen(48), device=DEV).to(dtype)[:, ::2, :d]
        wide = torch.full((total, hq + 1, d + 8), 7.0, dtype=dtype, device=DEV)
        cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
        start = torch.tensor(cached, dtype=torch.int32, device=DEV)
        kernels.paged_prefill(q, pool.k[0], pool.v[0], device_tables(tables), cu, start, max(new), bs, d**-0.5,
                              out=wide[:, :hq, :d], kv_scales=pool.kv_scales[0])
        assert (wide[:, hq:] == 7).all() and (wide[:, :, d:] == 7).all()
        row = 0
        for t, c, n in zip(tables, cached, new):
            o, a, reach = quant.attend(q[row : row + n], values, t, bs, c, d**-0.5)
            tol = fp32_tolerance(o, a, reach, d) + small_probabilities(values, t, c + n, bs, hq, dtype)
            if dtype != torch.float32:
                tol = tol + prefill_tolerance(o, a, reach, dtype)
            assert ((wide[row : row + n, :hq, :d].double().cpu() - o).abs() <= tol).all(), (dtype, c, n)
            row += n


@pytest.mark.parametrize("dtype, d", [(torch.bfloat16, 64), (torch.float32, 128), (torch.float16, 128)])
def test_graphs_of_both_decodes_share_a_workspace(dtype, d):
    """Replayed in turn, with eager calls between, the counters zero after each."""
    hq, h, bs = 14, 2, 16
    lens = [(i * 331) % 1300 + 1 for i in range(40)]
    pool, tables, _ = filled(49, dtype, lens, h, d, bs)
    bt, ctx = device_tables(tables), torch.tensor(lens, dtype=torch.int32, device=DEV)
    qs = torch.randn(2, len(lens), hq, d, generator=gen(50), device=DEV).to(dtype)
    plan = kernels.decode_plan(bt, ctx, hq, pool.k[0], bs)
    need = max(kernels.planned_workspace_bytes(len(lens), hq, h, d),
               kernels.decode_workspace_bytes(len(lens), hq, h, d, bt.shape[1], bs))
    kw = {"workspace": torch.empty(need, dtype=torch.uint8, device=DEV),
          "counters": torch.zeros(kernels.decode_num_counters(len(lens), hq, h), dtype=torch.int32, device=DEV),
          "kv_scales": pool.kv_scales[0]}
    calls = [lambda q: kernels.paged_decode_planned(q, pool.k[0], pool.v[0], plan, 0.1, **kw),
             lambda q: kernels.paged_decode(q, pool.k[0], pool.v[0], bt, ctx, bs, 0.1, **kw)]
    want = [f(q).clone() for f, q in zip(calls, qs)]
    graphs = []
    for f, q in zip(calls, qs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = f(q)
        graphs.append((graph, out))
    for _ in range(3):
        for (graph, out), w in zip(graphs, want):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, w) and not kw["counters"].any()
        for f, q in zip(calls, qs.flip(0)):
            f(q)


# ---- rotation into the pool


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq, h, d, bs, n", [(28, 4, 128, 16, 70), (14, 2, 64, 32, 1), (5, 5, 64, 16, 2500)])
def test_rotation_into_the_4_bit_pool_is_the_rotation_then_the_write(dtype, hq, h, d, bs, n):
    """Without norms: bit for bit ``rope_kv_scatter`` and ``write`` of its keys."""
    g, blocks = gen(14), -(-n // bs) + 2
    q, k, v = rows(g, n, hq + 2 * h, d, dtype).split([hq, h, h], 1)
    cos, sin = rotation(g, n, d)
    slots = torch.arange(5, 5 + n, device=DEV)
    plain = PagedKVPool(1, blocks, bs, h, d, dtype)
    q1 = kernels.rope_kv_scatter(q, k, v, cos, sin, plain.k[0], plain.v[0], slots)
    a, b = (Quant4PagedKVPool(1, blocks, bs, h, d, dtype) for _ in range(2))
    a.write(0, plain.k[0, slots], v, slots)
    q2 = kernels.rope_kv_scatter_q4(q, k, v, cos, sin, b.k[0], b.v[0], b.kv_scales[0], slots, bs)
    assert torch.equal(q1, q2) and torch.equal(a.kv_scales, b.kv_scales)
    assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq, h, d, bs", [(28, 4, 128, 16), (14, 2, 64, 32)])
def test_normed_rotation_into_the_4_bit_pool(dtype, hq, h, d, bs):
    """Queries as the 16-bit pool's call gives them, and in fp32; keys to the code nearest the
    number in 64 bits, or the next where that lies within the fp32 error of the border."""
    g, n = gen(15), 61
    q, k, v = rows(g, n, hq + 2 * h, d, dtype).split([hq, h, h], 1)
    wq, wk = (1 + 0.3 * torch.randn(2, d, generator=g, device=DEV)).to(dtype)
    cos, sin = rotation(g, n, d)
    slots = torch.arange(3, 3 + n, device=DEV)
    plain = PagedKVPool(1, 6, bs, h, d, dtype)
    q1 = kernels.qk_norm_rope_kv_scatter(q, k, v, wq, wk, 1e-6, cos, sin, plain.k[0], plain.v[0], slots)
    pool, want = Quant4PagedKVPool(1, 6, bs, h, d, dtype), quant4.Quant4Cache(6 * bs, h, d, dtype)
    args = (q, k, v, cos, sin, pool.k[0], pool.v[0], pool.kv_scales[0], slots, bs, wq, wk, 1e-6)
    q2 = kernels.rope_kv_scatter_q4(*args)
    q3 = kernels.rope_kv_scatter_q4(*args, torch.empty(n, hq + 1, d, device=DEV)[:, 1:])
    assert torch.equal(q1, q2) and torch.equal(q1, q3.to(dtype))
    o = quant.norm_rope(k, wk, 1e-6, cos, sin)
    want.write(o, v, slots)
    got = held(pool)
    assert torch.equal(got[1], want.values[1])
    x, y = got[0, slots.cpu()], want.values[0, slots.cpu()]
    tol = norm_tolerance(k, wk, 1e-6, cos, sin, o, dtype, stored=False)
    # half a step at the number's own size, at the scale of its group
    e = quant4.exponents(o, dtype).double().repeat_interleave(32, -1)
    size = torch.frexp((o.abs() * torch.exp2(-e)).clamp(1.0, 6.0))[1].double() - 1
    assert ((x - o).abs() <= torch.exp2(e + size - 2) + tol).all()
    assert (x != y).double().mean() < 1e-3


# ---- as a step uses it


@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_sequence_lives_through_prefill_chunks_and_decodes(dtype, normed):
    """Two sequences prefilled in chunks, then decoded with a third, through the seam on a
    strict pool; every output against attention in 64 bits over the values read back."""
    hq, h, d, bs = 14, 2, 64, 16
    g = gen(16)
    pool = Quant4PagedKVPool(2, 40, bs, h, d, dtype, strict=True)
    tables = [list(range(20, 30)), list(range(3, 13)), list(range(30, 40))]
    wq, wk = (1 + 0.3 * torch.randn(2, d, generator=g, device=DEV)).to(dtype)
    norms = {"q_norm": wq, "k_norm": wk, "eps": 1e-5} if normed else {}
    cached = [0, 0, 0]
    for step in ([40, 3, 0], [1, 60, 0], [33, 1, 9], [1, 1, 1], [1, 1, 1]):
        live = [i for i, n in enumerate(step) if n]
        new, was = [step[i] for i in live], [cached[i] for i in live]
        decode = max(new) == 1
        if decode:
            paged, mask = metadata.decode_context(pool, [tables[i] for i in live], was)
        else:
            paged, mask = metadata.prefill_context(pool, [tables[i] for i in live], was, new)
        b, n = (len(live), 1) if decode else (1, sum(new))
        for layer in range(2):
            q, k, v, cos, sin = step_inputs(g, b, n, hq, h, d, dtype)
            out = rope_paged_attention(q, k, v, cos, sin, paged, mask, layer, d**-0.5, hq // h, **norms)
            # the queries as attended, from the call without attention
            args = (q.reshape(-1, hq, d), k.reshape(-1, h, d), v.reshape(-1, h, d))
            spare = PagedKVPool(1, 40, bs, h, d, dtype)
            cs = (cos.reshape(-1, d), sin.reshape(-1, d))
            if normed:
                qr = kernels.qk_norm_rope_kv_scatter(*args, wq, wk, 1e-5, *cs, spare.k[0], spare.v[0],
                                                     paged.write_slots)
            else:
                qr = kernels.rope_kv_scatter(*args, *cs, spare.k[0], spare.v[0], paged.write_slots)
            values = held(pool, layer)
            row = 0
            for i, m, c in zip(live, new, was):
                o, a, reach = quant.attend(qr[row : row + m], values, tables[i], bs, c, d**-0.5)
                tol = fp32_tolerance(o, a, reach, d) + prefill_tolerance(o, a, reach, dtype)
                tol = tol + small_probabilities(values, tables[i], c + m, bs, hq, dtype)
                err = (out.reshape(-1, hq, d)[row : row + m].double().cpu() - o).abs()
                assert (err <= tol).all(), (step, layer, i)
                row += m
        cached = [c + n for c, n in zip(cached, step)]


def test_seam_writes_then_attends_as_its_parts_do():
    """``paged_attention`` over decode metadata: the write, then the kernels' decode."""
    hq, h, d, bs = 28, 4, 128, 16
    g = gen(17)
    lens = [100, 1, 33, 1100] * 20  # (enough sequences, and keys of a table, for the balanced schedule)
    one, tables, _ = filled(40, torch.bfloat16, lens, h, d, bs)
    two, _, _ = filled(40, torch.bfloat16, lens, h, d, bs)
    paged, mask = metadata.decode_context(one, tables, lens)
    q, k, v, _, _ = step_inputs(g, len(lens), 1, hq, h, d, torch.bfloat16)
    out = paged_attention(q, k, v, paged, mask, 0, d**-0.5, hq // h)
    assert paged.decode_plan is not None
    two.write(0, k[:, 0], v[:, 0], paged.write_slots)
    want = run_decode(two, q[:, 0], paged.block_tables, paged.context_lens, True)
    assert torch.equal(out[:, 0], want) and torch.equal(one.kv_scales, two.kv_scales)
    few = metadata.decode_context(two, tables[:3], lens[:3])[0]
    few.write_slots = torch.full((3,), -1, device=DEV)  # (already written)
    out = paged_attention(q[:3], k[:3], v[:3], few, None, 0, d**-0.5, hq // h)
    want = run_decode(two, q[:3, 0], few.block_tables, few.context_lens, False)
    assert torch.equal(out[:, 0], want)
    at = [i for i, n in enumerate(lens) if n < 1000] * 2  # tables of few keys are not planned
    short = metadata.decode_context(two, [tables[i] for i in at], [lens[i] for i in at])[0]
    short.write_slots = torch.full((len(at),), -1, device=DEV)
    assert len(at) * h >= 256 and not kernels.decode_plan_pays(len(at), hq, h, short.block_tables.shape[1], bs, bits=4)
    out = paged_attention(q[at], k[at], v[at], short, None, 0, d**-0.5, hq // h)
    assert short.decode_plan is None
    want = run_decode(two, q[at, 0], short.block_tables, short.context_lens, False)
    assert torch.equal(out[:, 0], want)


def test_graph_decoder_replays_the_4_bit_step():
    """Decode steps through ``HipGraphDecoder``, several replays with eager work between
    them, each against the same step run eagerly on a copy of the pool."""
    hq, h, d, bs, dtype = 8, 2, 64, 16, torch.bfloat16
    g = gen(18)
    tables = [[0, 1, 2], [3, 4, 5], [6, 7, 8]]
    pools = [Quant4PagedKVPool(2, 9, bs, h, d, dtype) for _ in range(2)]
    fixed = [step_inputs(g, 4, 1, hq, h, d, dtype) for _ in range(2)]
    w = torch.ones(d, device=DEV, dtype=dtype)

    def layers(x, paged):
        outs = []
        for layer in range(2):
            q, k, v, cos, sin = fixed[layer]
            b = x.positions.shape[0]
            shift = (x.positions.view(b, 1, 1, 1) + 1).to(dtype) * 0.125  # (another step, other rows)
            outs.append(rope_paged_attention(q[:b] * shift, k[:b] * shift, v[:b] + shift, cos[:b], sin[:b], paged, None,
                                             layer, d**-0.5, hq // h, q_norm=w, k_norm=w))
        return torch.stack(outs, 1)

    decoder = HipGraphDecoder(None, pools[0], max_num_seqs=4, t_max=48, block_size=bs, step_fn=layers)
    for cached in ([0, 0, 0], [1, 1, 1], [2, 2, 2], [15, 3, 3], [16, 4, 4], [17, 5, 5]):
        got = decoder.decode(tables, cached, [1, 2, 3]).clone()
        x = build_decode_static_inputs(tables, cached, [1, 2, 3], 4, 48, bs, DEV, dtype)
        paged = PagedContext(pools[1], x.write_slots, x.gather_slots, True, x.block_tables, x.context_lens)
        want = layers(x, paged)[:3]
        torch.cuda.synchronize()
        assert torch.equal(got, want), cached
        assert torch.equal(pools[0].kv_scales, pools[1].kv_scales)
        assert torch.equal(pools[0].k, pools[1].k)


@pytest.mark.parametrize("overlap", [False, True])
def test_mixed_step_over_the_4_bit_pool(overlap):
    cfg = MixedConfig("t", 2, 70, 20, 300, 3, 40, 33, 28, 4, 128, 16, torch.bfloat16, seed=2)
    _, plain, batch, inputs = make_mixed_case(cfg, DEV)
    runs = []
    for _ in range(2):
        pool = Quant4PagedKVPool(cfg.num_layers, plain.num_blocks, 16, 4, 128, cfg.dtype)
        slots = torch.arange(pool.num_slots, device=DEV)
        for layer in range(cfg.num_layers):
            pool.write(layer, plain.k[layer], plain.v[layer], slots)
        runs.append(MixedStep(pool, batch, inputs, cfg.scale, overlap=overlap))
    runs[0].eager()
    eager = runs[0].out_dec.clone(), runs[0].out_pre.clone()
    for _ in range(3):
        runs[1].out_dec.zero_()
        runs[1].out_pre.zero_()
        runs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(runs[1].out_dec, eager[0]) and torch.equal(runs[1].out_pre, eager[1])
    for run in runs:
        assert int(run.err.item()) == 0
    values = held(runs[0].pool, 1)
    for i in (0, 69):
        n = int(batch.dec_ctx[i])
        o, a, reach = quant.attend(inputs.q_dec[1, i : i + 1], values, batch.dec_tables[i].tolist(), 16, n - 1,
                                   cfg.scale)
        tol = decode_tolerance(o, a, cfg.dtype) + fp32_tolerance(o, a, reach, 128)
        assert ((eager[0][1, i].double().cpu() - o).abs() <= tol).all()
    o, a, reach = quant.attend(inputs.q_pre[1, 40:80], values, batch.pre_tables[1].tolist(), 16, 33, cfg.scale)
    tol = prefill_tolerance(o, a, reach, cfg.dtype) + fp32_tolerance(o, a, reach, 128)
    assert ((eager[1][1, 40:80].double().cpu() - o).abs() <= tol).all()


def test_one_graph_of_every_call():
    """Writes, normed rotations, reading back and attention in one graph, replayed on other
    inputs with eager work and synchronizations between."""
    hq, h, d, bs, n, dtype = 8, 2, 64, 16, 50, torch.bfloat16
    g = gen(52)
    w = (1 + 0.3 * torch.randn(d, generator=g, device=DEV)).to(dtype)
    slots = torch.arange(n, device=DEV) + 16
    tables = torch.tensor([[1, 2, 3, 4]], dtype=torch.int32, device=DEV)
    ctx = torch.tensor([n], dtype=torch.int32, device=DEV)
    cu, start = torch.tensor([0, n], dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    x = rows(g, n, hq + 2 * h, d, dtype)
    cos, sin = rotation(g, n, d)

    def step(x, pool):
        q, k, v = x.split([hq, h, h], 1)
        pool.write(0, k, v, slots)
        q_out = torch.empty(n, hq, d, device=DEV)
        kernels.rope_kv_scatter_q4(q, k, v, cos, sin, pool.k[1], pool.v[1], pool.kv_scales[1], slots, bs, w, w, 1e-6,
                                   q_out)
        out = torch.empty(n, hq, d, dtype=dtype, device=DEV)
        plan = kernels.prefill_plan(cu, start, tables, n, n, bs, hq, h, d, dtype=dtype)
        kernels.paged_prefill(q_out, pool.k[1], pool.v[1], tables, cu, start, n, bs, d**-0.5, out=out, plan=plan,
                              kv_scales=pool.kv_scales[1])
        decode = kernels.decode_plan(tables, ctx, hq, pool.k[0], bs)
        last = q[-1:].contiguous()
        one = kernels.paged_decode_planned(last, pool.k[0], pool.v[0], decode, d**-0.5, kv_scales=pool.kv_scales[0])
        two = kernels.paged_decode(last, pool.k[0], pool.v[0], tables, ctx, bs, d**-0.5, kv_scales=pool.kv_scales[0])
        return (q_out, out, one, two, *pool.gather(0, slots), *pool.gather_blocks(1, tables, ctx, n))

    static = x.clone()
    mine, other = (Quant4PagedKVPool(2, 6, bs, h, d, dtype) for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static, mine)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(static, mine)
    for i in range(4):
        static.copy_(rows(g, n, hq + 2 * h, d, dtype) * 2.0 ** (3 * i - 4))
        want = [t.clone() for t in step(static, other)]
        graph.replay()
        if i % 2:
            torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), i


def test_layers_on_two_streams():
    """Two layers of a pool written and attended on streams of their own at the same time."""
    hq, h, d, bs, n, dtype = 28, 4, 128, 16, 700, torch.bfloat16
    g = gen(53)
    pools = [Quant4PagedKVPool(2, 50, bs, h, d, dtype) for _ in range(2)]
    data = [rows(g, n, hq + 2 * h, d, dtype).split([hq, h, h], 1) for _ in range(2)]
    slots = torch.randperm(n, generator=g, device=DEV)
    tables = torch.arange(44, dtype=torch.int32, device=DEV)[None]
    cu, start = torch.tensor([0, n], dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    ctx = torch.tensor([n], dtype=torch.int32, device=DEV)

    def run(pool, layer):
        q, k, v = data[layer]
        pool.write(layer, k, v, slots)
        s = pool.kv_scales[layer]
        a = kernels.paged_prefill(q, pool.k[layer], pool.v[layer], tables, cu, start, n, bs, d**-0.5, kv_scales=s)
        one = q[:1].contiguous()
        b = kernels.paged_decode(one, pool.k[layer], pool.v[layer], tables, ctx, bs, d**-0.5, kv_scales=s)
        return a, b, *pool.gather(layer, slots)

    want = [run(pools[0], layer) for layer in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(3):
        for layer, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[layer] = run(pools[1], layer)
    torch.cuda.synchronize()
    for layer in range(2):
        for a, b in zip(got[layer], want[layer]):
            assert torch.equal(a, b)


def test_rows_far_apart():
    """Queries, keys and values whose rows are more than 2^31 elements apart."""
    hq, h, d, bs, dtype = 4, 2, 64, 16, torch.bfloat16
    far = torch.empty(3, (1 << 30) + 64, dtype=dtype, device=DEV)
    g = gen(55)
    x = rows(g, 3, hq + 2 * h, d, dtype)
    far[:, : (hq + 2 * h) * d] = x.flatten(1)
    wide = far[:, : (hq + 2 * h) * d].unflatten(1, (hq + 2 * h, d))
    w = torch.ones(d, dtype=dtype, device=DEV)
    cos, sin = rotation(g, 3, d)
    slots = torch.arange(3, device=DEV)
    outs = []
    for t in (x, wide):
        q, k, v = t.split([hq, h, h], 1)
        pool = Quant4PagedKVPool(2, 1, bs, h, d, dtype)
        pool.write(0, k, v, slots)
        tables = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
        cu = torch.tensor([0, 3], dtype=torch.int32, device=DEV)
        args, sc = (pool.k[0], pool.v[0]), pool.kv_scales[0]
        outs.append([
            kernels.rope_kv_scatter_q4(q, k, v, cos, sin, pool.k[1], pool.v[1], pool.kv_scales[1], slots, bs, w, w,
                                       1e-6).contiguous(),
            kernels.paged_prefill(q, *args, tables, cu, cu[:1], 3, bs, 0.125, kv_scales=sc),
            kernels.paged_decode(q, *args, tables.expand(3, 1).contiguous(), cu[1:].expand(3).contiguous(), bs, 0.125,
                                 kv_scales=sc),
            pool.k, pool.v, pool.kv_scales])
    for a, b in zip(*outs):
        assert torch.equal(a, b)


# ---- refusals


def test_plans_of_another_kind_of_pool_write_nothing():
    """A decode plan built for another kind of layer is refused by the wrapper, and, where
    only the device could know, flagged."""
    h, d, bs, dtype = 2, 64, 16, torch.bfloat16
    pools = [Quant4PagedKVPool(1, 8, bs, h, d, dtype), QuantPagedKVPool(1, 8, bs, h, d, dtype),
             PagedKVPool(1, 8, bs, h, d, dtype)]
    tables = torch.arange(8, dtype=torch.int32, device=DEV).view(2, 4)
    ctx = torch.tensor([60, 33], dtype=torch.int32, device=DEV)
    q = torch.ones(2, 4, d, dtype=dtype, device=DEV)
    for i, mine in enumerate(pools):
        plan = kernels.decode_plan(tables, ctx, 4, mine.k[0], bs)
        for j, other in enumerate(pools):
            if i == j:
                continue
            sc = None if j == 2 else other.kv_scales[0]
            with pytest.raises(RuntimeError, match="plan"):
                kernels.paged_decode_planned(q, other.k[0], other.v[0], plan, 0.1, kv_scales=sc)
            # (the same buffer under another plan's name)
            fields = kernels.decode_plan(tables, ctx, 4, other.k[0], bs)
            fields.buf.copy_(plan.buf[: fields.buf.numel()])
            out = torch.full_like(q, 7.0)
            err = torch.zeros(1, dtype=torch.int32, device=DEV)
            kernels.paged_decode_planned(q, other.k[0], other.v[0], fields, 0.1, out=out, err_flags=err, kv_scales=sc)
            assert int(err) == 16 and (out == 7.0).all()


def test_refusals():
    h, d, bs = 2, 64, 16
    pool = Quant4PagedKVPool(1, 8, bs, h, d, torch.bfloat16)
    x = torch.zeros(1, 1, 4, d, device=DEV, dtype=torch.bfloat16)
    kv = x[:, :, :h]
    paged, mask = metadata.decode_context(pool, [[0, 1]], [5])
    bare = PagedContext(pool, paged.write_slots, paged.gather_slots)
    off = PagedContext(pool, paged.write_slots, paged.gather_slots, False, paged.block_tables, paged.context_lens)
    for p in (bare, off):
        with pytest.raises(RuntimeError, match="a 4-bit pool is attended through block_tables"):
            paged_attention(x, kv + 1, kv + 1, p, mask, 0, 0.1, 2)
    with pytest.raises(RuntimeError, match="4-bit pool's dtype"):
        paged_attention(x.half(), kv.half(), kv.half(), paged, mask, 0, 0.1, 2)
    with pytest.raises(RuntimeError, match="pool's dtype"):
        pool.write(0, kv[0].half(), kv[0].half(), paged.write_slots)
    with pytest.raises(RuntimeError, match="do not match"):
        pool.write(0, x[0], x[0], paged.write_slots)
    with pytest.raises(RuntimeError, match="int64"):
        pool.write(0, kv[0], kv[0], paged.write_slots.int())
    assert not pool.k.any() and not pool.v.any()
    q = x[0]
    args = (paged.block_tables, paged.context_lens, bs, 0.1)
    scales = pool.kv_scales[0]
    for s in (scales[:, :4], scales.double(), scales.transpose(0, 1)):
        with pytest.raises(RuntimeError, match="kv_scales"):
            kernels.paged_decode(q, pool.k[0], pool.v[0], *args, kv_scales=s)
    loose = pool.k[0].contiguous()
    with pytest.raises(RuntimeError, match="dense"):
        kernels.paged_decode(q, loose, loose, *args, kv_scales=scales)
    with pytest.raises(RuntimeError, match="whole blocks"):
        kernels.paged_decode(q, pool.k[0], pool.v[0], paged.block_tables, paged.context_lens, 48, 0.1,
                             kv_scales=scales)
    with pytest.raises(RuntimeError, match="mismatch"):
        kernels.paged_decode(q, pool.k[0], pool.v[0], *args)
    with pytest.raises(RuntimeError, match="out must be"):
        kernels.paged_decode(q, pool.k[0], pool.v[0], *args, out=q.float(), kv_scales=scales)
    cu = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="a 4-bit cache"):
        kernels.paged_prefill(q, pool.k[0], pool.v[0], paged.block_tables, cu, paged.context_lens, 1, bs, 0.1,
                              new_kv=(kv[0], kv[0], paged.write_slots), kv_scales=scales)
    cs, rows3 = torch.zeros(1, d, device=DEV), (q, kv[0], kv[0])
    with pytest.raises(RuntimeError, match="4-bit pool"):
        kernels.rope_kv_scatter_q8(*rows3, cs, cs, pool.k[0], pool.v[0], scales, paged.write_slots, bs)
    eight = QuantPagedKVPool(1, 8, bs, h, d, torch.bfloat16)
    with pytest.raises(RuntimeError, match="uint8"):
        kernels.rope_kv_scatter_q4(*rows3, cs, cs, eight.k[0], eight.v[0], eight.kv_scales[0], paged.write_slots, bs)
    with pytest.raises(RuntimeError, match="codes"):
        kernels.paged_decode(q, eight.k[0], eight.v[0], *args, kv_scales=torch.zeros(h, 8, d, dtype=torch.uint8,
                                                                                    device=DEV))
    with pytest.raises(RuntimeError, match="codes"):
        kernels.kv_scatter_q8(pool.k[0], pool.v[0], scales, *rows3[1:], paged.write_slots, bs)
    with pytest.raises(RuntimeError, match="codes|kv_scales"):
        kernels.kv_scatter_q4(eight.k[0], eight.v[0], eight.kv_scales[0], *rows3[1:], paged.write_slots, bs)
    with pytest.raises(RuntimeError, match="kv_scales"):
        kernels.paged_gather_q4(pool.k[0], pool.v[0], scales[:, :2], *args[:2], bs, 4, torch.bfloat16)
    torch.cuda.synchronize()


@pytest.mark.parametrize("n, spread", [(1025, 300), (1025, 1025), (2048, 1), (2049, 700), (5000, 4000), (8193, 8000), (20001, 9000)])
@pytest.mark.parametrize("d", [64, 128])
def test_the_last_of_equal_slots_is_written_in_calls_of_any_length(n, spread, d):
    """Rows that differ, their slots up to a whole call apart; skipped ones and one out of range between
    them. Plain, rotated, normed and turned by axes."""
    h, bs, dtype = 2, 16, torch.bfloat16
    g = gen(n + d)
    q, k, v = rows(g, n, 2 * h, d, dtype), rows(g, n, h, d, dtype, 3.0), rows(g, n, h, d, dtype, 3.0)
    slots = torch.randint(0, spread, (n,), generator=g, device=DEV)
    slots[n // 3], slots[n // 2] = -1, 2**31 + int(slots[5])
    slots[n - 1] = slots[0]
    blocks = spread // bs + 2
    valid = slots.clone()
    valid[valid >= blocks * bs] = -1
    last = {s: i for i, s in enumerate(valid.tolist()) if s >= 0}
    at = torch.tensor(sorted(last.values()), device=DEV)
    pool, want = (Quant4PagedKVPool(1, blocks, bs, h, d, dtype) for _ in range(2))
    held_values = quant4.Quant4Cache(blocks * bs, h, d, dtype)
    pool.write(0, k, v, slots)
    with pytest.raises(IndexError, match="write slot"):
        pool.check_errors()
    held_values.write(k[at], v[at], slots[at])
    assert same(held(pool), held_values.values)
    cos, sin = rotation(g, n, d)
    w = (1 + 0.3 * torch.randn(2, d, generator=g, device=DEV)).to(dtype)
    rotary = RotaryAxes.sections(d, (d // 4, d // 4))
    pos = torch.randint(0, 9999, (2, n), generator=g, device=DEV)
    for norms in ((), (w[0], w[1], 1e-6)):
        for axes in (False, True):
            out = []
            for p, i in ((pool, slice(None)), (want, at)):
                p.k.zero_(), p.v.zero_(), p.kv_scales.fill_(27)
                layer = (p.k[0], p.v[0])
                if axes:
                    out.append(kernels.rope_axes_kv_scatter(q[i], k[i], v[i], pos[:, i], rotary, *layer, slots[i], *norms,
                                                            kv_scales=p.kv_scales[0], block_size=bs))
                else:
                    out.append(kernels.rope_kv_scatter_q4(q[i], k[i], v[i], cos[i], sin[i], *layer, p.kv_scales[0],
                                                          slots[i], bs, *norms))
            case = (bool(norms), axes)
            assert torch.equal(pool.k, want.k) and torch.equal(pool.v, want.v), case
            assert torch.equal(pool.kv_scales, want.kv_scales) and torch.equal(out[0][at], out[1]), case


def test_refusals_name_the_rows_that_are_not_contiguous():
    n, h, d, bs = 3, 2, 64, 16
    even = torch.zeros(n, h, d, dtype=torch.bfloat16, device=DEV)
    odd = torch.zeros(n, h, 2 * d, dtype=torch.bfloat16, device=DEV)[:, :, ::2]
    slots, cs = torch.arange(n, device=DEV), torch.zeros(n, d, device=DEV)
    rotary, pos = RotaryAxes.sections(d, (d // 2,)), torch.arange(n, device=DEV)
    four, eight = (p(1, 2, bs, h, d, torch.bfloat16) for p in (Quant4PagedKVPool, QuantPagedKVPool))
    layers = [(p.k[0], p.v[0], p.kv_scales[0]) for p in (four, eight)]
    for which in range(3):
        q, k, v = (odd if i == which else even for i in range(3))
        bad = f" {'qkv'[which]}: the last"
        for layer, write, rope in zip(layers, (kernels.kv_scatter_q4, kernels.kv_scatter_q8),
                                      (kernels.rope_kv_scatter_q4, kernels.rope_kv_scatter_q8)):
            if which:
                with pytest.raises(RuntimeError, match=write.__name__ + bad):
                    write(*layer, k, v, slots, bs)
            with pytest.raises(RuntimeError, match=rope.__name__ + bad):
                rope(q, k, v, cs, cs, *layer, slots, bs)
        with pytest.raises(RuntimeError, match="rope_axes_kv_scatter" + bad):
            kernels.rope_axes_kv_scatter(q, k, v, pos, rotary, *layers[0][:2], slots, kv_scales=layers[0][2],
                                         block_size=bs)
        if which < 2:
            with pytest.raises(RuntimeError, match="rope_axes" + bad):
                kernels.rope_axes(q, k, pos, rotary)
    assert not four.k.any() and not eight.k.view(torch.uint8).any()


@pytest.mark.parametrize("pool_type, dtype, bits", [
    (PagedKVPool, torch.bfloat16, 16), (PagedKVPool, torch.float32, 32),
    (QuantPagedKVPool, torch.bfloat16, 8), (Quant4PagedKVPool, torch.bfloat16, 4),
])
@pytest.mark.parametrize("seqs, keys", [(64, 304), (64, 1024), (64, 1040), (8, 1024), (3, 9008)])
def test_the_seam_plans_what_pays_over_a_pool_of_its_bits(pool_type, dtype, bits, seqs, keys):
    hq, h, d, bs = 14, 2, 64, 16
    width = keys // bs
    pool = pool_type(1, width, bs, h, d, dtype)
    assert pool.bits == bits
    paged, mask = metadata.decode_context(pool, [list(range(width))] * seqs, [keys - 1] * seqs)
    q, k, v, _, _ = step_inputs(gen(seqs), seqs, 1, hq, h, d, dtype)
    paged_attention(q, k, v, paged, mask, 0, d**-0.5, hq // h)
    assert paged.block_tables.shape[1] == width
    assert (paged.decode_plan is not None) == kernels.decode_plan_pays(seqs, hq, h, width, bs, DEV, pool.bits)


# The queries that a step attends with are fp32 ones, off by turn_tolerance from the 64-bit rotation's: a
# score by delta = scale sum |that| |k|, an output by (e^(2 delta) - 1) a, delta < 0.01: 2.1 delta a. Their two
# pieces of the dtype leave 2^-18 of an element at most, which comes in the same way.
@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_step_turned_by_axes_over_the_4_bit_pool_is_attention_in_64_bits(dtype, normed):
    """Prompt chunks, then single tokens, of sequences two of which begin alike, through the seam."""
    hq, h, d, bs, scale = 14, 2, 64, 16, 0.125
    g = gen(50)
    rotary = RotaryAxes.sections(d, (8, 12, 12), scaling=0.9)
    pool = Quant4PagedKVPool(1, 40, bs, h, d, dtype)
    tables = [[20, 3, 7, 30, 31, 32], [20, 3, 8, 33, 34, 35], [1, 2, 36], [9, 10, 11]]
    w = (1 + 0.3 * torch.randn(2, d, generator=g, device=DEV)).to(dtype)
    norms = {"q_norm": w[0], "k_norm": w[1], "eps": 1e-5} if normed else {}
    cached = [0, 32, 0, 0]
    for new in ([70, 41, 1, 20], [1, 1, 30, 9], [1, 1, 1, 1], [1, 1, 1, 1]):
        total, decode = sum(new), max(new) == 1
        b, sq = (total, 1) if decode else (1, total)
        q, k, v = rows(g, total, hq + 2 * h, d, dtype, 0.7).view(b, sq, -1, d).split([hq, h, h], 2)
        pos = positions(g, 3, total).view(3, b, sq)
        paged, mask = (metadata.decode_context(pool, tables, cached) if decode
                       else metadata.prefill_context(pool, tables, cached, new))
        out = rope_axes_paged_attention(q, k, v, pos, rotary, paged, mask, 0, scale, hq // h, **norms)
        assert out.dtype == dtype
        pool.check_errors()
        values = held(pool)
        flat, weight, eps = q.reshape(-1, hq, d), (w[0] if normed else None), (1e-5 if normed else 0.0)
        turned = quant4.turn(flat, pos.view(3, -1), rotary.inv_freq, rotary.axis_of, weight, eps, rotary.scaling)
        off = turn_tolerance(flat, turned, torch.float32, weight, eps, rotary.scaling)
        row = 0
        for table, c, n in zip(tables, cached, new):
            at = slice(row, row + n)
            o, a, reach = quant.attend(turned[at], values, table, bs, c, scale)
            delta = quant.attend(off[at], values, table, bs, c, scale)[2] + 2.0**-18 * reach
            assert delta.max() < 0.01
            tol = fp32_tolerance(o, a, reach, d) + 2.1 * delta[..., None] * a
            tol = tol + small_probabilities(values, table, c + n, bs, hq, dtype)
            if dtype != torch.float32:
                tol = tol + (decode_tolerance(o, a, dtype) if decode else prefill_tolerance(o, a, reach, dtype))
            err = (out.reshape(-1, hq, d)[at].double().cpu() - o).abs()
            assert (err <= tol).all(), (new, c, (err / tol).max())
            row += n
        cached = [c + n for c, n in zip(cached, new)]


# Whole numbers of queries and keys, times powers of two, so that scores are exact in fp32 and the largest is
# ahead of the next by more than any exponential holds: the answer is the mean of the V of the keys that have it,
# rounded (V's sums of a few codes are exact too).
@pytest.mark.parametrize("path, sign", [("decode", 1), ("decode", -1), ("planned", 1), ("planned", -1), ("prefill", 1)])
@pytest.mark.parametrize("dtype, q_dtype, q_exp, scale_exp", [
    (dtype, q_dtype, q_exp, scale_exp)
    for dtype in DTYPES
    for q_dtype in sorted({dtype, torch.float32}, key=str)
    for q_exp, scale_exp in ((0, 100), (0, 12), (100, -3), (40, 0))
    if q_exp == 0 or q_dtype != torch.float16
])
def test_scores_of_any_size(path, sign, dtype, q_dtype, q_exp, scale_exp):
    bs, hq, h, d, lens = 16, 6, 2, 64, [700, 33, 1]
    g = gen(60)
    codes = torch.tensor(quant4.CODES, device=DEV)
    pool = Quant4PagedKVPool(1, 50, bs, h, d, dtype)
    tables = [list(range(44)), [44, 45, 46], [47]]
    k, v = ((codes[torch.randint(0, 8, (2, 800, h, d), generator=g, device=DEV)]
             * (2 * torch.randint(0, 2, (2, 800, h, d), generator=g, device=DEV) - 1)).to(dtype))
    k[:, :, ::32] = v[:, :, ::32] = 6.0  # (every group's scale is 1)
    pool.write(0, k, v, torch.arange(800, device=DEV))
    whole = torch.randint(-3, 4, (len(lens), hq, d), generator=g, device=DEV).double()
    q, scale = (whole * 2.0**q_exp).to(q_dtype), sign * 2.0**scale_exp
    bt, ctx = device_tables(tables), torch.tensor(lens, dtype=torch.int32, device=DEV)
    kw = {"out": torch.empty(len(lens), hq, d, dtype=dtype, device=DEV), "kv_scales": pool.kv_scales[0]}
    layer = (pool.k[0], pool.v[0])
    if path == "decode":
        out = kernels.paged_decode(q, *layer, bt, ctx, bs, scale, **kw)
    elif path == "planned":
        out = kernels.paged_decode_planned(q, *layer, kernels.decode_plan(bt, ctx, hq, pool.k[0], bs), scale, **kw)
    else:
        cu = torch.arange(len(lens) + 1, dtype=torch.int32, device=DEV)
        out = kernels.paged_prefill(q, *layer, bt, cu, ctx - 1, 1, bs, scale, **kw)
    for i, (table, n) in enumerate(zip(tables, lens)):
        for head in range(hq):
            at = slice(table[0] * bs, table[0] * bs + n)
            s = sign * (k[at, head // 3].double() @ whole[i, head])
            want = v[at, head // 3][s == s.max()].double().mean(0)
            err = (out[i, head].double() - want).abs()
            assert (err <= torch.finfo(dtype).eps / 2 * want.abs() + 2.0**-20).all(), (i, head, err.max())


def test_a_graph_of_a_long_write_replays():
    """A call of several launches, its slots repeated across them and changed between replays."""
    n, h, d, bs, dtype = 17000, 2, 64, 16, torch.bfloat16
    g = gen(70)
    mine, other = (Quant4PagedKVPool(1, 600, bs, h, d, dtype) for _ in range(2))
    k, v, slots = rows(g, n, h, d, dtype), rows(g, n, h, d, dtype), torch.arange(n, device=DEV) % mine.num_slots
    mine.write(0, k, v, slots)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mine.write(0, k, v, slots)
    for i in range(4):
        k.copy_(rows(g, n, h, d, dtype)), v.copy_(rows(g, n, h, d, dtype))
        slots.copy_(torch.randint(-1, mine.num_slots, (n,), generator=g, device=DEV))
        other.k.copy_(mine.k), other.v.copy_(mine.v), other.kv_scales.copy_(mine.kv_scales)
        other.write(0, k, v, slots)
        graph.replay()
        if i % 2:
            torch.cuda.synchronize()
        assert torch.equal(mine.k, other.k) and torch.equal(mine.v, other.v)
        assert torch.equal(mine.kv_scales, other.kv_scales), i
