"""The 8-bit pool on the GPU against its definition in 64 bits: the quantising write and
reading back exactly, attention and the normed rotation within bounds derived from
their roundings, and all of them together as a step uses them."""

from __future__ import annotations

import pytest
import torch

from infrared_amd import (
    PagedContext,
    PagedKVPool,
    QuantPagedKVPool,
    kernels,
    metadata,
    paged_attention,
    rope_paged_attention,
)
from infrared_amd.hip_graph import HipGraphDecoder, build_decode_static_inputs
from infrared_amd.mixed_step import MixedConfig, MixedStep, make_mixed_case
from oracle import quant

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
DEV = "cuda"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def rows(g, n, h, d, dtype, spread=1.0):
    """Rows whose magnitudes differ from token to token and channel to channel."""
    x = torch.randn(n, h, d, generator=g, device=DEV)
    x = x * torch.exp(spread * torch.randn(n, h, 1, generator=g, device=DEV))
    return (x * torch.exp(0.5 * torch.randn(d, generator=g, device=DEV))).to(dtype)


def same(a, b):
    """Equal values, NaN where NaN."""
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(torch.nan_to_num(a, nan=0.0), torch.nan_to_num(b, nan=0.0))


def check_cache(pool, want, layer=0):
    """The pool's scales, codes and values against the oracle's, bit for bit."""
    assert torch.equal(pool.kv_scales[layer].double().cpu(), torch.exp2(want.exps.double()))
    slots = torch.arange(pool.num_slots, device=DEV)
    k, v = pool.gather(layer, slots)
    assert k.dtype == pool.dtype
    assert same(torch.stack([k, v]).double().cpu(), want.values)


# ---- reading


@pytest.mark.parametrize("dtype", DTYPES)
def test_reads_every_code_at_every_scale(dtype):
    lo, hi, most = quant.BOUNDS[dtype]
    blocks = hi - lo + 1
    pool = QuantPagedKVPool(1, blocks, 16, 1, 64, dtype)
    codes = torch.arange(256, dtype=torch.uint8, device=DEV).repeat(4).view(torch.float8_e4m3fn)
    for cache in (pool.k, pool.v):
        cache[0] = codes.view(1, 16, 1, 64).expand(blocks, 16, 1, 64).reshape(blocks * 16, 1, 64)
    exps = torch.arange(lo, hi + 1, device=DEV)
    pool.kv_scales[0, 0, :, 0] = torch.exp2(exps.double()).float()
    pool.kv_scales[0, 0, :, 1] = torch.exp2(exps.flip(0).double()).float()
    k, v = pool.gather(0, torch.arange(blocks * 16, device=DEV))
    for got, e in ((k, exps), (v, exps.flip(0))):
        want = codes.double().view(1, -1) * torch.exp2(e.double())[:, None]
        got = got.double().view(blocks, -1)
        inside = ~(want.abs() > most)  # (codes past the dtype's range are never written)
        assert same(torch.where(inside, got, 0.0).cpu(), torch.where(inside, want, 0.0).cpu())


def test_reads_through_tables_and_flags_bad_slots():
    pool = QuantPagedKVPool(2, 12, 16, 3, 64, torch.bfloat16)
    g = gen(1)
    slots = torch.arange(pool.num_slots, device=DEV)
    pool.write(1, rows(g, pool.num_slots, 3, 64, torch.bfloat16), rows(g, pool.num_slots, 3, 64, torch.bfloat16), slots)
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
    assert pool.gather(1, bad[:0])[0].shape == (0, 2, 3, 64)


# ---- writing


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d, h, bs", [(128, 4, 16), (64, 2, 16), (64, 3, 32), (128, 1, 48), (64, 5, 256)])
def test_write_fills_blocks_in_order(dtype, d, h, bs):
    """Chunks that begin and end inside blocks, whole blocks, single tokens; the scales of
    kept tokens grow."""
    pool = QuantPagedKVPool(1, 9, bs, h, d, dtype, strict=True)
    want = quant.QuantCache(9, bs, h, d, dtype)
    g = gen(d + h + bs)
    table = [4, 8, 1, 0, 6]
    at = 0
    for n in (1, 1, 3, bs - 2, 2, 2 * bs, 1, 7):
        pos = range(at, at + n)
        slots = torch.tensor([table[p // bs] * bs + p % bs for p in pos], device=DEV)
        k, v = rows(g, n, h, d, dtype), rows(g, n, h, d, dtype, spread=3.0)
        pool.write(0, k, v, slots)
        want.write(k, v, slots)
        at += n
    check_cache(pool, want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_write_takes_tokens_in_any_order(dtype):
    """Shuffled slots, slots given twice (the last row is written), negative ones and
    slots past the pool, over blocks that hold tokens already."""
    bs, h, d, blocks = 16, 2, 64, 24
    pool = QuantPagedKVPool(1, blocks, bs, h, d, dtype)
    want = quant.QuantCache(blocks, bs, h, d, dtype)
    g = gen(3)
    total = blocks * bs
    for n in (total, 200, 1000):
        slots = torch.randint(-20, total + 20, (n,), generator=g, device=DEV)
        k, v = rows(g, n, h, d, dtype, 2.0), rows(g, n, h, d, dtype)
        pool.write(0, k, v, slots)
        want.write(k, v, slots)
        check_cache(pool, want)
        with pytest.raises(IndexError, match="write slot"):
            pool.check_errors()


@pytest.mark.parametrize("d, h, bs, n", [(64, 64, 16, 700), (128, 64, 48, 900), (64, 65, 1024, 1300)])
def test_write_of_long_calls(d, h, bs, n):
    """Calls whose workgroups share the reading of the slots (many heads make a call long):
    shuffled tokens, slots given twice, skipped and past the pool; then in order, over
    blocks that hold tokens already."""
    g, blocks, dtype = gen(d + bs), max(4, 1000 // bs), torch.bfloat16
    pool, want = QuantPagedKVPool(1, blocks, bs, h, d, dtype), quant.QuantCache(blocks, bs, h, d, dtype)
    slots = torch.randint(0, pool.num_slots, (n,), generator=g, device=DEV)
    slots[::17] = -1
    slots[5] = pool.num_slots
    k, v = rows(g, n, h, d, dtype), rows(g, n, h, d, dtype)
    pool.write(0, k, v, slots)
    with pytest.raises(IndexError, match="slot"):
        pool.check_errors()
    want.write(k, v, slots)
    check_cache(pool, want)
    m = min(n, pool.num_slots - 7)
    k, v = rows(g, m, h, d, dtype) * 4, rows(g, m, h, d, dtype) * 4
    pool.write(0, k, v, torch.arange(7, 7 + m, device=DEV))
    want.write(k, v, torch.arange(7, 7 + m))
    pool.check_errors()
    check_cache(pool, want)


def test_a_fresh_block_owes_nothing_to_what_it_held():
    pool = QuantPagedKVPool(1, 2, 16, 2, 64, torch.bfloat16)
    g = gen(4)
    slots = torch.arange(16, device=DEV)
    big = 1e6 * rows(g, 16, 2, 64, torch.bfloat16)
    pool.write(0, big, big, slots)
    k = rows(g, 5, 2, 64, torch.bfloat16)
    pool.write(0, k, k, slots[:5])
    want = quant.QuantCache(2, 16, 2, 64, torch.bfloat16)
    want.write(k, k, slots[:5])
    check_cache(pool, want)  # (the other eleven tokens are zero)


@pytest.mark.parametrize("dtype", DTYPES)
def test_write_of_extreme_numbers(dtype):
    """Zeros, the type's largest and smallest numbers, NaN and infinities, a block whose
    scale takes the largest step there is."""
    bs, h, d = 16, 1, 64
    f = torch.finfo(dtype)
    pool = QuantPagedKVPool(1, 8, bs, h, d, dtype)
    want = quant.QuantCache(8, bs, h, d, dtype)
    g = gen(5)

    def put(x, slots):
        x = x.to(dtype).view(-1, h, d)
        slots = torch.tensor(slots, device=DEV)
        pool.write(0, x, -x, slots)
        want.write(x, -x, slots)
        check_cache(pool, want)

    put(torch.zeros(3 * d, device=DEV), [0, 1, 2])
    ramp = torch.linspace(-1, 1, d, device=DEV, dtype=torch.float64)
    put(f.max * ramp, [16])
    put(f.max * ramp.flip(0) / 3, [17])
    put(f.smallest_normal * 64 * ramp, [32])  # least scale, then the largest
    put(f.max * ramp, [33])
    odd = torch.randn(d, generator=g, device=DEV)
    odd[3], odd[9], odd[20] = float("nan"), float("inf"), float("-inf")
    put(odd, [48])
    put(torch.randn(d, generator=g, device=DEV) * 100, [49])  # NaN codes stay as the scale grows
    put(torch.full((d,), float("nan"), device=DEV), [64])
    # both sides of the border where the scale steps, and of ties between codes
    edge = torch.tensor([448.0, 449.0, 447.0, 1.0625, 1.1875, 232.0, 240.0, 0.0009765625], device=DEV).repeat(8)
    put(edge, [80])
    put(edge * 0 + 448.0, [96])


def test_write_reads_strided_rows_and_runs_on_the_current_stream():
    bs, h, d, n = 16, 4, 128, 37
    pool = QuantPagedKVPool(3, 8, bs, h, d, torch.bfloat16)
    want = quant.QuantCache(8, bs, h, d, torch.bfloat16)
    qkv = rows(gen(6), n, 3 * h, d, torch.bfloat16)
    slots = torch.arange(60, 60 + n, device=DEV)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        pool.write(2, qkv[:, h : 2 * h], qkv[:, 2 * h :], torch.stack([slots, slots], 1)[:, 1])
    torch.cuda.current_stream().wait_stream(stream)
    want.write(qkv[:, h : 2 * h], qkv[:, 2 * h :], slots)
    check_cache(pool, want, layer=2)
    assert not pool.k[:2].view(torch.uint8).any()


def test_pool_over_four_gigabytes():
    """Codes whose offsets pass 32 bits: the last blocks of a 4.3 GB layer."""
    blocks, bs, h, d = (1 << 17) + 64, 64, 4, 128
    pool = QuantPagedKVPool(1, blocks, bs, h, d, torch.bfloat16)
    assert pool.k[0].numel() > 1 << 32
    g = gen(7)
    ids = [blocks - 1, 3, blocks - 2]
    n = 150
    slots = torch.tensor([ids[p // bs] * bs + p % bs for p in range(n)], device=DEV)
    k, v = rows(g, n, h, d, torch.bfloat16), rows(g, n, h, d, torch.bfloat16)
    pool.write(0, k, v, slots)
    small = quant.QuantCache(3, bs, h, d, torch.bfloat16)
    small.write(k, v, torch.arange(n))
    gk, gv = pool.gather(0, slots)
    assert torch.equal(torch.stack([gk, gv]).double().cpu(), small.values[:, :n])
    q = torch.randn(1, 8, d, generator=g, device=DEV).bfloat16()
    tables = torch.tensor([ids], dtype=torch.int32, device=DEV)
    ctx = torch.tensor([n], dtype=torch.int32, device=DEV)
    out = kernels.paged_decode(q, pool.k[0], pool.v[0], tables, ctx, bs, d**-0.5, kv_scales=pool.kv_scales[0])
    o, a, _ = quant.attend(q, small.values, [0, 1, 2], bs, n - 1, d**-0.5)
    assert ((out.double().cpu() - o).abs() <= decode_tolerance(o, a, torch.bfloat16)).all()
    cu = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    out = kernels.paged_prefill(q, pool.k[0], pool.v[0], tables, cu, ctx - 1, 1, bs, d**-0.5,
                                kv_scales=pool.kv_scales[0])
    o, a, reach = quant.attend(q, small.values, [0, 1, 2], bs, n - 1, d**-0.5)
    assert ((out.double().cpu() - o).abs() <= prefill_tolerance(o, a, reach, torch.bfloat16)).all()


# ---- attention
#
# Of an output o = sum p v / sum p, with a = sum p |v| / sum p and u half a step of the
# dtype: the decode rounds each p (u a) and the output (u |o|); fp32 sums, exponentials
# and the merges of parts add a few hundred steps of 2^-24 of a. The prefill also
# rounds the query times scale * log2 e: scores move by at most u * reach, reach =
# scale * sum |q k|, which moves o by at most 2 * u * reach * 2 a. In fp32 what is left
# are the fp32 sums: a score is off by at most (d + 8) 2^-24 reach.


def decode_tolerance(o, a, dtype):
    u = torch.finfo(dtype).eps / 2
    return u * (a + o.abs()) * 1.02 + 500 * 2.0**-24 * a


def prefill_tolerance(o, a, reach, dtype):
    u = torch.finfo(dtype).eps / 2
    return decode_tolerance(o, a, dtype) + 4 * u * reach[..., None] * a


def fp32_tolerance(o, a, reach, d):
    return 2.0**-24 * (500 * a + o.abs() + 4 * (d + 8) * reach[..., None] * a)


def filled(seed, dtype, lens, h, d, bs, spare=3):
    """A pool whose sequences of ``lens`` tokens were written, the rest of it poisoned: NaN
    codes, infinite scales in unused blocks, and NaN in the unwritten tokens of used ones."""
    g = gen(seed)
    need = [max(1, -(-n // bs)) for n in lens]
    blocks = sum(need) + spare
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).tolist()
    tables = [[order.pop() for _ in range(n)] for n in need]
    pool = QuantPagedKVPool(1, blocks, bs, h, d, dtype)
    slots = torch.tensor([metadata.slot(t, p, bs) for t, n in zip(tables, lens) for p in range(n)],
                         dtype=torch.long, device=DEV)
    total = len(slots)
    k, v = rows(g, total, h, d, dtype, 0.5), rows(g, total, h, d, dtype)
    pool.write(0, k, v, slots)
    values = torch.stack(pool.gather(0, torch.arange(pool.num_slots, device=DEV))).double().cpu()
    unused = torch.ones(pool.num_slots, dtype=torch.bool, device=DEV)
    unused[slots] = False
    for cache in (pool.k, pool.v):
        raw = cache[0].view(torch.uint8)
        raw[unused] = 0x7F
    for b in order:
        pool.kv_scales[0, :, b] = float("inf")
    return pool, tables, values


def device_tables(tables, width=None):
    return metadata.block_tables_tensor(tables, DEV, width)


def run_decode(pool, q, bt, ctx, planned, **kw):
    h, bs = pool.num_kv_heads, pool.block_size
    if not planned:
        return kernels.paged_decode(q, pool.k[0], pool.v[0], bt, ctx, bs, q.shape[2] ** -0.5, err_flags=pool.err_flags,
                                    kv_scales=pool.kv_scales[0], **kw)
    plan = kernels.decode_plan(bt, ctx, q.shape[1], pool.k[0], bs, err_flags=pool.err_flags, share_groups=True)
    return kernels.paged_decode_planned(q, pool.k[0], pool.v[0], plan, q.shape[2] ** -0.5, err_flags=pool.err_flags,
                                        kv_scales=pool.kv_scales[0], **kw)


@pytest.mark.parametrize("planned", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq, h, d, bs", [(28, 4, 128, 16), (14, 2, 64, 16), (8, 8, 64, 32), (20, 1, 128, 48),
                                          (3, 3, 128, 128), (33, 1, 64, 16)])
def test_decode(planned, dtype, hq, h, d, bs):
    lens = [1, 2, 15, 16, 17, 33, 300, 1100, 64, 0, 5]
    pool, tables, values = filled(hq + d, dtype, lens, h, d, bs)
    q = torch.randn(len(lens), hq, d, generator=gen(9), device=DEV).to(dtype)
    ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = run_decode(pool, q, device_tables(tables), ctx, planned)
    pool.check_errors()
    for i, n in enumerate(lens):
        if n == 0:
            assert not out[i].any()
            continue
        o, a, reach = quant.attend(q[i : i + 1], values, tables[i], bs, n - 1, d**-0.5)
        tol = fp32_tolerance(o, a, reach, d) if dtype == torch.float32 else (
            decode_tolerance(o, a, dtype) + 4 * (d + 8) * 2.0**-24 * reach[..., None] * a)
        err = (out[i : i + 1].double().cpu() - o).abs()
        assert (err <= tol).all(), (i, n, (err / tol).max())


@pytest.mark.parametrize("planned", [False, True])
def test_decode_of_long_contexts_and_shared_prefixes(planned):
    """Contexts cut into parts, pairs of sequences whose tables begin alike."""
    bs, hq, h, d = 16, 28, 4, 128
    lens = [9000, 700, 4097, 2500]
    pool, tables, values = filled(21, torch.bfloat16, lens, h, d, bs)
    tables.append(tables[3][:100] + tables[1][:20])
    tables.append(tables[3][:100] + tables[0][:7])
    lens = lens + [1600 + 311, 1600 + 112]
    q = torch.randn(len(lens), hq, d, generator=gen(10), device=DEV).bfloat16()
    ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
    bt = device_tables(tables)
    out = run_decode(pool, q, bt, ctx, planned)
    pool.check_errors()
    for i, n in enumerate(lens):
        o, a, reach = quant.attend(q[i : i + 1], values, tables[i], bs, n - 1, d**-0.5)
        tol = decode_tolerance(o, a, torch.bfloat16) + 4 * (d + 8) * 2.0**-24 * reach[..., None] * a
        err = (out[i : i + 1].double().cpu() - o).abs()
        assert (err <= tol).all(), (i, n, (err / tol).max())
    assert torch.equal(out, run_decode(pool, q, bt, ctx, planned))  # nothing of a call is left for the next


@pytest.mark.parametrize("dtype, hq, h, d, lens", [
    (torch.bfloat16, 28, 4, 128, [20011]), (torch.float16, 14, 2, 64, [9000, 0, 17]),
    (torch.float32, 6, 2, 128, [5000]),
    (torch.bfloat16, 40, 2, 64, [8191, 4000]), (torch.bfloat16, 8, 1, 128, [300, 1, 0]),
])
def test_decode_of_few_sequences_over_many_slices(dtype, hq, h, d, lens):
    """Few units, whose partial rows a launch of their own merges: groups of more than 16
    query heads, an empty sequence, and the same with a sequence that shares a prefix."""
    bs = 16
    pool, tables, values = filled(23, dtype, lens, h, d, bs)
    if lens[0] > 1000:
        tables.append(tables[0][:200])
        lens = lens + [200 * bs - 3]
        tables, lens = [tables[0], tables[-1], *tables[1:-1]], [lens[0], lens[-1], *lens[1:-1]]
    assert len(lens) * h * -(-hq // h // 16) * 12 <= 256
    q = torch.randn(len(lens), hq, d, generator=gen(10), device=DEV).to(dtype)
    ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
    bt = device_tables(tables)
    out = run_decode(pool, q, bt, ctx, True)
    pool.check_errors()
    for i, n in enumerate(lens):
        if n == 0:
            assert not out[i].any()
            continue
        o, a, reach = quant.attend(q[i : i + 1], values, tables[i], bs, n - 1, d**-0.5)
        tol = fp32_tolerance(o, a, reach, d) if dtype == torch.float32 else (
            decode_tolerance(o, a, dtype) + 4 * (d + 8) * 2.0**-24 * reach[..., None] * a)
        err = (out[i : i + 1].double().cpu() - o).abs()
        assert (err <= tol).all(), (i, n, (err / tol).max())
    assert torch.equal(out, run_decode(pool, q, bt, ctx, True))


@pytest.mark.parametrize("planned", [False, True])
def test_decode_masks_bad_blocks_and_lengths(planned):
    bs, hq, h, d = 16, 8, 2, 64
    pool, tables, values = filled(22, torch.bfloat16, [100, 50], h, d, bs)
    bt = device_tables(tables)
    q = torch.randn(2, hq, d, generator=gen(11), device=DEV).bfloat16()
    ctx = torch.tensor([100, 50], dtype=torch.int32, device=DEV)
    want = run_decode(pool, q, bt, ctx, planned)
    bt[0, 2] = pool.num_blocks
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
            tol = fp32_tolerance(o, a, reach, d)
            if dtype != torch.float32:
                tol = tol + prefill_tolerance(o, a, reach, dtype)
            err = (out[row : row + n].double().cpu() - o).abs()
            assert (err <= tol).all(), (c, n, (err / tol).max())
        row += n


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
    tol = fp32_tolerance(o, a, reach, d)
    if dtype != torch.float32:
        tol = tol + prefill_tolerance(o, a, reach, dtype)
    out = out.double().cpu()
    assert ((out - o).abs() <= tol)[~spoiled].all()
    assert out[spoiled].isnan().any(-1).all()


# Scores of some hundred: what is lost of them is lost of every probability. In the mean over
# many outputs a rounding to nearest is off by at most u / sqrt(3) of a number, and the
# probabilities and the output are rounded once each: sqrt(2 / 3) u, and 10% for the fp32
# sums and for rows where the values cancel.
@pytest.mark.parametrize("d", [64, 128])
def test_prefill_of_large_scores_in_fp16(d):
    bs, hq, h, n, cached = 16, 6, 2, 90, 1500
    pool, tables, values = filled(35, torch.float16, [cached + n], h, d, bs)
    q = (12.0 * torch.randn(n, hq, d, generator=gen(15), device=DEV)).half()
    cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    start = torch.tensor([cached], dtype=torch.int32, device=DEV)
    bt = device_tables(tables)
    o, _, reach = quant.attend(q, values, tables[0], bs, cached, d**-0.5)
    assert reach.max() > 200
    for plan in (None, kernels.prefill_plan(cu, start, bt, n, n, bs, hq, h, d, dtype=torch.float16)):
        out = kernels.paged_prefill(q, pool.k[0], pool.v[0], bt, cu, start, n, bs, d**-0.5, plan=plan,
                                    kv_scales=pool.kv_scales[0])
        off = (out.double().cpu() - o).norm() / o.norm()
        assert off <= 1.1 * (2 / 3) ** 0.5 * 2.0**-11, off


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
                x = torch.zeros(n, hq, d, device=DEV, dtype=dtype) + q[row : row + n]
                o, a, reach = quant.attend(x[:, heads] if h == 1 else x, values, t, bs, c, d**-0.5)
                tol = fp32_tolerance(o, a, reach, d)
                if dtype != torch.float32:
                    tol = tol + prefill_tolerance(o, a, reach, dtype)
                got = out[row : row + n]
                err = ((got[:, heads] if h == 1 else got).double().cpu() - o).abs()
                assert (err <= tol).all(), (hq, c, n, (err / tol).max())
                row += n


# fp32 queries of a 16-bit pool: the decode holds a query to 2^-16 of each element at least,
# the prefill to 2^-14, and the code products lose at most as much again where they align
# eight products. So scores move by at most 2^-13 reach. Rounding the queries to the dtype
# moves them by u * reach; at scale 1 that is far more than what the outputs' own
# roundings (u a + u |o|) leave, and shows that it is not done.
# (At scale 1 many probabilities are below fp16's smallest normal number, 2^-14 of the
# largest, where a rounding is off by up to 2^-25 and not by u of the probability: for
# the sums, whose divisor is at least the largest probability, 1, by 2^-25 sum |v|.)


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
        if dtype == torch.float16:
            t = torch.arange(n)
            v = values[1, torch.tensor(tables[i])[t // bs] * bs + t % bs]
            tol = tol + 2.0**-25 * v.abs().sum(0).repeat_interleave(hq // h, 0)
        err = (out[i : i + 1].double().cpu() - o).abs()
        assert (err <= tol).all(), (i, n, (err / tol).max())
        off += err.square().sum().item()
        r, _, _ = quant.attend(q[i : i + 1].to(dtype), values, tables[i], bs, n - 1, 1.0)
        rounded += (r - o).square().sum().item()
    assert off < 0.25 * rounded, (off, rounded)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq, h, d, bs", [(28, 4, 128, 16), (14, 2, 64, 32)])
def test_fp32_queries_of_sequences_that_share_blocks(dtype, hq, h, d, bs):
    """The planned decode's pairs, whose units hold the queries of two sequences."""
    pool, tables, values = filled(44, dtype, [700, 40, 530], h, d, bs)
    use, lens = [0, 0, 1, 2, 2, 0], [700, 655, 33, 1, 530, 90]
    q = torch.randn(len(lens), hq, d, generator=gen(45), device=DEV)
    bt = device_tables([tables[i] for i in use])
    ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
    plan = kernels.decode_plan(bt, ctx, hq, pool.k[0], bs, share_groups=True)
    out = kernels.paged_decode_planned(q, pool.k[0], pool.v[0], plan, d**-0.5, err_flags=pool.err_flags,
                                       out=torch.empty_like(q, dtype=dtype), kv_scales=pool.kv_scales[0])
    pool.check_errors()
    for i, n in enumerate(lens):
        o, a, reach = quant.attend(q[i : i + 1], values, tables[use[i]], bs, n - 1, d**-0.5)
        tol = fp32_tolerance(o, a, reach, d) + decode_tolerance(o, a, dtype) + 4 * 2.0**-13 * reach[..., None] * a
        err = (out[i : i + 1].double().cpu() - o).abs()
        assert (err <= tol).all(), (i, n, (err / tol).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq, h, d, bs", [(28, 4, 128, 16), (5, 5, 64, 32)])
def test_rotated_queries_in_fp32(dtype, hq, h, d, bs):
    """What the dtype's own output is the rounding of; without norms the same numbers."""
    g, n = gen(43), 37
    q, k, v = rows(g, n, hq + 2 * h, d, dtype).split([hq, h, h], 1)
    wq, wk = (1 + 0.3 * torch.randn(2, d, generator=g, device=DEV)).to(dtype)
    cos, sin = rotation(g, n, d)
    slots = torch.arange(n, device=DEV)
    for norms in ((wq, wk, 1e-6), ()):
        got = []
        for t in (dtype, torch.float32):
            pool = QuantPagedKVPool(1, 4, bs, h, d, dtype)
            q_out = torch.empty(n, hq + 1, d, dtype=t, device=DEV)[:, 1:]
            kernels.rope_kv_scatter_q8(q, k, v, cos, sin, pool.k[0], pool.v[0], pool.kv_scales[0], slots, bs, *norms,
                                       q_out=q_out)
            got.append((q_out, pool.k.view(torch.uint8).clone(), pool.kv_scales.clone()))
        assert torch.equal(got[0][0], got[1][0].to(dtype))
        assert torch.equal(got[0][1], got[1][1]) and torch.equal(got[0][2], got[1][2])
        if norms:
            o = quant.norm_rope(q, wq, 1e-6, cos, sin)
            tol = norm_tolerance(q, wq, 1e-6, cos, sin, o, dtype, stored=False)
            assert ((got[1][0].double().cpu() - o).abs() <= tol).all()
        else:
            assert torch.equal(got[1][0].to(dtype).float(), got[1][0])


def test_refusals_of_fp32_queries():
    pool = QuantPagedKVPool(1, 4, 16, 2, 64, torch.bfloat16)
    q = torch.zeros(1, 4, 64, device=DEV)
    tables, ctx = torch.zeros(1, 2, dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    caches, scales = (pool.k[0], pool.v[0]), pool.kv_scales[0]
    half, bf16 = q.half(), q.bfloat16()
    with pytest.raises(RuntimeError, match="out must be"):
        kernels.paged_decode(half, *caches, tables, ctx, 16, 0.1, out=bf16, kv_scales=scales)
    with pytest.raises(RuntimeError, match="out must be"):
        kernels.paged_prefill(half, *caches, tables, cu, ctx - 1, 1, 16, 0.1, out=q, kv_scales=scales)
    plan = kernels.prefill_plan(cu, ctx - 1, tables, 1, 1, 16, 4, 2, 64, dtype=torch.float32)
    with pytest.raises(RuntimeError, match="plan was built"):
        kernels.paged_prefill(q, *caches, tables, cu, ctx - 1, 1, 16, 0.1, out=bf16, plan=plan, kv_scales=scales)
    plain = PagedKVPool(1, 4, 16, 2, 64, torch.bfloat16)
    with pytest.raises(RuntimeError, match="mismatch"):
        kernels.paged_decode(q, plain.k[0], plain.v[0], tables, ctx, 16, 0.1, out=bf16)
    rows3, cs, w = (bf16, bf16[:, :2], bf16[:, :2]), torch.zeros(1, 64, device=DEV), torch.ones(64, device=DEV)
    slots = torch.zeros(1, dtype=torch.long, device=DEV)
    with pytest.raises(RuntimeError, match="out must be"):
        kernels.rope_kv_scatter_q8(*rows3, cs, cs, *caches, scales, slots, 16, q_out=half)
    with pytest.raises(RuntimeError, match="q_out must be"):
        kernels.qk_norm_rope_kv_scatter(*rows3, w.bfloat16(), w.bfloat16(), 1e-6, cs, cs, plain.k[0], plain.v[0],
                                        slots, q_out=q)
    assert not pool.k.view(torch.uint8).any() and not plain.k.any()


# ---- norms and rotation
#
# In fp32 the sum of squares of d numbers is off by at most d / 2 + 8 steps of 2^-24, the
# norm by half of that, the products and the sum by a few more, relative to
# |y cos| + |turned y sin| =: m; then half a step of the dtype.


def rotation(g, n, d):
    angle = torch.rand(n, d // 2, generator=g, device=DEV, dtype=torch.float64) * 6.3
    angle = torch.cat([angle, angle], 1)
    return angle.cos().float(), angle.sin().float()


def norm_tolerance(x, w, eps, cos, sin, o, dtype, stored=True):
    y = quant.norm_rope(x, w, eps, torch.ones_like(cos), torch.zeros_like(sin)).abs()
    a, b = y.chunk(2, dim=-1)
    m = y * cos.cpu().double().abs()[:, None] + torch.cat([b, a], -1) * sin.cpu().double().abs()[:, None]
    # (half a step: relative to the number, below the smallest normal number half the smallest one)
    f = torch.finfo(dtype)
    half = torch.maximum(f.eps / 2 * o.abs(), torch.tensor(f.smallest_normal * f.eps / 2, dtype=torch.float64))
    return (x.shape[-1] / 4 + 16) * 2.0**-24 * m + (half if stored else 0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, hq, h, d", [(1, 28, 4, 128), (5, 14, 2, 64), (77, 1, 1, 64), (2500, 9, 3, 128),
                                         (3, 40, 8, 64)])
def test_norm_rope_scatter(dtype, n, hq, h, d):
    g = gen(n)
    qkv = rows(g, n, hq + 2 * h, d, dtype, 2.0)
    q, k, v = qkv.split([hq, h, h], 1)
    wq, wk = (1 + 0.3 * torch.randn(2, d, generator=g, device=DEV)).to(dtype)
    cos, sin = rotation(g, n, d)
    for layout in ("head_major", "slot_major"):
        pool = PagedKVPool(1, n // 16 + 2, 16, h, d, dtype, layout=layout)
        slots = torch.randperm(pool.num_slots, generator=g, device=DEV)[:n]
        if n > 4:
            slots[2] = -1
        before = q.clone()
        out = kernels.qk_norm_rope_kv_scatter(q, k, v, wq, wk, 1e-6, cos, sin, pool.k[0], pool.v[0], slots,
                                              err_flags=pool.err_flags)
        pool.check_errors()
        assert torch.equal(q, before)
        o = quant.norm_rope(q, wq, 1e-6, cos, sin)
        assert ((out.double().cpu() - o).abs() <= norm_tolerance(q, wq, 1e-6, cos, sin, o, dtype)).all()
        kept = slots >= 0
        o = quant.norm_rope(k, wk, 1e-6, cos, sin)
        err = (pool.k[0, slots[kept]].double().cpu() - o[kept.cpu()]).abs()
        assert (err <= norm_tolerance(k, wk, 1e-6, cos, sin, o, dtype)[kept.cpu()]).all()
        assert torch.equal(pool.v[0, slots[kept]], v[kept])
        rest = torch.ones(pool.num_slots, dtype=torch.bool, device=DEV)
        rest[slots[kept]] = False
        assert not pool.k[0, rest].any() and not pool.v[0, rest].any()
    # in place
    mine = q.clone()
    kernels.qk_norm_rope_kv_scatter(mine, k, v, wq, wk, 1e-6, cos, sin, pool.k[0], pool.v[0], slots, q_out=mine)
    assert torch.equal(mine, out)


def test_norm_rope_of_zero_rows_and_slots_past_the_pool():
    d, n = 64, 4
    pool = PagedKVPool(1, 1, 16, 1, d, torch.bfloat16)
    x = torch.zeros(n, 1, d, device=DEV, dtype=torch.bfloat16)
    w = torch.ones(d, device=DEV, dtype=torch.bfloat16)
    cos, sin = rotation(gen(1), n, d)
    out = kernels.qk_norm_rope_kv_scatter(x, x, x, w, w, 1e-6, cos, sin, pool.k[0], pool.v[0],
                                          torch.tensor([0, 16, 3, -5], device=DEV), err_flags=pool.err_flags)
    assert not out.any() and not pool.k.any()
    with pytest.raises(IndexError, match="write slot"):
        pool.check_errors()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq, h, d, bs", [(28, 4, 128, 16), (14, 2, 64, 32), (5, 5, 64, 16)])
def test_rotation_into_the_8_bit_pool_is_the_rotation_then_the_write(dtype, hq, h, d, bs):
    """Without norms: bit for bit ``rope_kv_scatter`` and ``write`` of its keys."""
    g, n = gen(14), 70
    q, k, v = rows(g, n, hq + 2 * h, d, dtype).split([hq, h, h], 1)
    cos, sin = rotation(g, n, d)
    slots = torch.cat([torch.arange(5, 5 + 40), torch.arange(160, 160 + 30)]).to(DEV)
    plain = PagedKVPool(1, 20, bs, h, d, dtype)
    q1 = kernels.rope_kv_scatter(q, k, v, cos, sin, plain.k[0], plain.v[0], slots)
    a, b = (QuantPagedKVPool(1, 20, bs, h, d, dtype) for _ in range(2))
    a.write(0, plain.k[0, slots], v, slots)
    q2 = kernels.rope_kv_scatter_q8(q, k, v, cos, sin, b.k[0], b.v[0], b.kv_scales[0], slots, bs)
    assert torch.equal(q1, q2) and torch.equal(a.kv_scales, b.kv_scales)
    assert torch.equal(a.k.view(torch.uint8), b.k.view(torch.uint8))
    assert torch.equal(a.v.view(torch.uint8), b.v.view(torch.uint8))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq, h, d, bs", [(28, 4, 128, 16), (14, 2, 64, 32)])
def test_normed_rotation_into_the_8_bit_pool(dtype, hq, h, d, bs):
    """Queries as the 16-bit pool's call gives them; keys to the code nearest the number in
    64 bits, or the next where that lies within the fp32 error of the border; blocks that
    hold tokens already keep them."""
    g, n = gen(15), 61
    q, k, v = rows(g, n, hq + 2 * h, d, dtype).split([hq, h, h], 1)
    wq, wk = (1 + 0.3 * torch.randn(2, d, generator=g, device=DEV)).to(dtype)
    cos, sin = rotation(g, n, d)
    slots = torch.arange(3, 3 + n, device=DEV)
    plain = PagedKVPool(1, 6, bs, h, d, dtype)
    q1 = kernels.qk_norm_rope_kv_scatter(q, k, v, wq, wk, 1e-6, cos, sin, plain.k[0], plain.v[0], slots)
    pool, want = QuantPagedKVPool(1, 6, bs, h, d, dtype), quant.QuantCache(6, bs, h, d, dtype)
    old = rows(g, 3, h, d, dtype)
    pool.write(0, old, old, slots[:3] - 3)
    want.write(old, old, slots[:3] - 3)
    q2 = kernels.rope_kv_scatter_q8(q, k, v, cos, sin, pool.k[0], pool.v[0], pool.kv_scales[0], slots, bs, wq, wk, 1e-6)
    assert torch.equal(q1, q2)
    o = quant.norm_rope(k, wk, 1e-6, cos, sin)
    want.write(o, v, slots)
    assert torch.equal(pool.kv_scales[0].double().cpu(), torch.exp2(want.exps.double()))
    got = torch.stack(pool.gather(0, torch.arange(6 * bs, device=DEV))).double().cpu()
    assert torch.equal(got[1], want.values[1])
    assert torch.equal(got[0, :3], want.values[0, :3])
    tol = norm_tolerance(k, wk, 1e-6, cos, sin, o, dtype, stored=False)
    exps = want.exps[:, slots.cpu() // bs, 0].T[..., None].double()
    e = torch.maximum(torch.frexp(o.abs())[1].double() - 1, exps - 6)
    half = torch.exp2(e - 4)  # half a step at the number's own size
    err = (got[0, slots.cpu()] - o).abs()
    assert (err <= half + tol).all()
    assert (got[0, slots.cpu()] != want.values[0, slots.cpu()]).double().mean() < 1e-3


@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rotation_of_a_long_call_is_that_of_its_blocks(dtype, normed):
    """A call whose workgroups share the reading of the slots against calls of some blocks."""
    g, hq, h, d, bs, n = gen(17), 3, 64, 64, 16, 720
    q, k, v = rows(g, n, hq + 2 * h, d, dtype).split([hq, h, h], 1)
    w = (1 + 0.3 * torch.randn(2, d, generator=g, device=DEV)).to(dtype)
    norms = (*w, 1e-6) if normed else ()
    cos, sin = rotation(g, n, d)
    slots = (torch.randperm(n // bs, generator=g, device=DEV)[:, None] * bs + torch.arange(bs, device=DEV)).flatten()
    one, many = (QuantPagedKVPool(1, n // bs, bs, h, d, dtype) for _ in range(2))
    a = kernels.rope_kv_scatter_q8(q, k, v, cos, sin, one.k[0], one.v[0], one.kv_scales[0], slots, bs, *norms)
    for i in range(0, n, 5 * bs):
        t = slice(i, i + 5 * bs)
        b = kernels.rope_kv_scatter_q8(q[t], k[t], v[t], cos[t], sin[t], many.k[0], many.v[0], many.kv_scales[0],
                                       slots[t], bs, *norms)
        assert torch.equal(a[t], b)
    assert torch.equal(one.kv_scales, many.kv_scales)
    for x, y in ((one.k, many.k), (one.v, many.v)):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


# ---- together


def step_inputs(g, b, n, hq, h, d, dtype):
    q, k, v = rows(g, b * n, hq + 2 * h, d, dtype, 0.3).view(b, n, -1, d).split([hq, h, h], 2)
    cos, sin = rotation(g, b * n, d)
    return q, k, v, cos.view(b, n, d), sin.view(b, n, d)


@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_sequence_lives_through_prefill_chunks_and_decodes(dtype, normed):
    """Two sequences prefilled in chunks, then decoded with a third, through the seam on a
    strict pool; every output against attention in 64 bits over the values read back."""
    hq, h, d, bs = 14, 2, 64, 16
    g = gen(16)
    pool = QuantPagedKVPool(2, 40, bs, h, d, dtype, strict=True)
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
            values = torch.stack(pool.gather(layer, torch.arange(pool.num_slots, device=DEV))).double().cpu()
            row = 0
            for i, m, c in zip(live, new, was):
                o, a, reach = quant.attend(qr[row : row + m], values, tables[i], bs, c, d**-0.5)
                tol = fp32_tolerance(o, a, reach, d) + prefill_tolerance(o, a, reach, dtype)
                err = (out.reshape(-1, hq, d)[row : row + m].double().cpu() - o).abs()
                assert (err <= tol).all(), (step, layer, i)
                row += m
        cached = [c + n for c, n in zip(cached, step)]


def test_seam_writes_then_attends_as_its_parts_do():
    """``paged_attention`` over decode metadata: the write, then the kernels' decode."""
    hq, h, d, bs = 28, 4, 128, 16
    g = gen(17)
    lens = [100, 1, 33, 700] * 20  # (enough sequences for the balanced schedule)
    one, tables, _ = filled(40, torch.bfloat16, lens, h, d, bs)
    two, _, _ = filled(40, torch.bfloat16, lens, h, d, bs)
    for pool in (one, two):  # room for the new token in the last block
        assert all(n % bs for n in lens)
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


def test_graph_decoder_replays_the_8_bit_step():
    """Decode steps through ``HipGraphDecoder``, several replays with eager work between
    them, each against the same step run eagerly on a copy of the pool."""
    hq, h, d, bs, dtype = 8, 2, 64, 16, torch.bfloat16
    g = gen(18)
    tables = [[0, 1, 2], [3, 4, 5], [6, 7, 8]]
    pools = [QuantPagedKVPool(2, 9, bs, h, d, dtype) for _ in range(2)]
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
        assert torch.equal(pools[0].k.view(torch.uint8), pools[1].k.view(torch.uint8))


@pytest.mark.parametrize("overlap", [False, True])
def test_mixed_step_over_the_8_bit_pool(overlap):
    cfg = MixedConfig("t", 2, 70, 20, 300, 3, 40, 33, 28, 4, 128, 16, torch.bfloat16, seed=2)
    _, plain, batch, inputs = make_mixed_case(cfg, DEV)
    runs = []
    for _ in range(2):
        pool = QuantPagedKVPool(cfg.num_layers, plain.num_blocks, 16, 4, 128, cfg.dtype)
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
    pool = runs[0].pool
    values = torch.stack(pool.gather(1, torch.arange(pool.num_slots, device=DEV))).double().cpu()
    for i in (0, 69):
        n = int(batch.dec_ctx[i])
        o, a, reach = quant.attend(inputs.q_dec[1, i : i + 1], values, batch.dec_tables[i].tolist(), 16, n - 1,
                                   cfg.scale)
        tol = decode_tolerance(o, a, cfg.dtype) + fp32_tolerance(o, a, reach, 128)
        assert ((eager[0][1, i].double().cpu() - o).abs() <= tol).all()
    o, a, reach = quant.attend(inputs.q_pre[1, 40:80], values, batch.pre_tables[1].tolist(), 16, 33, cfg.scale)
    tol = prefill_tolerance(o, a, reach, cfg.dtype) + fp32_tolerance(o, a, reach, 128)
    assert ((eager[1][1, 40:80].double().cpu() - o).abs() <= tol).all()


@pytest.mark.parametrize("layout", ["head_major", "slot_major"])
def test_normed_seam_over_the_16_bit_pool(layout):
    """Norms through ``rope_paged_attention``: the normed rotation, then the attention alone."""
    hq, h, d, bs, dtype = 6, 2, 64, 16, torch.bfloat16
    g = gen(51)
    wq, wk = (1 + 0.3 * torch.randn(2, d, generator=g, device=DEV)).to(dtype)
    pools = [PagedKVPool(1, 12, bs, h, d, dtype, layout=layout) for _ in range(2)]
    for cached, new in (([0, 0], [20, 33]), ([20, 33], [1, 1])):
        for pool, whole in zip(pools, (True, False)):
            if max(new) > 1:
                paged, mask = metadata.prefill_context(pool, [[3, 1, 5], [0, 2, 4]], cached, new)
                b, n = 1, sum(new)
            else:
                paged, mask = metadata.decode_context(pool, [[3, 1, 5], [0, 2, 4]], cached)
                b, n = 2, 1
            if whole:
                x = step_inputs(g, b, n, hq, h, d, dtype)
            q, k, v, cos, sin = x
            if whole:
                want = rope_paged_attention(q, k, v, cos, sin, paged, mask, 0, d**-0.5, 3, q_norm=wq, k_norm=wk)
                continue
            spare = PagedKVPool(1, 12, bs, h, d, dtype)
            args = (q.reshape(-1, hq, d), k.reshape(-1, h, d), v.reshape(-1, h, d))
            qr = kernels.qk_norm_rope_kv_scatter(*args, wq, wk, 1e-6, cos.view(-1, d), sin.view(-1, d), spare.k[0],
                                                 spare.v[0], paged.write_slots)
            kr, vr = (t[0, paged.write_slots].view(b, n, h, d) for t in (spare.k, spare.v))
            got = paged_attention(qr.view(b, n, hq, d), kr, vr, paged, mask, 0, d**-0.5, 3)
            assert torch.equal(got, want)
    assert torch.equal(pools[0].k, pools[1].k) and torch.equal(pools[0].v, pools[1].v)


def test_one_graph_of_every_call():
    """Writes, normed rotations into both kinds of pool, reading back and attention in one
    graph, replayed on other inputs with eager work and synchronizations between."""
    hq, h, d, bs, n, dtype = 8, 2, 64, 16, 50, torch.bfloat16
    g = gen(52)
    w = (1 + 0.3 * torch.randn(d, generator=g, device=DEV)).to(dtype)
    slots = torch.arange(n, device=DEV) + 16
    tables = torch.tensor([[1, 2, 3, 4]], dtype=torch.int32, device=DEV)
    ctx = torch.tensor([n], dtype=torch.int32, device=DEV)
    cu, start = torch.tensor([0, n], dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    x = rows(g, n, hq + 2 * h, d, dtype)
    cos, sin = rotation(g, n, d)

    def pools():
        return QuantPagedKVPool(2, 6, bs, h, d, dtype), PagedKVPool(1, 6, bs, h, d, dtype)

    def step(x, quantised, plain):
        q, k, v = x.split([hq, h, h], 1)
        quantised.write(0, k, v, slots)
        q_out = torch.empty(n, hq, d, device=DEV)
        kernels.rope_kv_scatter_q8(q, k, v, cos, sin, quantised.k[1], quantised.v[1], quantised.kv_scales[1], slots, bs,
                                   w, w, 1e-6, q_out)
        q16 = kernels.qk_norm_rope_kv_scatter(q, k, v, w, w, 1e-6, cos, sin, plain.k[0], plain.v[0], slots)
        out = torch.empty(n, hq, d, dtype=dtype, device=DEV)
        plan = kernels.prefill_plan(cu, start, tables, n, n, bs, hq, h, d, dtype=dtype)
        kernels.paged_prefill(q_out, quantised.k[1], quantised.v[1], tables, cu, start, n, bs, d**-0.5, out=out,
                              plan=plan, kv_scales=quantised.kv_scales[1])
        decode = kernels.decode_plan(tables, ctx, hq, quantised.k[0], bs)
        one = kernels.paged_decode_planned(q16[:1], quantised.k[0], quantised.v[0], decode, d**-0.5,
                                           kv_scales=quantised.kv_scales[0])
        return (q_out, q16, out, one, *quantised.gather(0, slots), *quantised.gather_blocks(1, tables, ctx, n),
                plain.k, plain.v)

    static, mine, other = x.clone(), pools(), pools()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static, *mine)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(static, *mine)
    for i in range(4):
        static.copy_(rows(g, n, hq + 2 * h, d, dtype) * 2.0 ** (3 * i - 4))
        want = [t.clone() for t in step(static, *other)]
        graph.replay()
        if i % 2:
            torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), i


def test_layers_on_two_streams():
    """Two layers of a pool written and attended on streams of their own at the same time."""
    hq, h, d, bs, n, dtype = 28, 4, 128, 16, 700, torch.bfloat16
    g = gen(53)
    pools = [QuantPagedKVPool(2, 50, bs, h, d, dtype) for _ in range(2)]
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


def test_write_of_very_many_tokens_in_any_order():
    """One call of 70,000 shuffled tokens against calls that each take some whole blocks."""
    h, d, bs, dtype = 2, 64, 48, torch.bfloat16
    g = gen(54)
    blocks = 1459
    n = blocks * bs
    k, v = rows(g, n, h, d, dtype), rows(g, n, h, d, dtype)
    slots = torch.randperm(n, generator=g, device=DEV)
    one, many = (QuantPagedKVPool(1, blocks, bs, h, d, dtype) for _ in range(2))
    one.write(0, k, v, slots)
    order = slots.argsort()
    for lo in range(0, n, 200 * bs):
        i = order[lo : lo + 200 * bs]
        many.write(0, k[i], v[i], slots[i])
    assert torch.equal(one.kv_scales, many.kv_scales)
    for a, b in ((one.k, many.k), (one.v, many.v)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_rows_far_apart():
    """Queries, keys and values whose rows are more than 2^31 elements apart."""
    hq, h, d, bs, dtype = 4, 2, 64, 16, torch.bfloat16
    far = torch.empty(3, (1 << 30) + 64, dtype=dtype, device=DEV)
    g = gen(55)
    x = rows(g, 3, hq + 2 * h, d, dtype)
    far[:, : (hq + 2 * h) * d] = x.flatten(1)
    wide = far[:, : (hq + 2 * h) * d].unflatten(1, (hq + 2 * h, d))
    assert wide.stride(0) * 2 > 1 << 31
    w = torch.ones(d, dtype=dtype, device=DEV)
    cos, sin = rotation(g, 3, d)
    slots = torch.arange(3, device=DEV)
    outs = []
    for t in (x, wide):
        q, k, v = t.split([hq, h, h], 1)
        quantised, plain = QuantPagedKVPool(2, 1, bs, h, d, dtype), PagedKVPool(1, 1, bs, h, d, dtype)
        quantised.write(0, k, v, slots)
        tables = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
        cu = torch.tensor([0, 3], dtype=torch.int32, device=DEV)
        args = (quantised.k[0], quantised.v[0])
        outs.append([
            kernels.qk_norm_rope_kv_scatter(q, k, v, w, w, 1e-6, cos, sin, plain.k[0], plain.v[0], slots).contiguous(),
            kernels.rope_kv_scatter_q8(q, k, v, cos, sin, quantised.k[1], quantised.v[1], quantised.kv_scales[1], slots,
                                       bs, w, w, 1e-6).contiguous(),
            kernels.paged_prefill(q, *args, tables, cu, cu[:1], 3, bs, 0.125, kv_scales=quantised.kv_scales[0]),
            kernels.paged_decode(q, *args, tables.expand(3, 1).contiguous(), cu[1:].expand(3).contiguous(), bs, 0.125,
                                 kv_scales=quantised.kv_scales[0]),
            quantised.k.view(torch.uint8), quantised.v.view(torch.uint8), quantised.kv_scales, plain.k, plain.v])
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_refusals():
    h, d, bs = 2, 64, 16
    pool = QuantPagedKVPool(1, 8, bs, h, d, torch.bfloat16)
    x = torch.zeros(1, 1, 4, d, device=DEV, dtype=torch.bfloat16)
    kv = x[:, :, :h]
    paged, mask = metadata.decode_context(pool, [[0, 1]], [5])
    # nothing but block tables is attended, and nothing is written before that is refused
    bare = PagedContext(pool, paged.write_slots, paged.gather_slots)
    off = PagedContext(pool, paged.write_slots, paged.gather_slots, False, paged.block_tables, paged.context_lens)
    two = torch.zeros(1, 2, 4, d, device=DEV, dtype=torch.bfloat16)
    for p in (bare, off):
        with pytest.raises(RuntimeError, match="block_tables"):
            paged_attention(x, kv + 1, kv + 1, p, mask, 0, 0.1, 2)
    with pytest.raises(RuntimeError, match="block_tables"):
        paged_attention(two, two[:, :, :h], two[:, :, :h], paged, mask, 0, 0.1, 2)
    with pytest.raises(RuntimeError, match="dtype"):
        paged_attention(x.half(), kv.half(), kv.half(), paged, mask, 0, 0.1, 2)
    cos = torch.zeros(1, 1, d, device=DEV)
    w = torch.ones(d, device=DEV, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="go together"):
        rope_paged_attention(x, kv, kv, cos, cos, paged, mask, 0, 0.1, 2, q_norm=w)
    with pytest.raises(RuntimeError, match="q_norm"):
        rope_paged_attention(x, kv, kv, cos, cos, paged, mask, 0, 0.1, 2, q_norm=w.float(), k_norm=w)
    with pytest.raises(RuntimeError, match="pool's dtype"):
        pool.write(0, kv[0].half(), kv[0].half(), paged.write_slots)
    with pytest.raises(RuntimeError, match="do not match"):
        pool.write(0, x[0], x[0], paged.write_slots)
    with pytest.raises(RuntimeError, match="int64"):
        pool.write(0, kv[0], kv[0], paged.write_slots.int())
    assert not pool.k.view(torch.uint8).any()
    # kernels: scales of another shape, layouts that are not dense, caches that are no codes
    q = x[0]
    args = (paged.block_tables, paged.context_lens, bs, 0.1)
    scales = pool.kv_scales[0]
    for s in (scales[:, :4], scales.double(), scales.transpose(0, 1)):
        with pytest.raises(RuntimeError, match="kv_scales"):
            kernels.paged_decode(q, pool.k[0], pool.v[0], *args, kv_scales=s)
    loose = pool.k[0].contiguous()
    with pytest.raises(RuntimeError, match="dense"):
        kernels.paged_decode(q, loose, loose, *args, kv_scales=scales)
    with pytest.raises(RuntimeError, match="codes"):
        kernels.paged_decode(q, pool.k[0].float(), pool.v[0].float(), *args, kv_scales=scales)
    with pytest.raises(RuntimeError, match="mismatch"):
        kernels.paged_decode(q, pool.k[0], pool.v[0], *args)
    with pytest.raises(RuntimeError, match="out must be"):
        kernels.paged_decode(q, pool.k[0], pool.v[0], *args, out=q.float(), kv_scales=scales)
    cu = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="new_kv"):
        kernels.paged_prefill(q, pool.k[0], pool.v[0], paged.block_tables, cu, paged.context_lens, 1, bs, 0.1,
                              new_kv=(kv[0], kv[0], paged.write_slots), kv_scales=scales)
    other = PagedKVPool(1, 8, bs, h, d, torch.bfloat16)
    plan = kernels.decode_plan(paged.block_tables, paged.context_lens, 4, other.k[0], bs)
    with pytest.raises(RuntimeError, match="plan"):
        kernels.paged_decode_planned(q, pool.k[0], pool.v[0], plan, 0.1, kv_scales=scales)
    with pytest.raises(RuntimeError, match="kv_scales"):
        kernels.gather_slots_q8(pool.k[0], pool.v[0], scales, paged.write_slots, 32, torch.bfloat16)
    torch.cuda.synchronize()


def test_layers_are_those_of_the_tensors_the_pool_has_now():
    pool = QuantPagedKVPool(2, 2, 16, 2, 64, torch.bfloat16)
    assert all(a.data_ptr() == b[1].data_ptr() for a, b in zip(pool.layer(1), (pool.k, pool.v, pool.kv_scales)))
    first = pool.layer(0)
    assert pool.layer(0)[0] is first[0] and pool.layer(-1)[2] is pool.layer(1)[2]
    pool.kv_scales = pool.kv_scales.clone()
    assert pool.layer(1)[2].data_ptr() == pool.kv_scales[1].data_ptr()
    with pytest.raises(IndexError):
        pool.layer(2)
