"""Errors of the 8-bit pool's attention in the norm over a sequence's outputs, which a wrong
scale, a missing tile or a weight of a merge cannot hide in (``test_quant_errors.py`` shows
that on the CPU), and what its queries and probabilities keep of their bits."""

from __future__ import annotations

import dataclasses

import pytest
import torch

from infrared_amd import PagedKVPool, QuantPagedKVPool, kernels, metadata, rope_paged_attention
from infrared_amd._lib import ERR_PLAN
from infrared_amd.mixed_step import MixedConfig, MixedStep, make_mixed_case
from oracle import quant
from test_gpu_quant import device_tables, filled, gen, rotation, rows, run_decode, step_inputs

pytestmark = pytest.mark.gpu

DEV = "cuda"
HALF = [torch.bfloat16, torch.float16]


def check(out, q, values, table, bs, cached, scale, dtype, round_p, what=None):
    """A sequence's outputs within the bound of their roundings."""
    o, spread, reach = quant.attend_spread(q, values, table, bs, cached, scale)
    off, bound = float((out.double().cpu() - o).norm()), quant.error_bound(o, spread, reach, dtype, round_p)
    assert off <= bound, (what, off / float(o.norm()), bound / float(o.norm()))


def chunks(cached, new):
    """Device metadata of packed chunks."""
    cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
    return cu, torch.tensor(cached, dtype=torch.int32, device=DEV)


# ---- prefill: the probabilities and the output are rounded to the dtype, nothing else


@pytest.mark.parametrize("plan", [False, True])
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("hq, h, d, bs", [(28, 4, 128, 16), (14, 2, 64, 16), (8, 8, 64, 64), (20, 1, 128, 48)])
def test_prefill(plan, dtype, hq, h, d, bs):
    cached, new = [0, 37, 0, 512, 1, 130], [1, 70, 200, 1, 0, 65]
    pool, tables, values = filled(hq, dtype, [c + n for c, n in zip(cached, new)], h, d, bs)
    total = sum(new)
    q = torch.randn(total, 2 * hq, d, generator=gen(12), device=DEV).to(dtype)[:, :hq]
    cu, start = chunks(cached, new)
    bt = device_tables(tables)
    p = kernels.prefill_plan(cu, start, bt, total, max(new), bs, hq, h, d, dtype=dtype) if plan else None
    out = kernels.paged_prefill(q, pool.k[0], pool.v[0], bt, cu, start, max(new), bs, d**-0.5,
                                err_flags=pool.err_flags, plan=p, kv_scales=pool.kv_scales[0])
    pool.check_errors()
    row = 0
    for t, c, n in zip(tables, cached, new):
        if n:
            check(out[row : row + n], q[row : row + n], values, t, bs, c, d**-0.5, dtype, 1.0, (c, n))
        row += n


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("hq, h", [(8, 4), (130, 1)])
def test_prefill_over_many_workgroups_and_wide_groups(dtype, hq, h):
    bs, d = 16, 64
    cached, new = [6000, 0, 300], [700, 900, 257]
    pool, tables, values = filled(31, dtype, [c + n for c, n in zip(cached, new)], h, d, bs)
    total = sum(new)
    q = torch.randn(total, hq, d, generator=gen(13), device=DEV).to(dtype)
    cu, start = chunks(cached, new)
    bt = device_tables(tables)
    plan = kernels.prefill_plan(cu, start, bt, total, max(new), bs, hq, h, d, dtype=dtype)
    heads = slice(0, hq) if hq <= 8 else slice(hq - 3, hq)  # (the oracle's cost)
    for p in (plan, None):
        out = kernels.paged_prefill(q, pool.k[0], pool.v[0], bt, cu, start, max(new), bs, d**-0.5, plan=p,
                                    kv_scales=pool.kv_scales[0])
        row = 0
        for t, c, n in zip(tables, cached, new):
            check(out[row : row + n, heads], q[row : row + n, heads], values, t, bs, c, d**-0.5, dtype, 1.0, (hq, c))
            row += n


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("d", [64, 128])
def test_prefill_of_large_scores(d, dtype, wide):
    """Scores of some hundred, of queries of the dtype and of fp32: what a query or a sum of
    products loses shows in every probability."""
    bs, hq, h, n, cached = 16, 6, 2, 90, 1500
    pool, tables, values = filled(35, dtype, [cached + n], h, d, bs)
    q = 12.0 * torch.randn(n, hq, d, generator=gen(15), device=DEV)
    if not wide:
        q = q.to(dtype)
    cu, start = chunks([cached], [n])
    bt = device_tables(tables)
    for plan in (None, kernels.prefill_plan(cu, start, bt, n, n, bs, hq, h, d, dtype=dtype)):
        out = torch.empty(n, hq, d, dtype=dtype, device=DEV)
        kernels.paged_prefill(q, pool.k[0], pool.v[0], bt, cu, start, n, bs, d**-0.5, out=out, plan=plan,
                              kv_scales=pool.kv_scales[0])
        check(out, q, values, tables[0], bs, cached, d**-0.5, dtype, 1.0)


# ---- queries that one element dwarfs


def without_channel(seed, dtype, lens, h, d, bs, channel):
    """``filled`` whose keys are zero in a channel."""
    pool, tables, values = filled(seed, dtype, lens, h, d, bs)
    raw = pool.k[0].view(torch.uint8)
    written = (raw != 0x7F).any(-1).any(-1)
    raw[written, :, channel] = 0
    values[0, :, :, channel] = 0.0
    return pool, tables, values


def others_beside_a_large_one(path, hq, h, d, dtype, wide):
    """One element of a query is 30,000 (in bf16 and fp32 also a million) times the others, and
    no key has anything there: the scores are of the others alone, to their own bits. In fp32
    the large one is past fp16's range."""
    bs, lens, channel = 16, [700, 33, 250, 64], 5
    pool, tables, values = without_channel(36 + d, dtype, lens, h, d, bs, channel)
    q = torch.randn(len(lens), hq, d, generator=gen(16), device=DEV)
    q[:, :, channel] = 3e4
    if wide or dtype == torch.bfloat16:
        q[1:, :, channel] = -1e6
    if not wide:
        q = q.to(dtype)
    ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
    bt, out = device_tables(tables), torch.empty(len(lens), hq, d, dtype=dtype, device=DEV)
    attend(path, pool, q, bt, ctx, d**-0.5, out)
    rest = q.clone()
    rest[:, :, channel] = 0.0  # (reach is that of the others too)
    for i, n in enumerate(lens):
        check(out[i : i + 1], rest[i : i + 1], values, tables[i], bs, n - 1, d**-0.5, dtype, 1.0, i)


def attend(path, pool, q, bt, ctx, scale, out):
    """One token of each sequence by the decode, planned or not, or the prefill, with a plan or without."""
    n, hq, d = q.shape
    bs, h = pool.block_size, pool.num_kv_heads
    if path in ("decode", "planned"):
        run = {"err_flags": pool.err_flags, "kv_scales": pool.kv_scales[0], "out": out}
        if path == "decode":
            kernels.paged_decode(q, pool.k[0], pool.v[0], bt, ctx, bs, scale, **run)
        else:
            plan = kernels.decode_plan(bt, ctx, hq, pool.k[0], bs, err_flags=pool.err_flags)
            kernels.paged_decode_planned(q, pool.k[0], pool.v[0], plan, scale, **run)
    else:
        cu, plan = torch.arange(n + 1, dtype=torch.int32, device=DEV), None
        if path == "prefill_plan":
            plan = kernels.prefill_plan(cu, ctx - 1, bt, n, 1, bs, hq, h, d, dtype=pool.dtype)
        kernels.paged_prefill(q, pool.k[0], pool.v[0], bt, cu, ctx - 1, 1, bs, scale, plan=plan, out=out,
                              err_flags=pool.err_flags, kv_scales=pool.kv_scales[0])
    pool.check_errors()


def fp32_queries(path, size, dtype):
    """Queries whose numbers leave fp16's range on either side, with the scale that makes up for
    it; a query of zeros attends all keys alike."""
    hq, h, d, bs, lens = 14, 2, 64, 16, [300, 5, 64, 40]
    pool, tables, values = filled(37, dtype, lens, h, d, bs)
    q = size * torch.randn(len(lens), hq, d, generator=gen(17), device=DEV)
    q[3] = 0.0
    ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = torch.empty(len(lens), hq, d, dtype=dtype, device=DEV)
    scale = d**-0.5 / size
    attend(path, pool, q, device_tables(tables), ctx, scale, out)
    for i, n in enumerate(lens):
        check(out[i : i + 1], q[i : i + 1], values, tables[i], bs, n - 1, scale, dtype, 1.0, i)


@pytest.mark.parametrize("path", ["prefill", "prefill_plan"])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("hq, h, d", [(28, 4, 128), (14, 2, 64)])
def test_prefill_of_a_large_element(hq, h, d, dtype, wide, path):
    others_beside_a_large_one(path, hq, h, d, dtype, wide)


@pytest.mark.parametrize("path", ["prefill", "prefill_plan"])
@pytest.mark.parametrize("size", [1e-30, 1e-7, 1e6, 1e30])
@pytest.mark.parametrize("dtype", HALF)
def test_prefill_of_fp32_queries_of_any_size(path, size, dtype):
    fp32_queries(path, size, dtype)


@pytest.mark.parametrize("path", ["decode", "planned"])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("hq, h, d", [(28, 4, 128), (14, 2, 64)])
def test_decode_of_a_large_element(hq, h, d, dtype, wide, path):
    others_beside_a_large_one(path, hq, h, d, dtype, wide)


@pytest.mark.parametrize("path", ["decode", "planned"])
@pytest.mark.parametrize("size", [1e-30, 1e-7, 1e6, 1e30])
@pytest.mark.parametrize("dtype", HALF)
def test_decode_of_fp32_queries_of_any_size(path, size, dtype):
    fp32_queries(path, size, dtype)


# ---- decode: the output is rounded, the probabilities keep what shows in it


@pytest.mark.parametrize("planned", [False, True])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("hq, h, d, bs", [(28, 4, 128, 16), (14, 2, 64, 16), (8, 8, 64, 32), (20, 1, 128, 48),
                                          (33, 1, 64, 16)])
def test_decode(planned, dtype, wide, hq, h, d, bs):
    lens = [1, 2, 15, 16, 17, 33, 300, 1100, 64, 0, 5]
    pool, tables, values = filled(hq + d, dtype, lens, h, d, bs)
    q = torch.randn(len(lens), hq, d, generator=gen(9), device=DEV)
    kw = {"out": torch.empty(len(lens), hq, d, dtype=dtype, device=DEV)} if wide else {}
    q = q if wide else q.to(dtype)
    out = run_decode(pool, q, device_tables(tables), torch.tensor(lens, dtype=torch.int32, device=DEV), planned, **kw)
    pool.check_errors()
    for i, n in enumerate(lens):
        if n:
            check(out[i : i + 1], q[i : i + 1], values, tables[i], bs, n - 1, d**-0.5, dtype, 0.0, n)
        else:
            assert not out[i].any()


@pytest.mark.parametrize("dtype, hq, h, d, lens", [
    (torch.bfloat16, 28, 4, 128, [9000, 700, 4097, 2500]), (torch.bfloat16, 28, 4, 128, [20011]),
    (torch.float16, 14, 2, 64, [9000, 0, 17]), (torch.bfloat16, 40, 2, 64, [8191, 4000]),
])
def test_decode_of_long_contexts(dtype, hq, h, d, lens):
    """Contexts cut into parts, merged at arrival or by a launch of their own; pairs."""
    bs = 16
    pool, tables, values = filled(23, dtype, lens, h, d, bs)
    tables.insert(1, tables[0][:200])
    lens = [lens[0], 200 * bs - 3, *lens[1:]]
    q = torch.randn(len(lens), hq, d, generator=gen(10), device=DEV).to(dtype)
    ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
    for planned in (True, False):
        out = run_decode(pool, q, device_tables(tables), ctx, planned)
        pool.check_errors()
        for i, n in enumerate(lens):
            if n:
                check(out[i : i + 1], q[i : i + 1], values, tables[i], bs, n - 1, d**-0.5, dtype, 0.0, (planned, n))


# ---- together


@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("dtype", HALF)
def test_a_sequence_through_the_seam(dtype, normed):
    """Prefill chunks, then decodes, through ``rope_paged_attention``, against attention in 64 bits of
    the queries as they leave the rotation over the values read back."""
    hq, h, d, bs = 14, 2, 64, 16
    g = gen(16)
    pool = QuantPagedKVPool(1, 40, bs, h, d, dtype, strict=True)
    tables = [list(range(20, 30)), list(range(3, 13)), list(range(30, 40))]
    wq, wk = (1 + 0.3 * torch.randn(2, d, generator=g, device=DEV)).to(dtype)
    norms = {"q_norm": wq, "k_norm": wk, "eps": 1e-5} if normed else {}
    cached = [0, 0, 0]
    for step in ([40, 3, 0], [1, 60, 0], [33, 1, 9], [1, 1, 1], [1, 1, 1]):
        live = [i for i, n in enumerate(step) if n]
        new, was = [step[i] for i in live], [cached[i] for i in live]
        decode = max(new) == 1
        context = metadata.decode_context if decode else metadata.prefill_context
        paged, mask = context(pool, [tables[i] for i in live], was, *(() if decode else (new,)))
        b, n = (len(live), 1) if decode else (1, sum(new))
        q, k, v, cos, sin = step_inputs(g, b, n, hq, h, d, dtype)
        out = rope_paged_attention(q, k, v, cos, sin, paged, mask, 0, d**-0.5, hq // h, **norms).reshape(-1, hq, d)
        spare = QuantPagedKVPool(1, 40, bs, h, d, dtype)
        qr = torch.empty(b * n, hq, d, device=DEV)
        kernels.rope_kv_scatter_q8(q.reshape(-1, hq, d), k.reshape(-1, h, d), v.reshape(-1, h, d), cos.reshape(-1, d),
                                   sin.reshape(-1, d), spare.k[0], spare.v[0], spare.kv_scales[0], paged.write_slots,
                                   bs, *(norms.values()), q_out=qr)
        values = torch.stack(pool.gather(0, torch.arange(pool.num_slots, device=DEV))).double().cpu()
        row = 0
        for i, m, c in zip(live, new, was):
            check(out[row : row + m], qr[row : row + m], values, tables[i], bs, c, d**-0.5, dtype, 1.0, (step, i))
            row += m
        cached = [c + n for c, n in zip(cached, step)]


@pytest.mark.parametrize("dtype", HALF)
def test_mixed_step(dtype):
    cfg = MixedConfig("t", 1, 70, 20, 300, 3, 40, 33, 28, 4, 128, 16, dtype, seed=2)
    _, plain, batch, inputs = make_mixed_case(cfg, DEV)
    pool = QuantPagedKVPool(1, plain.num_blocks, 16, 4, 128, dtype)
    slots = torch.arange(pool.num_slots, device=DEV)
    pool.write(0, plain.k[0], plain.v[0], slots)
    step = MixedStep(pool, batch, inputs, cfg.scale)
    step.eager()
    assert int(step.err.item()) == 0
    values = torch.stack(pool.gather(0, slots)).double().cpu()
    for i in range(0, 70, 3):
        check(step.out_dec[0, i : i + 1], inputs.q_dec[0, i : i + 1], values, batch.dec_tables[i].tolist(), 16,
              int(batch.dec_ctx[i]) - 1, cfg.scale, dtype, 0.0, i)
    for i in range(3):
        t = slice(40 * i, 40 * i + 40)
        check(step.out_pre[0, t], inputs.q_pre[0, t], values, batch.pre_tables[i].tolist(), 16, 33, cfg.scale, dtype, 1.0)


# ---- writes whose workgroups take several blocks in turn


@pytest.mark.parametrize("mode", ["plain", "rotated", "normed"])
@pytest.mark.parametrize("n, window", [(70, 2), (260, 8), (520, 16)])
def test_write_of_windows_of_some_tokens(n, window, mode):
    """Every token of a window may own a block: shuffled tokens with slots given twice, skipped and past
    the pool; one token a block; runs that begin inside blocks. 64 KV heads make 32 workgroups a token."""
    h, hq, d, bs, dtype = 64, 2, 64, 16, torch.bfloat16
    assert max(1, n * (2 * h // 4) // 1024) == window
    g, blocks = gen(n), 640
    pool, want = QuantPagedKVPool(1, blocks, bs, h, d, dtype), quant.QuantCache(blocks, bs, h, d, dtype)
    total = pool.num_slots
    shuffled = torch.randint(0, 40 * bs, (n,), generator=g, device=DEV)
    shuffled[::9] = -1
    shuffled[6] = total
    shuffled[1::2] = shuffled[0::2][: len(shuffled[1::2])]  # (given twice, next to each other)
    decode = torch.randperm(blocks, generator=g, device=DEV)[:n] * bs + torch.randint(0, bs, (n,), generator=g, device=DEV)
    runs = torch.arange(n, device=DEV) + 7
    calls = [(shuffled, True), (runs, False), (runs.flip(0), False)]
    if mode == "plain" or n == 70:  # (the oracle's cost)
        calls.append((decode, False))
    for slots, bad in calls:
        q, k, v = rows(g, n, hq + 2 * h, d, dtype, 2.0).split([hq, h, h], 1)
        if mode == "plain":
            pool.write(0, k, v, slots)
            want.write(k, v, slots)
        else:
            w = (1 + 0.3 * torch.randn(2, d, generator=g, device=DEV)).to(dtype)
            cos, sin = rotation(g, n, d)
            norms = (*w, 1e-6) if mode == "normed" else ()
            kernels.rope_kv_scatter_q8(q, k, v, cos, sin, pool.k[0], pool.v[0], pool.kv_scales[0], slots, bs, *norms,
                                       err_flags=pool.err_flags)
            # the keys as the pool takes them: the same call's over a 32-bit pool (normed: fp32, of
            # rows that fp32 holds exactly), the last row of a slot given twice where it comes to rest
            wide = torch.float32 if mode == "normed" else dtype
            turned = torch.empty(n, h, d, dtype=wide, device=DEV)
            x = [t.to(wide) for t in (k, k, v)]
            spare_k, spare_v = torch.empty(2, n, h, d, dtype=wide, device=DEV)
            if norms:
                kernels.qk_norm_rope_kv_scatter(*x, w[1].to(wide), w[1].to(wide), 1e-6, cos, sin, spare_k, spare_v,
                                                torch.arange(n, device=DEV), q_out=turned)
            else:
                kernels.rope_kv_scatter(*x, cos, sin, spare_k, spare_v, torch.arange(n, device=DEV), q_out=turned)
            want.write(turned, v, slots)
        if bad:
            with pytest.raises(IndexError, match="slot"):
                pool.check_errors()
        pool.check_errors()
        assert torch.equal(pool.kv_scales[0].double().cpu(), torch.exp2(want.exps.double()))
        k, v = pool.gather(0, torch.arange(total, device=DEV))
        assert torch.equal(torch.stack([k, v]).double().cpu(), want.values)


# ---- plans of the other kind of pool


@pytest.mark.parametrize("share", [False, True])
@pytest.mark.parametrize("lens", [[4000], [700, 900, 300] * 20])
def test_a_plan_of_another_kind_of_pool_writes_nothing(lens, share):
    """Plans of 8-bit and of other pools lie differently in memory: a run over the other's flags it
    and touches neither the output nor the counters, in the launch that merges too."""
    hq, h, d, bs, dtype = 8, 2, 64, 16, torch.bfloat16
    pool, tables, _ = filled(61, dtype, lens, h, d, bs)
    plain = PagedKVPool(1, pool.num_blocks, bs, h, d, dtype)
    bt, ctx = device_tables(tables), torch.tensor(lens, dtype=torch.int32, device=DEV)
    q = torch.randn(len(lens), hq, d, generator=gen(62), device=DEV).to(dtype)
    plans = [kernels.decode_plan(bt, ctx, hq, p.k[0], bs, share_groups=share) for p in (pool, plain)]
    as_other = [dataclasses.replace(a, buf=b.buf) for a, b in (plans, plans[::-1])]
    ctr = torch.zeros(kernels.decode_num_counters(len(lens), hq, h), dtype=torch.int32, device=DEV)
    for p, plan, kw in ((pool, as_other[0], {"kv_scales": pool.kv_scales[0]}), (plain, as_other[1], {})):
        out, err = torch.full_like(q, 3.0), torch.zeros(1, dtype=torch.int32, device=DEV)
        kernels.paged_decode_planned(q, p.k[0], p.v[0], plan, d**-0.5, out=out, err_flags=err, counters=ctr, **kw)
        torch.cuda.synchronize()
        assert err.item() == ERR_PLAN and bool((out == 3.0).all()) and not ctr.any()
        right = plans[0] if kw else plans[1]
        err.zero_()
        kernels.paged_decode_planned(q, p.k[0], p.v[0], right, d**-0.5, out=out, err_flags=err, counters=ctr, **kw)
        assert err.item() == 0 and not (out == 3.0).all()
