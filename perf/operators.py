"""Operators of a layer whose K/V cache is held in 8 bits, measured through the
framework's public calls (``own``) or as plain torch operations.

- ``rope``: norms of queries and keys for each head and the position rotation in
  one pass, the keys and values written to a 16- or 32-bit pool.
- ``store``: the step's new K/V quantised into an 8-bit pool (e4m3 codes, a power
  of two as scale for each block of tokens and KV head) and the blocks they fell
  into read back.
- ``decode`` / ``prefill``: attention over an 8-bit pool, for one query token a
  sequence and for packed chunks after cached prefixes.
- ``layer``: all of it as a decoder layer of a mixed step uses it: norms and
  rotation, the quantising write, attention of decode rows and chunks.

The cache of one layer: codes ``[H_kv, blocks, block size, D]`` for K and for V,
scales ``[H_kv, blocks, 2]`` (K, V). A value is ``code * 2^k``, ``k`` the least
integer with ``amax <= 448 * 2^k`` over the block's tokens, at least -100 (fp16:
-15). Writing a block's first token starts it anew; otherwise its scale only grows.
"""

import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ESIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
SMALL = {"hq": 14, "hkv": 2, "d": 64}
LARGE = {"hq": 28, "hkv": 4, "d": 128}
GROUPS8 = {"hq": 32, "hkv": 4, "d": 128}
EPS = 1e-6


def listed():
    return [
        # a decode step of 64 chats: launch latency decides
        {"name": "rope-decode-bf16", "kind": "rope", **LARGE, "dtype": "bf16", "bs": 16, "shape": 1,
         "seqs": 64, "new_lo": 1, "new_hi": 1, "cached_lo": 1, "cached_hi": 4096},
        # eight 512-token prompt chunks
        {"name": "rope-prefill-bf16", "kind": "rope", **LARGE, "dtype": "bf16", "bs": 16, "shape": 2,
         "seqs": 8, "new_lo": 512, "new_hi": 512, "cached_lo": 0, "cached_hi": 4096},
        # prompts of odd lengths on a small model, fp32
        {"name": "rope-odd-fp32", "kind": "rope", **SMALL, "dtype": "fp32", "bs": 16, "shape": 3,
         "seqs": 11, "new_lo": 1, "new_hi": 140, "cached_lo": 0, "cached_hi": 900},
        # a decode step: one token more in blocks that are partly full
        {"name": "store-decode-bf16", "kind": "store", **LARGE, "dtype": "bf16", "bs": 16, "shape": 4,
         "seqs": 64, "new_lo": 1, "new_hi": 1, "cached_lo": 1, "cached_hi": 4096},
        # prompt chunks: whole blocks at once
        {"name": "store-prefill-bf16", "kind": "store", **LARGE, "dtype": "bf16", "bs": 16, "shape": 5,
         "seqs": 8, "new_lo": 512, "new_hi": 512, "cached_lo": 0, "cached_hi": 4096},
        # ragged chunks that begin and end inside blocks, larger blocks, fp16
        {"name": "store-odd-fp16", "kind": "store", **SMALL, "dtype": "fp16", "bs": 32, "shape": 6,
         "seqs": 23, "new_lo": 1, "new_hi": 130, "cached_lo": 0, "cached_hi": 700},
        # a handful of chats on the small model
        {"name": "decode-small-fp16", "kind": "decode", **SMALL, "dtype": "fp16", "bs": 16, "shape": 7,
         "seqs": 8, "cached_lo": 0, "cached_hi": 511},
        # 64 chats of 512..4096 tokens
        {"name": "decode-chats-bf16", "kind": "decode", **LARGE, "dtype": "bf16", "bs": 16, "shape": 8,
         "seqs": 64, "cached_lo": 511, "cached_hi": 4095},
        # few sequences with documents in their context: the keys have to be split
        {"name": "decode-long-bf16", "kind": "decode", **GROUPS8, "dtype": "bf16", "bs": 32, "shape": 9,
         "seqs": 3, "cached_lo": 20000, "cached_hi": 60000},
        # 512-token chunks after cached prefixes of up to 8k
        {"name": "prefill-chunks-bf16", "kind": "prefill", **LARGE, "dtype": "bf16", "bs": 16, "shape": 10,
         "seqs": 8, "new_lo": 512, "new_hi": 512, "cached_lo": 0, "cached_hi": 8192},
        # odd chunks of an fp32 model, some of one token
        {"name": "prefill-odd-fp32", "kind": "prefill", **SMALL, "dtype": "fp32", "bs": 16, "shape": 11,
         "seqs": 6, "new_lo": 1, "new_hi": 300, "cached_lo": 0, "cached_hi": 1500},
        # a layer of a continuous-batching step: 224 decode rows and four 256-token chunks
        {"name": "layer-mixed-bf16", "kind": "layer", **LARGE, "dtype": "bf16", "bs": 16, "shape": 12,
         "seqs": 4, "new_lo": 256, "new_hi": 256, "cached_lo": 0, "cached_hi": 2048, "rows": 224,
         "row_cached_lo": 255, "row_cached_hi": 4095},
    ]


def _spread(rng, lo, hi):
    """An integer of [lo, hi], its logarithm uniform."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["rope", "store", "decode", "prefill", "layer"])
    heads = rng.choice([SMALL, LARGE, GROUPS8, {"hq": 8, "hkv": 8, "d": 64}, {"hq": 20, "hkv": 1, "d": 128},
                        {"hq": 12, "hkv": 4, "d": 64}])
    case = {"kind": kind, **heads, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
            "bs": rng.choice([16, 16, 32, 64, 48]), "shape": rng.randrange(1 << 30)}
    if kind in ("rope", "store"):
        seqs = _spread(rng, 1, 64)
        most = max(1, 4096 // (seqs * (2 if case["dtype"] == "fp32" else 1)))
        hi = _spread(rng, 1, most)
        return case | {"seqs": seqs, "new_lo": rng.randint(1, hi), "new_hi": hi, "cached_lo": 0,
                       "cached_hi": _spread(rng, 1, 4000)}
    if kind == "decode":
        seqs = _spread(rng, 1, 64)
        hi = _spread(rng, 1, min(50000, 120000 // seqs))
        return case | {"seqs": seqs, "cached_lo": rng.randint(0, hi - 1), "cached_hi": hi}
    if kind == "layer" and case["dtype"] == "fp32":
        # (its keys are rounded to codes from fp32: a last-bit difference before that is a whole code after)
        case["dtype"] = "bf16"
    fp32 = case["dtype"] == "fp32"
    seqs, hi = _spread(rng, 1, 6), _spread(rng, 1, 200 if fp32 else 400)
    case |= {"seqs": seqs, "new_lo": rng.randint(1, hi), "new_hi": hi, "cached_lo": 0,
             "cached_hi": _spread(rng, 1, 1500 if fp32 else 4000)}
    if kind == "layer":
        rows = _spread(rng, 1, 64)
        case |= {"rows": rows, "row_cached_lo": 0, "row_cached_hi": _spread(rng, 1, min(4000, 100000 // rows))}
    return case


def _lengths(case):
    """(new tokens, tokens already cached) of each sequence; a layer's one-token rows come first."""
    rng = random.Random(case["shape"])
    both = [(1, rng.randint(case["row_cached_lo"], case["row_cached_hi"])) for _ in range(case.get("rows", 0))]
    new = case.get("new_lo", 1), case.get("new_hi", 1)
    return both + [(rng.randint(*new), rng.randint(case["cached_lo"], case["cached_hi"])) for _ in range(case["seqs"])]


# ---- inputs


def _exponent(amax, fp16):
    """Least k with amax <= 448 * 2^k (448 = 0.875 * 2^9), within the bounds of the type."""
    m, e = torch.frexp(amax)
    k = torch.where(m <= 0.875, e - 9, e - 8)
    lowest, highest = (-15, 8) if fp16 else (-100, 119)
    return torch.where(amax > 0, k, torch.full_like(k, lowest)).clamp(lowest, highest)


def _pow2(k):
    return ((k + 127).int() << 23).view(torch.float32)


def _history(case, gen, blocks):
    """Codes [2, H_kv, blocks, bs, D] and scales [H_kv, blocks, 2] of a filled cache."""
    hkv, d, bs = case["hkv"], case["d"], case["bs"]
    # keys have a few large channels, values none
    wide = torch.exp(0.5 * torch.randn(2, hkv, 1, 1, d, generator=gen, device="cuda"))
    wide[1] = 1.0
    x = torch.randn(2, hkv, blocks, bs, d, generator=gen, device="cuda").mul_(wide)
    k = _exponent(x.abs().amax((3, 4)), case["dtype"] == "fp16")
    codes = x.mul_(_pow2(-k)[..., None, None]).to(torch.float8_e4m3fn)
    return codes, _pow2(k).permute(1, 2, 0).contiguous()


def _inputs(case, seed):
    """The tensors of a pass, and the host's lists they come from."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    hq, hkv, d, bs = case["hq"], case["hkv"], case["d"], case["bs"]
    dtype = DTYPES[case["dtype"]]
    lens = _lengths(case)
    need = [-(-(n + c) // bs) for n, c in lens]
    blocks = sum(need) + sum(need) // 4 + 1
    ids = rng.sample(range(blocks), sum(need))
    tables = [[ids.pop() for _ in range(n)] for n in need]
    s = {"tables": tables, "new": [n for n, _ in lens], "cached": [c for _, c in lens], "scale": d**-0.5}
    width = max(need)
    s["bt"] = torch.tensor([t + [0] * (width - len(t)) for t in tables], dtype=torch.int32, device="cuda")
    s["ctx"] = torch.tensor([n + c for n, c in lens], dtype=torch.int32, device="cuda")
    s["start"] = torch.tensor(s["cached"], dtype=torch.int32, device="cuda")
    total = sum(s["new"])
    if case["kind"] in ("decode", "prefill"):
        s["q"] = torch.randn(total, hq, d, generator=gen, device="cuda").to(dtype)
    else:
        # q, k and v are slices of one projection's rows
        qkv = torch.randn(total, hq + 2 * hkv, d, generator=gen, device="cuda").to(dtype)
        s["q"], s["k"], s["v"] = qkv.split([hq, hkv, hkv], dim=1)
        pos = torch.tensor([p for n, c in lens for p in range(c, c + n)], dtype=torch.float64, device="cuda")
        freq = 1e6 ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
        angle = torch.cat([pos[:, None] * freq] * 2, dim=1)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["q_norm"] = (1 + 0.2 * torch.randn(d, generator=gen, device="cuda")).to(dtype)
        s["k_norm"] = (1 + 0.2 * torch.randn(d, generator=gen, device="cuda")).to(dtype)
        s["slots"] = torch.tensor(
            [t[p // bs] * bs + p % bs for t, (n, c) in zip(tables, lens) for p in range(c, c + n)], device="cuda")
    if case["kind"] == "rope":
        s["kc"], s["vc"] = torch.zeros(2, hkv, blocks * bs, d, dtype=dtype, device="cuda").transpose(1, 2)
    else:
        s["codes"], s["scales"] = _history(case, gen, blocks)
    if case["kind"] == "store":
        # every slot of the blocks that the new tokens fall into
        touched = [t[j] for t, (n, c) in zip(tables, lens) for j in range(c // bs, (c + n - 1) // bs + 1)]
        s["read"] = torch.tensor([b * bs + o for b in touched for o in range(bs)], device="cuda")
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    kind, dtype, bs = case["kind"], DTYPES[case["dtype"]], case["bs"]
    if kind in ("prefill", "layer"):
        s["cu"] = torch.tensor([sum(s["new"][:i]) for i in range(len(s["new"]) + 1)], dtype=torch.int32, device="cuda")
    if own and kind != "rope":
        from infrared_amd import QuantPagedKVPool, kernels, metadata

        blocks = s["scales"].shape[1]
        pool = QuantPagedKVPool(1, blocks, bs, case["hkv"], case["d"], dtype)
        pool.k[0].copy_(s["codes"][0].flatten(1, 2).transpose(0, 1))
        pool.v[0].copy_(s["codes"][1].flatten(1, 2).transpose(0, 1))
        pool.kv_scales[0].copy_(s["scales"])
        del s["codes"], s["scales"]
        s["pool"] = pool
        hq, hkv, d = case["hq"], case["hkv"], case["d"]
        nseq, width = s["bt"].shape
        s["plan"] = s["work"] = s["counters"] = None
        # what a step shares over its layers: the work plan, the workspace
        if kind == "decode":
            s["counters"] = pool.decode_counters(kernels.decode_num_counters(nseq, hq, hkv))
            if kernels.decode_plan_pays(nseq, hq, hkv, width, bs, "cuda"):
                s["plan"] = kernels.decode_plan(s["bt"], s["ctx"], hq, pool.k[0], bs)
                s["work"] = pool.workspace(kernels.planned_workspace_bytes(nseq, hq, hkv, d))
            else:
                s["work"] = pool.workspace(kernels.decode_workspace_bytes(nseq, hq, hkv, d, width, bs))
        if kind == "prefill":
            longest = max(s["new"])
            if kernels.prefill_plan_pays(nseq, longest, hq, hkv, "cuda", max_keys=width * bs, dtype=dtype):
                s["plan"] = kernels.prefill_plan(s["cu"], s["start"], s["bt"], len(s["q"]), longest, bs, hq, hkv, d,
                                                 dtype=dtype)
        if kind == "layer":
            s["paged"], _ = metadata.prefill_context(pool, s["tables"], s["cached"], s["new"])
    return s


def run(s):
    return _run_own(s) if own else _PLAIN[s["case"]["kind"]](s)


def _run_own(s):
    from infrared_amd import kernels, rope_paged_attention

    case, kind = s["case"], s["case"]["kind"]
    if kind == "rope":
        q = kernels.qk_norm_rope_kv_scatter(s["q"], s["k"], s["v"], s["q_norm"], s["k_norm"], EPS, s["cos"], s["sin"],
                                            s["kc"], s["vc"], s["slots"])
        return q, s["kc"], s["vc"]
    pool = s["pool"]
    if kind == "store":
        pool.write(0, s["k"], s["v"], s["slots"])
        return pool.gather(0, s["read"])
    if kind == "decode" and s["plan"] is not None:
        return kernels.paged_decode_planned(s["q"], pool.k[0], pool.v[0], s["plan"], s["scale"], workspace=s["work"],
                                            counters=s["counters"], kv_scales=pool.kv_scales[0])
    if kind == "decode":
        return kernels.paged_decode(s["q"], pool.k[0], pool.v[0], s["bt"], s["ctx"], case["bs"], s["scale"],
                                    workspace=s["work"], counters=s["counters"], kv_scales=pool.kv_scales[0])
    if kind == "prefill":
        return kernels.paged_prefill(s["q"], pool.k[0], pool.v[0], s["bt"], s["cu"], s["start"], max(s["new"]),
                                     case["bs"], s["scale"], plan=s["plan"], kv_scales=pool.kv_scales[0])
    out = rope_paged_attention(s["q"][None], s["k"][None], s["v"][None], s["cos"][None], s["sin"][None], s["paged"],
                               None, 0, s["scale"], case["hq"] // case["hkv"], q_norm=s["q_norm"],
                               k_norm=s["k_norm"], eps=EPS)
    return (out[0], *pool.gather(0, s["slots"]))


# ---- plain forms


def _norm_rope(x, w, cos, sin):
    x = x.float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    half = y.shape[-1] // 2
    turned = torch.cat([-y[..., half:], y[..., :half]], dim=-1)
    return y * cos[:, None] + turned * sin[:, None]


def _plain_rope(s):
    q = _norm_rope(s["q"], s["q_norm"], s["cos"], s["sin"]).to(s["q"].dtype)
    s["kc"][s["slots"]] = _norm_rope(s["k"], s["k_norm"], s["cos"], s["sin"]).to(s["k"].dtype)
    s["vc"][s["slots"]] = s["v"]
    return q, s["kc"], s["vc"]


def _plain_write(s, new):
    """Quantises ``new`` [2, n, H_kv, D] (fp32) into the slots of the codes and scales."""
    bs, fp16 = s["case"]["bs"], s["case"]["dtype"] == "fp16"
    codes, scales, slots = s["codes"], s["scales"], s["slots"]
    ids, at = torch.unique(slots // bs, return_inverse=True)
    amax = torch.zeros(2, len(ids), new.shape[2], device=new.device)
    amax.index_reduce_(1, at, new.abs().amax(-1), "amax")
    fresh = torch.zeros(len(ids), device=new.device).index_add_(0, at, (slots % bs == 0).float()) > 0
    need = _exponent(amax, fp16).transpose(1, 2)  # [2, H_kv, touched]
    old = scales[:, ids].permute(2, 0, 1)
    held = torch.frexp(old)[1] - 1
    k = torch.where(fresh, need, torch.maximum(held, need))
    kept = codes[:, :, ids].float() * torch.where(fresh, torch.zeros_like(old), old)[..., None, None]
    limit = 61440.0 if fp16 else 448.0 * 2.0**119
    kept[:, :, at, slots % bs] = new.transpose(1, 2).clamp(-limit, limit)
    codes[:, :, ids] = (kept * _pow2(-k)[..., None, None]).to(codes.dtype)
    scales[:, ids] = _pow2(k).permute(1, 2, 0)


def _plain_read(s, slots):
    bs = s["case"]["bs"]
    x = s["codes"][:, :, slots // bs, slots % bs].float() * s["scales"][:, slots // bs].permute(2, 0, 1)[..., None]
    k, v = x.transpose(1, 2).to(DTYPES[s["case"]["dtype"]])
    return k, v


def _plain_store(s):
    _plain_write(s, torch.stack([s["k"], s["v"]]).float())
    return _plain_read(s, s["read"])


def _attend(s, q, at, bt, pos):
    """Attention of the query tokens ``q`` [n, H_q, D] (fp32): ``at`` is each one's row of
    ``bt`` and place in it, ``pos`` [rows, longest] the position each place attends up to."""
    hkv, d, bs = s["case"]["hkv"], s["case"]["d"], s["case"]["bs"]
    rows, width = bt.shape
    x = s["codes"][:, :, bt].float() * s["scales"][:, bt].permute(3, 0, 1, 2)[..., None, None]
    k, v = x.reshape(2, hkv, rows, width * bs, d)
    queries = torch.zeros(rows, pos.shape[1], hkv, q.shape[1] // hkv, d, device=q.device)
    queries[at] = q.unflatten(1, (hkv, -1)) * s["scale"]
    queries = queries.permute(2, 0, 1, 3, 4).flatten(2, 3)  # [H_kv, rows, places * group, D]
    scores = (queries @ k.transpose(2, 3)).unflatten(2, (pos.shape[1], -1))
    hidden = torch.arange(width * bs, device=q.device) > pos[:, :, None]
    scores.masked_fill_(hidden[None, :, :, None], float("-inf"))
    scores -= scores.amax(-1, keepdim=True)
    weights = scores.exp_()
    weights /= weights.sum(-1, keepdim=True)
    out = (weights.flatten(2, 3) @ v).unflatten(2, (pos.shape[1], -1))
    return out.permute(1, 2, 0, 3, 4)[at].flatten(1, 2)


def _plain_decode(s):
    one = torch.zeros_like(s["ctx"], dtype=torch.long)
    at = (torch.arange(len(one), device=one.device), one)
    return _attend(s, s["q"].float(), at, s["bt"].long(), (s["ctx"].long() - 1)[:, None]).to(s["q"].dtype)


def _plain_chunks(s, q, first):
    """Attention of the packed chunks of the sequences ``first``.. (fp32)."""
    cu = s["cu"].long()[first:] - s["cu"].long()[first]
    new = cu.diff()
    row = torch.repeat_interleave(torch.arange(len(new), device=q.device), new, output_size=len(q))
    place = torch.arange(len(q), device=q.device) - cu[row]
    longest = max(s["new"][first:])
    pos = s["start"].long()[first:, None] + torch.arange(longest, device=q.device)
    width = max(len(t) for t in s["tables"][first:])
    return _attend(s, q, (row, place), s["bt"].long()[first:, :width], pos)


def _plain_prefill(s):
    return _plain_chunks(s, s["q"].float(), 0).to(s["q"].dtype)


def _plain_layer(s):
    rows, dtype = s["case"]["rows"], s["q"].dtype
    q = _norm_rope(s["q"], s["q_norm"], s["cos"], s["sin"])
    _plain_write(s, torch.stack([_norm_rope(s["k"], s["k_norm"], s["cos"], s["sin"]), s["v"].float()]))
    one = torch.zeros(rows, dtype=torch.long, device=q.device)
    at = (torch.arange(rows, device=q.device), one)
    width = max(len(t) for t in s["tables"][:rows])
    out = torch.cat([_attend(s, q[:rows], at, s["bt"].long()[:rows, :width], s["start"].long()[:rows, None]),
                     _plain_chunks(s, q[rows:], rows)])
    return (out.to(dtype), *_plain_read(s, s["slots"]))


_PLAIN = {"rope": _plain_rope, "store": _plain_store, "decode": _plain_decode, "prefill": _plain_prefill,
          "layer": _plain_layer}


# ---- what a pass cannot do without


def work(case):
    lens = _lengths(case)
    es, hq, hkv, d, bs = ESIZE[case["dtype"]], case["hq"], case["hkv"], case["d"], case["bs"]
    n = sum(a for a, _ in lens)
    touched = sum((c + a - 1) // bs - c // bs + 1 for a, c in lens)
    row, scale = 2 * hkv * d, 8 * hkv  # bytes of a token's codes, of a block's scales
    nbytes = flops = 0
    if case["kind"] in ("rope", "layer"):
        nbytes += n * (hq + 2 * hkv) * d * es + 8 * n * d + 2 * d * es + 8 * n
        flops += 10 * n * (hq + hkv) * d
    if case["kind"] == "rope":
        nbytes += n * (hq + 2 * hkv) * d * es
    if case["kind"] == "store":
        nbytes += n * row * es + 8 * n
        nbytes += touched * (bs * row * (1 + es) + 8 * bs)
    if case["kind"] in ("store", "layer"):
        nbytes += n * row + 2 * touched * scale
    if case["kind"] == "layer":
        nbytes += n * row * (1 + es)
    if case["kind"] in ("decode", "prefill", "layer"):
        keys = sum(a + c for a, c in lens)
        nbytes += keys * row + sum(-(-(a + c) // bs) for a, c in lens) * (scale + 4)
        nbytes += n * hq * d * es * (1 if case["kind"] == "layer" else 2)
        flops += 4 * hq * d * sum(a * c + a * (a + 1) // 2 for a, c in lens)
    return {"bytes": nbytes, "flops": flops}


# ---- the definition in 64 bits


def _exact_values(x, fp16):
    """The values an 8-bit block [tokens, D] of the numbers x holds, and their scale's exponent."""
    amax = x.abs().max().item()
    low, high = (-15, 8) if fp16 else (-100, 119)
    k = low
    while 448.0 * 2.0**k < amax and k < high:
        k += 1
    return _exact_round(x, k, fp16), k


def _exact_round(x, k, fp16):
    """x to the nearest multiple of 2^(k - 9) with four significant bits, ties to even."""
    x = x.clamp(-61440.0, 61440.0) if fp16 else x.clamp(-448.0 * 2.0**119, 448.0 * 2.0**119)
    e = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** (k - 6))))
    e = torch.where(torch.exp2(e + 1) <= x.abs(), e + 1, e)
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def _exact_rope(x, w, cos, sin):
    x, w, cos, sin = x.double(), w.double(), cos.double()[:, None], sin.double()[:, None]
    y = w * x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS)
    a, b = y.chunk(2, dim=-1)
    c1, c2 = cos.chunk(2, dim=-1)
    s1, s2 = sin.chunk(2, dim=-1)
    return torch.cat([a * c1 - b * s1, b * c2 + a * s2], dim=-1)


def _exact_cache(s):
    """Values [2, slots, H_kv, D] of the cache as it is before the pass."""
    x = s["codes"].double() * s["scales"].double().permute(2, 0, 1)[..., None, None]
    return x.flatten(2, 3).transpose(1, 2).contiguous()


def _exact_write(s, cache, new):
    """The cache's values after the new rows [2, n, H_kv, D] went into their slots."""
    bs, fp16 = s["case"]["bs"], s["case"]["dtype"] == "fp16"
    by_block = {}
    for i, slot in enumerate(s["slots"].tolist()):
        by_block.setdefault(slot // bs, []).append((i, slot % bs))
    log2 = s["scales"].double().log2().round().long().tolist()
    for b, rows in by_block.items():
        i, o = [r[0] for r in rows], [r[1] for r in rows]
        block = cache[:, b * bs:(b + 1) * bs]
        if 0 in o:
            block.zero_()
        for kv in range(2):
            for h in range(new.shape[2]):
                x = new[kv, i, h]
                value, k = _exact_values(x, fp16)
                held = log2[h][b][kv]
                if 0 not in o and held >= k:
                    value = _exact_round(x, held, fp16)
                elif 0 not in o:
                    block[kv, :, h] = _exact_round(block[kv, :, h], k, fp16)
                block[kv, o, h] = value


def _exact_attend(s, q, cache):
    bs, hkv = s["case"]["bs"], s["case"]["hkv"]
    out, row = [], 0
    for table, n, c in zip(s["tables"], s["new"], s["cached"]):
        t = torch.arange(n + c, device=q.device)
        k, v = cache[:, torch.tensor(table, device=q.device)[t // bs] * bs + t % bs].transpose(1, 2)
        x = q[row:row + n].double().unflatten(1, (hkv, -1)).permute(1, 2, 0, 3)  # [H_kv, group, n, D]
        scores = torch.matmul(x, k.transpose(1, 2)[:, None]) * s["scale"]
        scores = torch.where(t <= torch.arange(c, c + n, device=q.device)[:, None], scores, -torch.inf)
        out.append(torch.matmul(torch.softmax(scores, -1), v[:, None]).permute(2, 0, 1, 3).flatten(1, 2))
        row += n
    return torch.cat(out)


def exact(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    kind, slots = case["kind"], s.get("slots")
    if kind in ("store", "layer") and 2 * case["hkv"] * sum(-(-a // case["bs"]) + 1 for a, _ in _lengths(case)) > 20000:
        return None
    if kind == "rope":
        kc, vc = s["kc"].double(), s["vc"].double()
        kc[slots] = _exact_rope(s["k"], s["k_norm"], s["cos"], s["sin"])
        vc[slots] = s["v"].double()
        return _exact_rope(s["q"], s["q_norm"], s["cos"], s["sin"]), kc, vc
    cache = _exact_cache(s)
    if kind == "store":
        _exact_write(s, cache, torch.stack([s["k"], s["v"]]).double())
        return cache[0, s["read"]], cache[1, s["read"]]
    if kind == "layer":
        k = _exact_rope(s["k"], s["k_norm"], s["cos"], s["sin"])
        _exact_write(s, cache, torch.stack([k, s["v"].double()]))
        q = _exact_rope(s["q"], s["q_norm"], s["cos"], s["sin"])
        return _exact_attend(s, q, cache), cache[0, slots], cache[1, slots]
    return _exact_attend(s, s["q"], cache)
