"""Operators of a layer whose K/V cache is held in 4 bits and whose tokens have a
position for each of several axes, measured through the framework's public calls
(``own``) or as plain torch operations.

- ``turn``: queries and keys rotated by positions with several axes, optionally normed
  for each head before, the keys and values written to a 16- or 32-bit pool.
- ``patch``: the same rotation of an image encoder's rows, without a cache.
- ``store``: the step's new K/V quantised into a 4-bit pool, and the blocks they fell
  into read back.
- ``decode`` / ``prefill``: attention over a 4-bit pool, for one query token a
  sequence and for packed chunks after cached prefixes.

The cache: of each token, KV head and K or V, groups of 32 channels share a scale
``2^k``, ``k`` the least integer with ``amax <= 7 * 2^k``, in [-100, 125] (fp16: [-23,
13]). A value is the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the even code,
nothing above 6) times the scale.

The rotation: pair ``j`` of a head, elements ``j`` and ``j + D/2``, turns by
``position[axis of j] * inv_freq[j]``.
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
        # a decode step of 64 chats about images: launch latency decides
        {"name": "turn-decode-bf16", "kind": "turn", **LARGE, "dtype": "bf16", "bs": 16, "shape": 1, "norm": True,
         "sections": "16,24,24", "theta": 1e6, "seqs": 64, "new_lo": 1, "new_hi": 1, "cached_lo": 1, "cached_hi": 30000},
        # eight 512-token prompt chunks, text and images
        {"name": "turn-prompt-bf16", "kind": "turn", **LARGE, "dtype": "bf16", "bs": 16, "shape": 2, "norm": False,
         "sections": "16,24,24", "theta": 1e6, "seqs": 8, "new_lo": 512, "new_hi": 512, "cached_lo": 0,
         "cached_hi": 4096},
        # odd chunks far into long videos on a small model, fp32
        {"name": "turn-odd-fp32", "kind": "turn", **SMALL, "dtype": "fp32", "bs": 16, "shape": 3, "norm": True,
         "sections": "8,12,12", "theta": 1e6, "seqs": 11, "new_lo": 1, "new_hi": 140, "cached_lo": 0,
         "cached_hi": 900000},
        # four images of up to 60 x 60 patches in an encoder with heads of 80, rows and columns as axes
        {"name": "patch-images-fp16", "kind": "patch", "hq": 16, "hkv": 16, "d": 80, "dtype": "fp16", "shape": 4,
         "norm": False, "sections": "20,20", "theta": 1e4, "seqs": 4, "new_lo": 1200, "new_hi": 3600},
        # a decode step: one token more in blocks that are partly full
        {"name": "store-decode-bf16", "kind": "store", **LARGE, "dtype": "bf16", "bs": 16, "shape": 5,
         "seqs": 64, "new_lo": 1, "new_hi": 1, "cached_lo": 1, "cached_hi": 4096},
        # prompt chunks: whole blocks at once
        {"name": "store-prefill-bf16", "kind": "store", **LARGE, "dtype": "bf16", "bs": 16, "shape": 6,
         "seqs": 8, "new_lo": 512, "new_hi": 512, "cached_lo": 0, "cached_hi": 4096},
        # ragged chunks that begin and end inside blocks, larger blocks, fp16
        {"name": "store-odd-fp16", "kind": "store", **SMALL, "dtype": "fp16", "bs": 32, "shape": 7,
         "seqs": 23, "new_lo": 1, "new_hi": 130, "cached_lo": 0, "cached_hi": 700},
        # a handful of chats on the small model
        {"name": "decode-small-fp16", "kind": "decode", **SMALL, "dtype": "fp16", "bs": 16, "shape": 8,
         "seqs": 8, "cached_lo": 0, "cached_hi": 511},
        # 64 chats of 512..4096 tokens
        {"name": "decode-chats-bf16", "kind": "decode", **LARGE, "dtype": "bf16", "bs": 16, "shape": 9,
         "seqs": 64, "cached_lo": 511, "cached_hi": 4095},
        # few sequences with documents in their context: the keys have to be split
        {"name": "decode-long-bf16", "kind": "decode", **GROUPS8, "dtype": "bf16", "bs": 32, "shape": 10,
         "seqs": 3, "cached_lo": 40000, "cached_hi": 90000},
        # 512-token chunks after cached prefixes of up to 8k
        {"name": "prefill-chunks-bf16", "kind": "prefill", **LARGE, "dtype": "bf16", "bs": 16, "shape": 11,
         "seqs": 8, "new_lo": 512, "new_hi": 512, "cached_lo": 0, "cached_hi": 8192},
        # odd chunks of an fp32 model, some of one token
        {"name": "prefill-odd-fp32", "kind": "prefill", **SMALL, "dtype": "fp32", "bs": 16, "shape": 12,
         "seqs": 6, "new_lo": 1, "new_hi": 300, "cached_lo": 0, "cached_hi": 1500},
    ]


def _spread(rng, lo, hi):
    """An integer of [lo, hi], its logarithm uniform."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def _split(rng, total, axes):
    """``total`` in ``axes`` parts, each at least one, as a text."""
    cuts = sorted(rng.sample(range(1, total), axes - 1))
    return ",".join(str(b - a) for a, b in zip([0, *cuts], [*cuts, total]))


def draw(rng):
    kind = rng.choice(["turn", "patch", "store", "decode", "prefill"])
    case = {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "shape": rng.randrange(1 << 30)}
    if kind == "patch":
        heads = rng.choice([8, 12, 16])
        d = rng.choice([64, 80, 96, 128])
        seqs = _spread(rng, 1, 8)
        hi = _spread(rng, 9, 3600 // seqs)
        return case | {"hq": heads, "hkv": heads, "d": d, "norm": False, "sections": _split(rng, d // 2, 2),
                       "theta": 1e4, "seqs": seqs, "new_lo": rng.randint(1, hi), "new_hi": hi}
    case |= rng.choice([SMALL, LARGE, GROUPS8, {"hq": 8, "hkv": 8, "d": 64}, {"hq": 20, "hkv": 1, "d": 128},
                        {"hq": 12, "hkv": 4, "d": 64}])
    case["bs"] = rng.choice([16, 16, 32, 64, 48])
    if kind in ("turn", "store"):
        seqs = _spread(rng, 1, 64)
        most = max(1, 4096 // (seqs * (2 if case["dtype"] == "fp32" else 1)))
        hi = _spread(rng, 1, most)
        case |= {"seqs": seqs, "new_lo": rng.randint(1, hi), "new_hi": hi, "cached_lo": 0,
                 "cached_hi": _spread(rng, 1, 4000)}
    if kind == "turn":
        case |= {"norm": rng.random() < 0.5, "sections": _split(rng, case["d"] // 2, rng.choice([1, 2, 3, 4])),
                 "theta": rng.choice([1e4, 1e6]), "cached_hi": _spread(rng, 1, 900000)}
    if kind == "decode":
        seqs = _spread(rng, 1, 64)
        hi = _spread(rng, 1, min(90000, 140000 // seqs))
        case |= {"seqs": seqs, "cached_lo": rng.randint(0, hi - 1), "cached_hi": hi}
    if kind == "prefill":
        fp32 = case["dtype"] == "fp32"
        seqs, hi = _spread(rng, 1, 6), _spread(rng, 1, 200 if fp32 else 400)
        case |= {"seqs": seqs, "new_lo": rng.randint(1, hi), "new_hi": hi, "cached_lo": 0,
                 "cached_hi": _spread(rng, 1, 1500 if fp32 else 4000)}
    return case


def _lengths(case):
    """(new tokens, tokens already cached) of each sequence."""
    rng = random.Random(case["shape"])
    new, cached = (case.get("new_lo", 1), case.get("new_hi", 1)), (case.get("cached_lo", 0), case.get("cached_hi", 0))
    return [(rng.randint(*new), rng.randint(*cached)) for _ in range(case["seqs"])]


def _held(case):
    """Tokens of each sequence that its block table covers: where nothing is attended and only
    the blocks of the new tokens matter, at most the last 5,000 before them."""
    most = 1 << 30 if case["kind"] in ("decode", "prefill") else 5000
    return [n + min(c, most) for n, c in _lengths(case)]


# ---- inputs


def _positions(case, seed):
    """Positions [axes][tokens]: runs of text, whose axes are equal, and images, whose later
    axes count rows and columns and whose first one stands still."""
    rng = random.Random(seed)
    axes = case["sections"].count(",") + 1
    out = [[] for _ in range(axes)]
    for n, at in _lengths(case):
        left = n
        while left:
            if case["kind"] == "patch":
                width, run = max(1, round(left**0.5)), left
            else:
                width, run = rng.randint(1, 24), min(left, rng.randint(1, 200))
            if case["kind"] == "patch" or (axes > 1 and rng.random() < 0.5):
                still = axes - 2 if axes > 2 else 0
                for a in range(axes):
                    out[a] += [at if a < still else at + (i // width if a == axes - 2 else i % width)
                               for i in range(run)]
                at += max(width, run // width + 1)
            else:
                for a in range(axes):
                    out[a] += range(at, at + run)
                at += run
            left -= run
    return torch.tensor(out, device="cuda")


def _frequencies(case):
    """(inv_freq, axis) of each pair. An encoder's axes each have a run of frequencies of their
    own; a language model's run on from one axis to the next."""
    sections = [int(n) for n in case["sections"].split(",")]
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    if case["kind"] == "patch":
        return [case["theta"] ** (-j / n) for n in sections for j in range(n)], axis
    return [case["theta"] ** (-j / len(axis)) for j in range(len(axis))], axis


def _exponent(amax, fp16):
    """Least k with amax <= 7 * 2^k (7 = 0.875 * 2^3), within the bounds of the type."""
    m, e = torch.frexp(amax)
    k = torch.where(m <= 0.875, e - 3, e - 2)
    lowest, highest = (-23, 13) if fp16 else (-100, 125)
    return torch.where(amax > 0, k, torch.full_like(k, lowest)).clamp(lowest, highest)


def _pow2(k):
    return ((k.int() + 127) << 23).view(torch.float32)


def _quantise(x, fp16):
    """Twice the codes' numbers (whole) of ``x`` [.., D] and the exponents [.., D / 32], as bytes."""
    groups = x.float().unflatten(-1, (-1, 32))
    k = _exponent(groups.abs().amax(-1), fp16)
    y = groups * _pow2(-k)[..., None]
    step = _pow2(torch.frexp(y.abs().clamp_min(1.0))[1] - 2)  # 0.5 below 2, 1 below 4, 2 from there
    y = (torch.round(y / step) * step).clamp(-6.0, 6.0)
    return (2 * y).to(torch.int8).flatten(-2), k.to(torch.int8)


def _values(codes, k):
    """The numbers that codes and exponents stand for (fp32)."""
    return (codes.float().unflatten(-1, (-1, 32)) * _pow2(k - 1)[..., None]).flatten(-2)


def _inputs(case, seed):
    """The tensors of a pass, and the host's lists they come from."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    kind, hq, hkv, d = case["kind"], case["hq"], case["hkv"], case["d"]
    dtype = DTYPES[case["dtype"]]
    lens = _lengths(case)
    total = sum(n for n, _ in lens)
    s = {"case": case, "new": [n for n, _ in lens], "cached": [c for _, c in lens], "scale": d**-0.5}
    if kind in ("decode", "prefill"):
        s["q"] = torch.randn(total, hq, d, generator=gen, device="cuda").to(dtype)
    else:
        # q, k and v are slices of one projection's rows
        qkv = torch.randn(total, hq + 2 * hkv, d, generator=gen, device="cuda").to(dtype)
        s["q"], s["k"], s["v"] = qkv.split([hq, hkv, hkv], dim=1)
    if kind in ("turn", "patch"):
        s["pos"] = _positions(case, seed)
        s["q_norm"] = s["k_norm"] = None
        if case["norm"]:
            s["q_norm"] = (1 + 0.2 * torch.randn(d, generator=gen, device="cuda")).to(dtype)
            s["k_norm"] = (1 + 0.2 * torch.randn(d, generator=gen, device="cuda")).to(dtype)
    if kind == "patch":
        return s
    bs = case["bs"]
    held = _held(case)
    need = [-(-h // bs) for h in held]
    blocks = sum(need) + sum(need) // 4 + 1
    ids = rng.sample(range(blocks), sum(need))
    s["tables"] = tables = [[ids.pop() for _ in range(n)] for n in need]
    width = max(need)
    s["bt"] = torch.tensor([t + [0] * (width - len(t)) for t in tables], dtype=torch.int32, device="cuda")
    s["ctx"] = torch.tensor([n + c for n, c in lens], dtype=torch.int32, device="cuda")
    s["start"] = torch.tensor(s["cached"], dtype=torch.int32, device="cuda")
    if kind in ("decode", "prefill"):
        s["cu"] = torch.tensor([sum(s["new"][:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")
    else:
        s["slots"] = torch.tensor([t[p // bs] * bs + p % bs for t, h, (n, _) in zip(tables, held, lens)
                                   for p in range(h - n, h)], device="cuda")
    if kind == "turn":
        s["kc"], s["vc"] = torch.zeros(2, hkv, blocks * bs, d, dtype=dtype, device="cuda").transpose(1, 2)
        return s
    # keys have a few large channels, values none
    wide = torch.exp(0.5 * torch.randn(2, hkv, 1, 1, d, generator=gen, device="cuda"))
    wide[1] = 1.0
    x = torch.randn(2, hkv, blocks, bs, d, generator=gen, device="cuda").mul_(wide)
    s["codes"], s["exps"] = _quantise(x, case["dtype"] == "fp16")
    if kind == "store":
        # every slot of the blocks that the new tokens fall into
        touched = [t[j] for t, h, (n, _) in zip(tables, held, lens) for j in range((h - n) // bs, (h - 1) // bs + 1)]
        s["read"] = torch.tensor([b * bs + o for b in touched for o in range(bs)], device="cuda")
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    if kind in ("turn", "patch"):
        freq, axis = _frequencies(case)
        if own:
            from infrared_amd import RotaryAxes

            s["rotary"] = RotaryAxes(freq, axis)
        else:
            s["freq"] = torch.tensor(freq, dtype=torch.float64, device="cuda")
            s["axis"] = torch.tensor(axis, device="cuda")
    elif own:
        from infrared_amd import Quant4PagedKVPool, kernels

        hq, hkv, d, bs = case["hq"], case["hkv"], case["d"], case["bs"]
        nseq, width = s["bt"].shape
        blocks = s["codes"].shape[2]
        s["pool"] = pool = Quant4PagedKVPool(1, blocks, bs, hkv, d, dtype)
        rows = _values(s.pop("codes"), s.pop("exps")).to(dtype).flatten(2, 3).transpose(1, 2)
        pool.write(0, rows[0], rows[1], torch.arange(blocks * bs, device="cuda"))
        del rows
        s["plan"] = s["work"] = s["counters"] = None
        # what a step shares over its layers: the work plan, the workspace
        if kind == "decode":
            s["counters"] = pool.decode_counters(kernels.decode_num_counters(nseq, hq, hkv))
            if kernels.decode_plan_pays(nseq, hq, hkv, width, bs, "cuda", pool.bits):
                s["plan"] = kernels.decode_plan(s["bt"], s["ctx"], hq, pool.k[0], bs)
                s["work"] = pool.workspace(kernels.planned_workspace_bytes(nseq, hq, hkv, d))
            else:
                s["work"] = pool.workspace(kernels.decode_workspace_bytes(nseq, hq, hkv, d, width, bs))
        if kind == "prefill":
            longest = max(s["new"])
            if kernels.prefill_plan_pays(nseq, longest, hq, hkv, "cuda", max_keys=width * bs, dtype=dtype):
                s["plan"] = kernels.prefill_plan(s["cu"], s["start"], s["bt"], len(s["q"]), longest, bs, hq, hkv, d,
                                                 dtype=dtype)
    return s


def run(s):
    return _run_own(s) if own else _PLAIN[s["case"]["kind"]](s)


def _run_own(s):
    from infrared_amd import kernels

    case, kind = s["case"], s["case"]["kind"]
    if kind == "patch":
        return kernels.rope_axes(s["q"], s["k"], s["pos"], s["rotary"])
    if kind == "turn":
        q = kernels.rope_axes_kv_scatter(s["q"], s["k"], s["v"], s["pos"], s["rotary"], s["kc"], s["vc"], s["slots"],
                                         s["q_norm"], s["k_norm"], EPS)
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
    return kernels.paged_prefill(s["q"], pool.k[0], pool.v[0], s["bt"], s["cu"], s["start"], max(s["new"]),
                                 case["bs"], s["scale"], plan=s["plan"], kv_scales=pool.kv_scales[0])


# ---- plain forms


def _turn(x, w, cos, sin):
    """The rows x [n, heads, D], normed if there is a weight and turned (fp32)."""
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _angles(s):
    angle = s["pos"][s["axis"]].double().T * s["freq"]
    return angle.cos().float()[:, None], angle.sin().float()[:, None]


def _plain_patch(s):
    cos, sin = _angles(s)
    return _turn(s["q"], None, cos, sin).to(s["q"].dtype), _turn(s["k"], None, cos, sin).to(s["k"].dtype)


def _plain_turn(s):
    cos, sin = _angles(s)
    q = _turn(s["q"], s["q_norm"], cos, sin).to(s["q"].dtype)
    s["kc"][s["slots"]] = _turn(s["k"], s["k_norm"], cos, sin).to(s["k"].dtype)
    s["vc"][s["slots"]] = s["v"]
    return q, s["kc"], s["vc"]


def _plain_store(s):
    bs, dtype = s["case"]["bs"], s["k"].dtype
    block, place = s["slots"] // bs, s["slots"] % bs
    codes, exps = _quantise(torch.stack([s["k"], s["v"]]).transpose(1, 2), dtype == torch.float16)
    s["codes"][:, :, block, place] = codes
    s["exps"][:, :, block, place] = exps
    block, place = s["read"] // bs, s["read"] % bs
    k, v = _values(s["codes"][:, :, block, place], s["exps"][:, :, block, place]).transpose(1, 2).to(dtype)
    return k, v


def _attend(s, q, at, pos):
    """Attention of the query tokens ``q`` [n, H_q, D] (fp32): ``at`` is each one's sequence and
    place in it, ``pos`` [sequences, longest] the position each place attends up to."""
    hkv, d, bs = s["case"]["hkv"], s["case"]["d"], s["case"]["bs"]
    bt = s["bt"].long()
    rows, width = bt.shape
    k, v = _values(s["codes"][:, :, bt], s["exps"][:, :, bt]).reshape(2, hkv, rows, width * bs, d)
    queries = torch.zeros(rows, pos.shape[1], hkv, q.shape[1] // hkv, d, device=q.device)
    queries[at] = q.unflatten(1, (hkv, -1)) * s["scale"]
    queries = queries.permute(2, 0, 1, 3, 4).flatten(2, 3)  # [H_kv, sequences, places * group, D]
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
    return _attend(s, s["q"].float(), at, (s["ctx"].long() - 1)[:, None]).to(s["q"].dtype)


def _plain_prefill(s):
    q, cu = s["q"], s["cu"].long()
    new = cu.diff()
    row = torch.repeat_interleave(torch.arange(len(new), device=q.device), new, output_size=len(q))
    place = torch.arange(len(q), device=q.device) - cu[row]
    pos = s["start"].long()[:, None] + torch.arange(max(s["new"]), device=q.device)
    return _attend(s, q.float(), (row, place), pos).to(q.dtype)


_PLAIN = {"turn": _plain_turn, "patch": _plain_patch, "store": _plain_store, "decode": _plain_decode,
          "prefill": _plain_prefill}


# ---- what a pass cannot do without


def work(case):
    lens = _lengths(case)
    kind, es, hq, hkv, d = case["kind"], ESIZE[case["dtype"]], case["hq"], case["hkv"], case["d"]
    n = sum(a for a, _ in lens)
    row = 2 * hkv * (d // 2 + d // 32)  # bytes of a token's codes and scales
    if kind in ("turn", "patch"):
        axes = case["sections"].count(",") + 1
        rows = hq + hkv + (hkv if kind == "turn" else 0)
        nbytes = 2 * n * rows * d * es + 8 * axes * n + (8 * n if kind == "turn" else 0)
        return {"bytes": nbytes, "flops": (7 if case["norm"] else 3) * n * (hq + hkv) * d}
    if kind == "store":
        bs = case["bs"]
        read = sum((h - 1) // bs - (h - a) // bs + 1 for (a, _), h in zip(lens, _held(case))) * bs
        return {"bytes": n * (2 * hkv * d * es + 8 + row) + read * (row + 2 * hkv * d * es + 8), "flops": 0}
    keys = sum(a + c for a, c in lens)
    nbytes = keys * row + 4 * sum(-(-(a + c) // case["bs"]) for a, c in lens) + 2 * n * hq * d * es
    return {"bytes": nbytes, "flops": 4 * hq * d * sum(a * c + a * (a + 1) // 2 for a, c in lens)}


# ---- the definition in 64 bits


def _exact_values(x, fp16):
    """The numbers that the cache holds of ``x`` [.., D]."""
    x = x.double().unflatten(-1, (-1, 32))
    low, high = (-23, 13) if fp16 else (-100, 125)
    # (the logarithm of a border is a whole number, of what lies above it at least 2^-24 more)
    k = torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True) / 7) - 1e-9).clamp(low, high)
    y = (x / torch.exp2(k)).abs()
    number = torch.zeros_like(y)
    # borders between the codes; a tie goes to the even one, so every other border is open
    for border, tie_up, up in ((0.25, False, 0.5), (0.75, True, 1.0), (1.25, False, 1.5), (1.75, True, 2.0),
                               (2.5, False, 3.0), (3.5, True, 4.0), (5.0, False, 6.0)):
        number = torch.where(y >= border if tie_up else y > border, torch.full_like(y, up), number)
    return (number * torch.sign(x) * torch.exp2(k)).flatten(-2)


def _exact_turn(case, s, x, w):
    x = x.double()
    if w is not None:
        x = w.double() * x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS)
    freq, axis = _frequencies(case)
    turns = torch.stack([s["pos"][a].double() * f for f, a in zip(freq, axis)], dim=1)
    half = case["d"] // 2
    z = torch.complex(x[..., :half], x[..., half:]) * torch.polar(torch.ones_like(turns), turns)[:, None]
    return torch.cat([z.real, z.imag], dim=-1)


def exact(case, seed):
    s = _inputs(case, seed)
    kind, fp16 = case["kind"], case["dtype"] == "fp16"
    if kind == "patch":
        return _exact_turn(case, s, s["q"], None), _exact_turn(case, s, s["k"], None)
    if kind == "turn":
        kc, vc = s["kc"].double(), s["vc"].double()
        kc[s["slots"]] = _exact_turn(case, s, s["k"], s["k_norm"])
        vc[s["slots"]] = s["v"].double()
        return _exact_turn(case, s, s["q"], s["q_norm"]), kc, vc
    bs, hkv = case["bs"], case["hkv"]
    step = torch.exp2(s["exps"].double() - 1).repeat_interleave(32, dim=-1)
    cache = (s["codes"].double() * step).flatten(2, 3).transpose(1, 2).contiguous()  # [2, slots, H_kv, D]
    if kind == "store":
        cache[:, s["slots"]] = _exact_values(torch.stack([s["k"], s["v"]]), fp16)
        return cache[0, s["read"]], cache[1, s["read"]]
    out, row = [], 0
    for table, n, c in zip(s["tables"], s["new"], s["cached"]):
        t = torch.arange(n + c, device="cuda")
        k, v = cache[:, torch.tensor(table, device="cuda")[t // bs] * bs + t % bs].transpose(1, 2)
        x = s["q"][row:row + n].double().unflatten(1, (hkv, -1)).permute(1, 2, 0, 3)  # [H_kv, group, n, D]
        scores = torch.matmul(x, k.transpose(1, 2)[:, None]) * s["scale"]
        scores = torch.where(t <= torch.arange(c, c + n, device="cuda")[:, None], scores, -torch.inf)
        out.append(torch.matmul(torch.softmax(scores, -1), v[:, None]).permute(2, 0, 1, 3).flatten(1, 2))
        row += n
    return torch.cat(out)
