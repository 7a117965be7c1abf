"""That the bound of an output's error in the norm (``quant.error_bound``) holds for the
roundings it counts and not for mistakes: modelled in 64 bits on the CPU."""

from __future__ import annotations

import pytest
import torch

from oracle import quant

BS = 16
# (query heads, KV heads, head_dim, cached, new)
CASES = [(28, 4, 128, 512, 1), (14, 2, 64, 512, 1), (8, 4, 64, 6000, 100), (14, 2, 64, 0, 200)]


def case(seed, hq, h, d, cached, new, dtype, spread=1.0):
    """Values a pool holds, rows whose magnitudes differ by ``spread``, and queries."""
    g = torch.Generator().manual_seed(seed)
    n = -(-(cached + new) // BS) * BS
    want = quant.QuantCache(n // BS, BS, h, d, dtype)

    def rows(s):
        x = torch.randn(n, h, d, generator=g) * torch.exp(s * spread * torch.randn(n, h, 1, generator=g))
        return (x * torch.exp(0.5 * spread * torch.randn(d, generator=g))).to(dtype)

    # (whole blocks at once: QuantCache goes block by block)
    x = torch.stack([rows(0.5), rows(1.0)]).double().view(2, n // BS, BS, h, d)
    for b in range(n // BS):
        for kv in range(2):
            for i in range(h):
                e = quant.scale_exponent(x[kv, b, :, i].abs().max().item(), dtype)
                want.values[kv, b * BS : (b + 1) * BS, i] = quant.round_code(x[kv, b, :, i], e, dtype)
    q = torch.randn(new, hq, d, generator=g).to(dtype)
    return q, want.values, list(range(n // BS))


def kernel_model(q, values, table, cached, scale, dtype, round_p, drop=None):
    """Probabilities and the output rounded to ``dtype``, all else in 64 bits; ``drop``: keys left out."""
    s, _, v = quant._scores(q, values, table, BS, cached, scale)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    if round_p:
        p = p.to(dtype).double()
    if drop is not None:
        p[..., drop] = 0.0
    return (p @ v / p.sum(-1, keepdim=True)).transpose(0, 1).to(dtype).double()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", CASES)
def test_bound_holds_for_roundings_and_shows_mistakes(shape, dtype):
    hq, h, d, cached, new = shape
    q, values, table = case(sum(shape), *shape, dtype)
    scale = d**-0.5
    o, spread, reach = quant.attend_spread(q, values, table, BS, cached, scale)
    bound = quant.error_bound(o, spread, reach, dtype, round_p=1.0)

    def off(values=values, q=q, **kw):
        kw = {"round_p": True, **kw}
        return (kernel_model(q, values, table, cached, scale, dtype, **kw) - o).norm()

    assert off() <= bound
    assert off(round_p=False) <= quant.error_bound(o, spread, reach, dtype)
    # a block's V scale doubled, its K scale doubled, one of its 64-key tiles left out, the queries
    # of a head another's
    for kv in (1, 0):
        wrong = values.clone()
        wrong[kv, :BS] *= 2.0
        assert off(values=wrong) > bound, kv
    assert off(drop=slice(64, 128)) > bound
    assert off(q=q.roll(1, 1)) > bound


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
def test_bound_shows_probabilities_and_queries_of_few_bits(d, dtype):
    """Over many outputs: probabilities rounded where only the output's rounding is allowed; at scores of
    some hundred, queries rounded to the dtype once more (as a scaled query would be)."""
    hq, h, cached, new = 6, 2, 300, 90
    q, values, table = case(d, hq, h, d, cached, new, dtype, spread=0.0)
    scale = d**-0.5
    o, spread, reach = quant.attend_spread(q, values, table, BS, cached, scale)
    out = kernel_model(q, values, table, cached, scale, dtype, True)
    assert (out - o).norm() > quant.error_bound(o, spread, reach, dtype)
    q = (12.0 * q.double()).to(dtype)
    o, spread, reach = quant.attend_spread(q, values, table, BS, cached, scale)
    bound = quant.error_bound(o, spread, reach, dtype, round_p=1.0)
    assert (kernel_model(q, values, table, cached, scale, dtype, True) - o).norm() <= bound
    scaled = (q.double() * scale).to(dtype).double() / scale if d == 128 else (q.double() * 1.1).to(dtype).double() / 1.1
    assert (kernel_model(scaled, values, table, cached, scale, dtype, True) - o).norm() > bound
