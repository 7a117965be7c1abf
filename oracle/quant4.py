"""The 4-bit K/V cache and the rotation by several axes in 64 bits on the CPU: e2m1 codes
with a power of two as the scale of 32 channels of a token's head."""

from __future__ import annotations

import torch

# exponents a scale may have, by the pool's dtype
BOUNDS = {torch.float16: (-23, 13), torch.bfloat16: (-100, 125), torch.float32: (-100, 125)}
CODES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def scale_exponent(amax: float, dtype: torch.dtype) -> int:
    """The least k within the dtype's bounds with ``amax <= 7 * 2^k``."""
    lo, hi = BOUNDS[dtype]
    k = lo
    while k < hi and amax > 7.0 * 2.0**k:
        k += 1
    return k


def exponents(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """``scale_exponent`` of each group of 32 of ``x`` (fp64 ``[..., D]``), -1000 where one of it is
    no finite number."""
    g = x.unflatten(-1, (-1, 32))
    amax = g.abs().amax(-1)
    lo, hi = BOUNDS[dtype]
    k = torch.full(amax.shape, lo, dtype=torch.int64)
    for e in range(lo, hi):
        k += amax > 7.0 * 2.0**e
    return torch.where(torch.isfinite(g).all(-1), k, torch.full_like(k, -1000))


def round_code(y: torch.Tensor) -> torch.Tensor:
    """``y`` to the nearest code, ties to the even one (whose last bit is 0)."""
    codes = torch.tensor(CODES, dtype=torch.float64)
    off = (y.abs()[..., None] - codes).abs()
    least = off.amin(-1, keepdim=True)
    # of two codes as near, the one at an even place
    rank = torch.where(off == least, torch.arange(8) % 2, torch.full((8,), 2))
    return codes[rank.argmin(-1)] * torch.sign(y)


def quantise(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """What the cache holds of ``x`` (fp64 ``[..., D]``); NaN groups whole."""
    k = exponents(x, dtype)
    step = torch.exp2(k.double())[..., None]
    bad = (k == -1000)[..., None]
    y = torch.where(bad, torch.zeros(()).double(), x.unflatten(-1, (-1, 32)) / step)
    return torch.where(bad, torch.full((), float("nan")).double(), round_code(y) * step).flatten(-2)


class Quant4Cache:
    """One layer's values ``[2, num_slots, H_kv, D]``."""

    def __init__(self, num_slots: int, h_kv: int, d: int, dtype: torch.dtype) -> None:
        self.dtype = dtype
        self.values = torch.zeros(2, num_slots, h_kv, d, dtype=torch.float64)

    def write(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """One call's rows ``[N, H_kv, D]``."""
        slots = slots.cpu()
        ok = (slots >= 0) & (slots < self.values.shape[1])
        new = torch.stack([k.cpu().double(), v.cpu().double()])
        self.values[:, slots[ok]] = quantise(new[:, ok], self.dtype)


def turn(x: torch.Tensor, positions: torch.Tensor, inv_freq, axis_of, w: torch.Tensor | None = None, eps: float = 0.0,
         scaling: float = 1.0) -> torch.Tensor:
    """Rows ``[N, H, D]`` rotated by ``positions`` ``[axes, N]``, normed per head before if ``w``.
    Each pair is a complex number; whole turns are taken off the angle in Python's integers."""
    x = x.cpu().double()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.cpu().double()
    half = x.shape[-1] // 2
    angles = torch.tensor([[_angle(int(p), f) for f, p in zip(inv_freq, [row[a] for a in axis_of])]
                           for row in positions.cpu().T.tolist()], dtype=torch.float64).view(-1, half)
    z = torch.complex(x[..., :half], x[..., half:]) * torch.polar(torch.ones_like(angles), angles)[:, None] * scaling
    return torch.cat([z.real, z.imag], dim=-1)


# 2 pi in units of 2^-200
_TURN = 2 * 31415926535897932384626433832795028841971693993751058209749445923078164062862089986280348253421170679 * (
    1 << 200) // 10**100


def _angle(position: int, freq: float) -> float:
    """``position * freq`` less whole turns."""
    num, den = freq.as_integer_ratio()
    rest = (position * num * (1 << 200) // den) % _TURN
    if rest * 2 > _TURN:
        rest -= _TURN
    return rest / (1 << 200)
