"""The 8-bit K/V cache in 64 bits on the CPU: e4m3 codes with a power of two as the
scale of each (block, KV head, K or V), and attention over the values they stand for."""

from __future__ import annotations

import torch

# exponents a scale may have, and the largest magnitude held, by the pool's dtype
BOUNDS = {
    torch.float16: (-15, 8, 61440.0),
    torch.bfloat16: (-100, 119, 448.0 * 2.0**119),
    torch.float32: (-100, 119, 448.0 * 2.0**119),
}


def scale_exponent(amax: float, dtype: torch.dtype) -> int:
    """The least k within the dtype's bounds with ``amax <= 448 * 2^k``."""
    lo, hi, _ = BOUNDS[dtype]
    k = lo
    while k < hi and amax > 448.0 * 2.0**k:
        k += 1
    return k


def round_code(x: torch.Tensor, k: int, dtype: torch.dtype) -> torch.Tensor:
    """``x`` (fp64) to the nearest ``code * 2^k``, ties to the even code: three bits after
    the leading one, multiples of 2^(k - 9) below 2^(k - 6). Past the dtype's largest
    magnitude saturated, not finite: NaN."""
    most = BOUNDS[dtype][2]
    y = x.clamp(-most, most)
    e = torch.frexp(y.abs().clamp_min(2.0 ** (k - 6)))[1].double() - 1
    step = torch.exp2(e - 3)
    y = torch.round(y / step) * step
    return torch.where(torch.isfinite(x), y, torch.full_like(y, float("nan")))


class QuantCache:
    """One layer's values ``[2, num_slots, H_kv, D]`` and scale exponents ``[H_kv, num_blocks, 2]``."""

    def __init__(self, num_blocks: int, block_size: int, h_kv: int, d: int, dtype: torch.dtype) -> None:
        self.bs, self.dtype = block_size, dtype
        self.values = torch.zeros(2, num_blocks * block_size, h_kv, d, dtype=torch.float64)
        self.exps = torch.full((h_kv, num_blocks, 2), BOUNDS[dtype][0], dtype=torch.int64)

    def write(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """One call's rows ``[N, H_kv, D]``: its blocks one after the other."""
        bs, total = self.bs, self.values.shape[1]
        new = torch.stack([k.cpu().double(), v.cpu().double()])
        rows: dict[int, dict[int, int]] = {}  # block -> offset -> row, the last given
        for i, s in enumerate(slots.tolist()):
            if 0 <= s < total:
                rows.setdefault(s // bs, {})[s % bs] = i
        for b, at in rows.items():
            held = self.values[:, b * bs : (b + 1) * bs]
            offs, idx = list(at), list(at.values())
            for kv in range(2):
                for h in range(held.shape[2]):
                    x = new[kv, idx, h]
                    fin = x[torch.isfinite(x)]
                    need = scale_exponent(fin.abs().max().item() if fin.numel() else 0.0, self.dtype)
                    old = int(self.exps[h, b, kv])
                    if 0 in at:
                        held[kv, :, h] = 0.0
                        exp = need
                    else:
                        exp = max(old, need)
                        if exp > old:
                            held[kv, :, h] = round_code(held[kv, :, h], exp, self.dtype)
                    held[kv, offs, h] = round_code(x, exp, self.dtype)
                    self.exps[h, b, kv] = exp


def _scores(q: torch.Tensor, values: torch.Tensor, table, block_size: int, start: int, scale: float):
    """Scores ``[H_q, n, T]`` (-inf where unseen), their ``scale * sum |q k|`` (0 there) and V ``[H_q, T, D]``."""
    n, hq, d = q.shape
    h_kv = values.shape[2]
    t = torch.arange(start + n)
    slots = torch.tensor(table, dtype=torch.long)[t // block_size] * block_size + t % block_size
    k, v = values[:, slots].transpose(1, 2).repeat_interleave(hq // h_kv, dim=1)  # [H_q, T, D]
    x = q.cpu().double().transpose(0, 1)
    seen = t[None, :] <= torch.arange(start, start + n)[:, None]
    s = torch.where(seen, x @ k.transpose(1, 2) * scale, -torch.inf)
    return s, torch.where(seen, x.abs() @ k.abs().transpose(1, 2) * scale, torch.zeros(())), v


def attend(q: torch.Tensor, values: torch.Tensor, table, block_size: int, start: int, scale: float):
    """Queries ``[n, H_q, D]`` at positions ``start ..`` over ``values`` ``[2, slots, H_kv, D]``
    through a block table. Returns the output and, per (query, head), what bounds a
    kernel's error: the attention over ``|V|`` and the largest ``scale * sum |q k|``."""
    s, reach, v = _scores(q, values, table, block_size, start, scale)
    p = torch.softmax(s, -1)
    return (p @ v).transpose(0, 1), (p @ v.abs()).transpose(0, 1), reach.amax(-1).transpose(0, 1)


def attend_spread(q: torch.Tensor, values: torch.Tensor, table, block_size: int, start: int, scale: float):
    """The output of ``attend`` and what errors of the keys' probabilities, each on its own
    and relative to it, come to in an output: ``sqrt(sum p^2 v^2)``; with the largest
    ``scale * sum |q k|``."""
    s, reach, v = _scores(q, values, table, block_size, start, scale)
    p = torch.softmax(s, -1)
    return ((p @ v).transpose(0, 1), (p.square() @ v.square()).sqrt().transpose(0, 1),
            reach.amax(-1).transpose(0, 1))


def error_bound(o: torch.Tensor, spread: torch.Tensor, reach: torch.Tensor, dtype: torch.dtype,
                round_p: float = 0.0) -> float:
    """Bound of ``|out - o|`` in the norm over all elements, for outputs ``o`` of ``attend_spread``
    rounded to ``dtype`` once, 5% above what the roundings come to:

    - the output's own: that of ``o``;
    - with ``round_p``, each probability's to ``dtype``, half a step u at most: uniform
      within it, u / sqrt(3) in the mean square, times ``round_p``;
    - fp32 sums: a score's partial sums are some reach / sqrt(d), d of them, so it is off by a step
      or two of 2^-24 of ``reach``; the exponential and the sums over keys by a few dozen."""
    u = torch.finfo(dtype).eps / 2
    own = (o.to(dtype).double() - o).norm()
    p = round_p * u / 3**0.5 * spread.norm()
    fp32 = 2.0**-24 * (((32 + 2 * reach[..., None]) * spread).norm() + 32 * o.norm())
    return float(1.05 * torch.sqrt(own**2 + p**2 + fp32**2))


def norm_rope(x: torch.Tensor, w: torch.Tensor, eps: float, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """Rows ``[N, H, D]`` normed per head and rotated, in 64 bits."""
    x, w = x.cpu().double(), w.cpu().double()
    cos, sin = cos.cpu().double()[:, None], sin.cpu().double()[:, None]
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w
    a, b = y.chunk(2, dim=-1)
    return y * cos + torch.cat([-b, a], dim=-1) * sin
