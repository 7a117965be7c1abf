"""Rotary positions with several axes.

Tokens of images and video have a position for each of several axes (time, height,
width); text has the same one for all. Pair ``j`` of a head (elements ``j`` and ``j + D/2``,
the halves that ``infrared/model/layers.py:79-89`` rotates) belongs to one axis and turns by
that axis's position times its own frequency. ``RotaryAxes`` holds the frequencies as the
kernels take them; ``kernels.rope_axes``, ``kernels.rope_axes_kv_scatter`` and
``rope_axes_paged_attention`` rotate with it.
"""

from __future__ import annotations

import math
from collections.abc import Sequence
from fractions import Fraction

import torch

from infrared_amd._lib import ROTARY_MAX_AXES

# (49 decimals: the steps below are of 64 bits)
_TWO_PI = 2 * Fraction(31415926535897932384626433832795028841971693993751, 10**49)


def _step(freq: float) -> int:
    """``freq`` radians in units of 2^-64 turns, without whole turns."""
    return round(Fraction(freq) / _TWO_PI * 2**64) % 2**64


class RotaryAxes:
    """Frequencies and axes of a head's pairs.

    ``inv_freq`` and ``axis_of``: ``head_dim / 2`` numbers each, the frequency of pair
    ``j`` in radians and its axis. ``scaling`` multiplies the rotated rows (the factor that
    some long-context schemes put on cos and sin). :meth:`sections` and :meth:`grid` make the
    two usual arrangements.

    A frequency is kept as turns in units of 2^-64, so position times frequency, modulo
    2^64, is the angle as a fraction of a turn: a wrap of the integer product instead of a
    reduction of a large floating-point angle, off by at most ``abs(position)`` * 2^-65 turns.
    """

    def __init__(
        self,
        inv_freq: Sequence[float],
        axis_of: Sequence[int],
        *,
        scaling: float = 1.0,
        device: torch.device | str = "cuda",
    ) -> None:
        self.inv_freq = tuple(float(f) for f in inv_freq)
        self.axis_of = tuple(int(a) for a in axis_of)
        self.scaling = float(scaling)
        self.head_dim = 2 * len(self.inv_freq)
        if not self.inv_freq or len(self.axis_of) != len(self.inv_freq):
            raise ValueError(
                f"{len(self.inv_freq)} frequencies and {len(self.axis_of)} axes: one of each a pair expected")
        if self.head_dim % 16 or self.head_dim > 256:
            raise ValueError(f"heads of {self.head_dim}: a multiple of 16 up to 256 expected")
        if not all(math.isfinite(f) for f in (*self.inv_freq, self.scaling)):
            raise ValueError("frequencies and scaling must be finite")
        if min(self.axis_of) < 0 or max(self.axis_of) >= ROTARY_MAX_AXES:
            raise ValueError(f"axes must be in 0..{ROTARY_MAX_AXES - 1}")
        self.num_axes = max(self.axis_of) + 1
        steps = [_step(f) for f in self.inv_freq]
        rows = [[s - 2**64 if s >= 2**63 else s, a] for s, a in zip(steps, self.axis_of)]
        self._host = torch.tensor(rows, dtype=torch.int64)  # ir_rotary_pair, 16 bytes each
        self._pairs: dict[torch.device, torch.Tensor] = {}
        self.pairs(device)

    @classmethod
    def sections(cls, head_dim: int, sections: Sequence[int], theta: float = 1e6, **kw) -> RotaryAxes:
        """The first ``sections[0]`` pairs turn by axis 0, the next ``sections[1]`` by axis 1, and so on;
        the frequencies ``theta ** (-2 j / head_dim)`` run on from one to the next, so that equal
        positions are the usual rotation."""
        if sum(sections) * 2 != head_dim:
            raise ValueError(f"sections {tuple(sections)} are {sum(sections)} pairs, heads of {head_dim} have {head_dim // 2}")
        return cls([theta ** (-2 * j / head_dim) for j in range(head_dim // 2)],
                   [a for a, n in enumerate(sections) for _ in range(n)], **kw)

    @classmethod
    def grid(cls, head_dim: int, axes: int = 2, theta: float = 1e4, **kw) -> RotaryAxes:
        """Each of ``axes`` axes has the same number of pairs and the same run of frequencies."""
        n = head_dim // 2 // axes
        if n * axes * 2 != head_dim:
            raise ValueError(f"heads of {head_dim} have {head_dim // 2} pairs, which {axes} axes do not share")
        return cls([theta ** (-j / n) for _ in range(axes) for j in range(n)],
                   [a for a in range(axes) for _ in range(n)], **kw)

    def pairs(self, device: torch.device | str) -> torch.Tensor:
        """The pairs on ``device`` as the kernels take them (int64 ``[head_dim / 2, 2]``, kept)."""
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError(f"RotaryAxes lives in ROCm device memory; device {device} is not supported")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        held = self._pairs.get(device)
        if held is None:
            held = self._pairs[device] = self._host.to(device)
        return held

    def bind(self, name: str, positions: torch.Tensor, like: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """``positions`` as ``[axes, N]`` and the pairs on ``like``'s device, checked."""
        held = self._pairs.get(like.device)
        if held is None:
            held = self.pairs(like.device)
        if positions.dim() == 2 and positions.shape[0] == self.num_axes:
            return positions, held
        if positions.dim() == 1:
            positions = positions[None]
        if positions.dim() != 2 or positions.shape[0] < self.num_axes:
            raise RuntimeError(f"{name}: positions {tuple(positions.shape)} for a rotary of {self.num_axes} axes")
        return positions[: self.num_axes], held
