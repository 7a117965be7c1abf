"""Paths over the 8-bit pool without a GPU: what they refuse before any device work."""

from __future__ import annotations

import pytest
import torch

from infrared_amd import QuantPagedKVPool
from infrared_amd.mixed_step import MixedInputs, MixedStep


def test_mixed_step_refuses_inputs_of_another_dtype():
    """Rows of another dtype would be written with scales the pool's values have no room for."""
    pool = object.__new__(QuantPagedKVPool)  # (its tensors are not asked for)
    pool.dtype = torch.float16
    for name in ("q_dec", "q_pre", "k_new", "v_new"):
        for dtype in (torch.bfloat16, torch.float32):
            x = {n: torch.zeros(1, 1, 2, 64, dtype=torch.float16) for n in ("q_dec", "q_pre", "k_new", "v_new")}
            x[name] = x[name].to(dtype)
            with pytest.raises(RuntimeError, match=f"{name} is {dtype}, the 8-bit pool's dtype is torch.float16"):
                MixedStep(pool, None, MixedInputs(**x), 0.1)
