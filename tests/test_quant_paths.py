"""Paths of the pools without a GPU: what they refuse and copy before any device work."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from infrared_amd import QuantPagedKVPool, kernels
from infrared_amd.mixed_step import MixedInputs, MixedStep
from infrared_amd.paged_attention import _prefill


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


class Copies(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.n = 0

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.n += func._schema.name in ("aten::clone", "aten::copy_", "aten::_to_copy")
        return func(*args, **(kwargs or {}))


def test_prefill_copies_queries_that_are_no_view_once(monkeypatch):
    taken = []
    monkeypatch.setattr(kernels, "prefill_plan_pays", lambda *a, **k: False)
    monkeypatch.setattr(kernels, "paged_prefill", lambda q, *a, **k: taken.append(q) or q)
    pool = SimpleNamespace(k=torch.zeros(1, 32, 1, 64), v=torch.zeros(1, 32, 1, 64), block_size=16)
    q = torch.randn(3, 2, 4, 64).transpose(0, 1)
    with Copies() as copies:
        out = _prefill(q, pool, 0, torch.zeros(2, 2, dtype=torch.int32), None, torch.zeros(2), 3, None, 0.1, None)
    assert copies.n == 1 and len(taken) == 1
    assert torch.equal(taken[0].view(2, 3, 4, 64), q) and out.shape == q.shape
