"""Calls of the linear operators that their use brings along, beside the sizes and types of test_linear.py
(whose helpers and float64 restatement are used here)."""
from __future__ import annotations

import pytest
import torch

from oracle import linear as ref
from ops3d_amd import fused_linear
from test_linear import DTYPES, gpu, log


# act' far out, small beside 1: z, and act's names
SATURATED = [("silu", -10.0), ("silu", -12.0), ("silu", -6.0), ("gelu", -3.5), ("gelu", -4.0), ("gelu_tanh", -3.5),
             ("gelu_tanh", -4.0), ("silu", -1.5), ("gelu", -1.0), ("gelu", 0.25), ("gelu", 3.0)]


@gpu
@pytest.mark.parametrize("rows", [40, 2000])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("activation,z", SATURATED)
def test_saturated_units_keep_their_gradients(gpu_device, activation, z, dtype, rows):
    """Units that share a saturated z: their act' is held relative to its size, so the gradients' errors,
    which add up over the rows, stay within the roundings."""
    dt = DTYPES[dtype]
    log(f"[case] saturated {activation} {z} {dtype} {rows}")
    x = torch.ones(rows, 32, dtype=dt, device="cuda").requires_grad_(True)
    w = torch.zeros(40, 32, dtype=dt, device="cuda").requires_grad_(True)
    b = torch.full((40,), z, dtype=dt, device="cuda").requires_grad_(True)
    u = torch.full((rows, 40), 16.0, dtype=dt, device="cuda")
    y = fused_linear(x, w, b, activation)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), u)
    d = ref.act(torch.tensor(z, dtype=torch.float64), activation)[1].item()
    # act' evaluated to 2^-14 of itself out here (the error function's polynomial is off by 6e-4 of its tail,
    # which is at most 1 / z^2 of act'), held to 2^-11; dz and the result rounded by half a step each, and a
    # sum of equal fp32 terms of up to 2000 2^-24
    rel = 2.0 ** -14 + 2.0 ** -11 + 2 * torch.finfo(dt).eps / 2 + 2000 * 2.0 ** -24
    want = rows * 16.0 * d
    for name, got in (("db", db), ("dw", dw)):
        err = (got.double() / want - 1).abs().max().item()
        assert err <= rel, f"{name}: off by {err:.2e} of {want:.3e}"
    assert not dx.any()
