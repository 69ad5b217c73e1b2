"""Float64 restatement of rotary positions (PyTorch, CPU or GPU), with componentwise error bounds.

Beside the result stands a bound on how far a computation may be off that forms the angles in 64 bits,
their cosines and sines in fp32 and rounds once: an angle is off by a few 2^-53 of itself, its fraction of a
turn is rounded to fp32 (pi 2^-24 radians at most), cosine and sine are good to 2 units in the last place
(2^-22 at most); their two products and the sum round twice more.
"""
from __future__ import annotations

import math

import torch

U = 2.0 ** -24


def run(x, positions, sections, frequencies, layout, inverse=False):
    """(value, bound) for x [..., S, H, D] and positions [..., S, A]."""
    dtype = x.dtype
    pairs = sum(sections)
    axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)], dtype=torch.int64, device=x.device)
    freq = torch.tensor(list(frequencies), dtype=torch.float64, device=x.device)
    angle = (positions.double()[..., axis] * freq)[..., None, :]
    if inverse:
        angle = -angle
    at = [list(range(pairs)), list(range(pairs, 2 * pairs))] if layout == "halves" else [
        list(range(0, 2 * pairs, 2)), list(range(1, 2 * pairs, 2))]
    x = x.double()
    a, b = x[..., at[0]], x[..., at[1]]
    y, bound = x.clone(), torch.zeros_like(x)
    y[..., at[0]] = a * torch.cos(angle) - b * torch.sin(angle)
    y[..., at[1]] = a * torch.sin(angle) + b * torch.cos(angle)
    off = (a.abs() + b.abs()) * (angle.abs() * 2.0 ** -50 + math.pi * U + 4 * U + 3 * U)
    info = torch.finfo(dtype)
    for part in at:
        bound[..., part] = off + y[..., part].abs() * (info.eps / 2) + info.smallest_normal * info.eps / 2
    return y, bound
