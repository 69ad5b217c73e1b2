"""Rotary positions along several axes: depth, height and width of a volume, or time, height and width.

No counterpart in the reference.  Pairs of channels of every head turn by their token's position along
one of the axes times the pair's frequency, so that a query's product with a key depends on how far they are
apart along each axis (csrc/rotary.hip).  Angles are formed and reduced in 64 bits: positions far out lose
nothing.
"""
from __future__ import annotations

import math
from functools import lru_cache

import torch
from torch.autograd import Function

from . import _extension

LAYOUTS = {"halves": 0, "pairs": 1}


@lru_cache(maxsize=256)
def _pairs(sections, theta):
    """(frequency, axis) of every pair, as two lists."""
    return ([theta ** (-i / n) for n in sections for i in range(n)],
            [axis for axis, n in enumerate(sections) for _ in range(n)])


def axial_frequencies(sections, theta=10000.0):
    """The default frequencies of ``rotary_positions``: pair i of the n pairs of an axis has theta^(-i/n)
    radians a unit, each axis from 1 on."""
    return tuple(_pairs(_sections(sections), float(theta))[0])


def _sections(sections):
    sections = (sections,) if isinstance(sections, int) else tuple(sections)
    if not sections or not all(isinstance(n, int) and n >= 0 for n in sections):
        raise ValueError(f"sections must be numbers of pairs, one for each axis, got {sections!r}")
    return sections


class RotaryFunction(Function):
    """Autograd of rotary_positions for the binding without the extension module (which has its own node):
    the gradient is the turn back."""

    @staticmethod
    def forward(ctx, x, positions, frequencies, axis_of, layout, inverse, native):
        ctx.save_for_backward(positions)
        ctx.rest = frequencies, axis_of, layout, not inverse, native
        return native.rotary_apply(x, positions, frequencies, axis_of, layout, inverse)

    @staticmethod
    def backward(ctx, grad_output):
        (positions,) = ctx.saved_tensors
        return (RotaryFunction.apply(grad_output, positions, *ctx.rest),) + (None,) * 6


def rotary_positions(x, positions, sections, theta=10000.0, frequencies=None, layout="halves"):
    """x with its channel pairs turned by their tokens' positions.

    x [S, H, D] or [B, S, H, D] of float32, float16 or bfloat16; positions [S, A] or, beside a batch,
    [B, S, A], float32 or int64 (no gradient).  sections: how many pairs turn along each of the A axes, in
    the order of the pairs (an int for one axis); together at most D / 2, and at most 128.  Channels behind
    them are copied.  Pair p turns by ``positions[.., axis of p] * frequencies[p]`` radians; frequencies
    default to ``axial_frequencies(sections, theta)``.  layout "halves" pairs channel p with channel
    P + p (P pairs in all), "pairs" pairs channels 2 p and 2 p + 1.  x may be strided between items,
    tokens and heads (a part of a projection); with strided channels it is copied.  Returns a
    contiguous tensor of x's shape and dtype.
    """
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {list(LAYOUTS)}, got {layout!r}")
    sections = _sections(sections)
    if not (theta > 0 and math.isfinite(theta)):
        raise ValueError(f"theta must be positive and finite, got {theta!r}")
    if positions.dim() and positions.shape[-1] != len(sections):
        raise ValueError(f"positions have {positions.shape[-1]} axes, sections {len(sections)}")
    default, axis_of = _pairs(sections, float(theta))
    if frequencies is None:
        frequencies = default
    else:
        frequencies = [float(f) for f in frequencies]
        if len(frequencies) != len(axis_of):
            raise ValueError(f"there are {len(axis_of)} pairs and {len(frequencies)} frequencies")
    if 2 * len(axis_of) > x.shape[-1]:
        raise ValueError(f"{len(axis_of)} pairs do not fit heads of {x.shape[-1]} channels")
    if _extension._C is None:
        raise RuntimeError("ops3d_amd native library (libops3d_fda.so) not built; rotary_positions requires it.")
    return _extension._C.rotary(x, positions, frequencies, axis_of, LAYOUTS[layout])
