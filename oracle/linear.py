"""Float64 restatement of the linear operators (PyTorch, CPU or GPU), with componentwise error bounds.

``forward`` / ``backward`` compute y and the gradients of
``y[r] = act(x[r] W[g(r)]^T + b[g(r)]) + residual[r]`` in 64 bits, and beside each result a bound on
how far a computation with fp32 sums of the same inputs, rounded once to ``dtype``, may be off.

The bounds count roundings: a sum of n products in fp32, in any order, is off by at most
``n 2^-24 sum |a b|`` (twice that where the products are formed apart from the sums; the bias is one
more term); a result rounded to a type by half a step, ``eps / 2`` of its size.  Activations are
evaluated to ``|z| 2^-21 + 2^-24`` and their derivatives to 2^-20 (error function by a polynomial of
error 1.5e-7, exponential and reciprocal of a few units in the last place, arguments rounded to fp32).
Behind an activation the gradient is rounded to ``dtype`` before it is multiplied, and its factor
act'(z) is held in 16 bits unless ``dtype`` is float32: above 1/8 in steps of 2^-14, below as fp16
(``held_derivative``).
"""
from __future__ import annotations

import math

import torch

U = 2.0 ** -24


def group_of_rows(rows, group_start, groups):
    """Group of each of an item's rows, -1 for none: entries count as the largest of themselves and
    those before them, held to [0, rows]; a missing last entry is the rows' end."""
    out = torch.full((rows,), -1, dtype=torch.int64)
    bounds, top = [], 0
    for v in list(group_start) + [rows] * (groups + 1 - len(group_start)):
        top = max(top, min(max(int(v), 0), rows))
        bounds.append(top)
    for g in range(groups):
        out[bounds[g]:bounds[g + 1]] = g
    return out


def act(z, name):
    """act(z), act'(z)."""
    if name is None:
        return z, torch.ones_like(z)
    if name == "relu":
        return torch.where(z <= 0, torch.zeros_like(z), z), torch.where(z <= 0, 0.0, 1.0).to(z)
    if name == "gelu":
        cdf = 0.5 * torch.special.erfc(-z * math.sqrt(0.5))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c, a = math.sqrt(2 / math.pi), 0.044715
        s = torch.sigmoid(2 * c * (z + a * z ** 3))
        return z * s, s + z * s * (1 - s) * 2 * c * (1 + 3 * a * z * z)
    s = torch.sigmoid(z)
    return z * s, s + z * s * (1 - s)


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _tiny(dtype):
    """Half the distance of the type's smallest numbers."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def held_derivative(d, off):
    """How far act'(z) = d, evaluated to within ``off``, moves when it is held in 16 bits: half a step, above
    1/8 of 2^-14, below of fp16's numbers, which have 11 significant bits down to 2^-14 and steps of 2^-24
    below that."""
    exponent = torch.frexp(d.abs() + off)[1].clamp(min=-13)         # |d| + off < 2^exponent
    return torch.where(d - off >= 0.125, torch.full_like(d, 2.0 ** -15), torch.ldexp(torch.ones_like(d), exponent - 12))


def _select(rows_group, weight, bias):
    """Per group: (group, rows, W, b)."""
    for g in range(weight.shape[0]):
        at = (rows_group == g).nonzero().flatten().to(weight.device)
        yield g, at, weight[g], None if bias is None else bias[g]


def run(x, weight, bias, residual, activation, group, grad=None):
    """x [R, K], weight [E, N, K], bias [E, N] or None, residual [R, N] or None, group [R] (-1: none),
    grad [R, N] or None.  Returns {name: (value, bound)} for y and, with grad, dx, dw, db."""
    dtype = x.dtype
    step, tiny = _half_step(dtype), _tiny(dtype)
    x, weight = x.double(), weight.double()
    bias = None if bias is None else bias.double()
    r = None if residual is None else residual.double()
    u = None if grad is None else grad.double()
    R, (E, N, K) = x.shape[0], weight.shape
    y, ey = x.new_zeros(R, N), x.new_zeros(R, N)
    dx, edx = x.new_zeros(R, K), x.new_zeros(R, K)
    dw, edw, db, edb = (x.new_zeros(s) for s in ((E, N, K), (E, N, K), (E, N), (E, N)))
    for g, at, w, b in _select(group, weight, bias):
        xs = x[at]
        z, size = xs @ w.t(), xs.abs() @ w.t().abs()
        if b is not None:
            z, size = z + b, size + b.abs()
        ez = 2 * (K + 1) * U * size
        a, d = act(z, activation)
        ea = 1.13 * ez + (0 if activation is None else z.abs() * 2.0 ** -21 + U)
        out = a if r is None else a + r[at]
        y[at] = out
        ey[at] = ea + 2 * U * (a.abs() + out.abs()) + step * (out.abs() + ea) + tiny
        if u is None:
            continue
        us = u[at]
        dz = us * d
        if activation is None:
            edz = torch.zeros_like(dz)
        else:
            # |act''| <= 1.13; relu's derivative is not known within ez of its step
            ed = (z.abs() <= ez).double() if activation == "relu" else 1.13 * ez + 2.0 ** -20
            if dtype != torch.float32 and activation != "relu":    # 0 and 1 are held exactly
                ed = ed + held_derivative(d, ed)
            edz = us.abs() * ed
            edz = edz + step * (dz.abs() + edz) + tiny
        dx[at] = dz @ w
        edx[at] = edz @ w.abs() + 2 * N * U * ((dz.abs() + edz) @ w.abs())
        dw[g], edw[g] = dz.t() @ xs, edz.t() @ xs.abs() + 2 * len(at) * U * ((dz.abs() + edz).t() @ xs.abs())
        db[g], edb[g] = dz.sum(0), edz.sum(0) + 2 * len(at) * U * (dz.abs() + edz).sum(0)
    res = {"y": (y, ey)}
    if u is not None:
        for name, v, e in (("dx", dx, edx), ("dw", dw, edw), ("db", db, edb)):
            res[name] = (v, e + step * (v.abs() + e) + tiny)
    return res
