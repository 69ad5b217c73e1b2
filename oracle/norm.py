"""Float64 restatement of layer norm (PyTorch, CPU or GPU), with componentwise error bounds.

Beside each result stands a bound on how far a computation with fp32 statistics and sums, rounded once to
``dtype``, may be off.  The bounds count roundings of 2^-24: a sum is off by at most its depth times that
times the sum of its terms' sizes.  A row's sum adds at most max(16, C / 256) terms a lane, then over
lanes and waves (10 more); a column's sum at most rows / 256 terms a lane, then over a block's lanes, the
blocks' partial sums and their tree (100 more).  The mean may be off by its sum's error r0; the deviations
from it are formed again, and their mean is taken off, which leaves that mean's own error.
"""
from __future__ import annotations

import torch

U = 2.0 ** -24


def _round(value, dtype):
    info = torch.finfo(dtype)
    return value.abs() * (info.eps / 2) + info.smallest_normal * info.eps / 2


def run(x, weight, bias, eps, grad=None, dtype=None, vector_dtype=None):
    """{"y", "dx", "dw", "db"} -> (value, bound) for x [rows, C]; the gradients where grad is given."""
    dtype, vector_dtype = dtype or x.dtype, vector_dtype or (x.dtype if weight is None else weight.dtype)
    rows, C = x.shape
    x = x.double()
    w = torch.ones(C, dtype=x.dtype, device=x.device) if weight is None else weight.double()
    b = torch.zeros(C, dtype=x.dtype, device=x.device) if bias is None else bias.double()
    h = max(16, C / 256) + 10

    def mean(t):
        return t.mean(-1, keepdim=True)

    d = x - mean(x)
    var = mean(d * d)
    rstd = 1 / torch.sqrt(var + eps)
    n = d * rstd
    r0 = (h + 2) * U * mean(x.abs())
    e_rest = (h + 2) * U * (mean(d.abs()) + r0)
    e_var = (h + 8) * U * (var + 2 * r0 * r0) + e_rest * e_rest
    rel = 0.5 * e_var / torch.clamp(var + eps - e_var, min=1e-300) + 4 * U
    e_n = rstd * (2 * U * (d.abs() + r0) + e_rest) * (1 + rel) + n.abs() * (rel + 2 * U)
    y = n * w + b
    out = {"y": (y, w.abs() * e_n + 2 * U * ((n * w).abs() + b.abs()) + _round(y, dtype))}
    if grad is None:
        return out
    g = grad.double()
    gw = g * w
    s, sn = mean(gw), mean(gw * n)
    e_s = (h + 3) * U * mean(gw.abs())
    e_sn = (h + 4) * U * mean((gw * n).abs()) + mean(gw.abs() * e_n)
    inner = gw - s - n * sn
    e_inner = 4 * U * (gw.abs() + s.abs() + (n * sn).abs()) + e_s + n.abs() * e_sn + sn.abs() * e_n
    dx = rstd * inner
    out["dx"] = dx, rstd * e_inner * (1 + rel) + dx.abs() * (rel + 2 * U) + _round(dx, dtype)
    hr = min(rows, rows / 256 + 100) + 2
    dw, db = (g * n).sum(0), g.sum(0)
    out["dw"] = dw, hr * U * (g * n).abs().sum(0) + (g.abs() * e_n).sum(0) + _round(dw, vector_dtype)
    out["db"] = db, hr * U * g.abs().sum(0) + _round(db, vector_dtype)
    return out
