"""Float64 restatement of attention over all tokens (PyTorch, CPU or GPU), with componentwise error bounds.

Beside each result stands a bound on how far a computation may be off whose logits and sums are fp32, whose
probabilities P and gradients of logits dS are rounded to ``dtype`` before they are multiplied, whose
statistics are the sum's reference and logarithm in fp32, and whose results are rounded once.  The bounds
count roundings (U = 2^-24, u half a step of dtype):

* a logit is off by (D + 2) U sum |q k|; as an exponent of 2 it and the reference are rounded three times
  more, and the power is good to 2^-22.  The reference is at most the largest logit's size, or its
  logarithm's.  The relative error of a probability is the sum of these, natural logarithm times;
* in 16 bits the output's denominator is the sum of the rounded probabilities: each term is off by u of itself, and so is the
  sum (the logarithm that the backward's probabilities come from is of the sum as it is);
* a sum of n products is off by (n / 4 + 40) U of the sum of their sizes: four at least are added at a time,
  a sum is rescaled some times, and parts are joined;
* fp16: P is held 2^10 up, so that one below 2^-14 is off by 2^-35 at most; dS is held so that the largest of what is
  summed, for a query's gradient or for a key's, is 2^8 at least: one far below it is off by 2^-33 of that largest;
* every type: a power, and a product in fp32 or an operand of bf16, below 2^-126 may count as 0, so that a P is off by
  2^-125 more, and a dS by that times its factor and once more;
* the sum of out grad_out is formed from the rounded out and what rounding took from it, itself rounded.
"""
from __future__ import annotations

import math

import torch

U = 2.0 ** -24
LN2 = math.log(2.0)


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _round(value, dtype):
    info = torch.finfo(dtype)
    return value.abs() * (info.eps / 2) + info.smallest_normal * info.eps / 2


def sequence(q, k, v, causal, scale, grad=None):
    """{"y", "dq", "dk", "dv"} -> (value, bound) for one sequence, q [nq, H, D], k and v [nk, Hk, D]; the
    gradients where grad is given."""
    dtype = q.dtype
    nq, H, D = q.shape
    nk, Hk = k.shape[:2]
    G = H // Hk
    u = 0.0 if dtype == torch.float32 else _half(dtype)
    tiny = 2.0 ** -125
    low_p, low_ds = (2.0 ** -35, 2.0 ** -33) if dtype == torch.float16 else (tiny, 0.0)
    q, k, v = q.double(), k.double(), v.double()
    grad = None if grad is None else grad.double()
    out = {"y": [torch.zeros_like(q), torch.zeros_like(q)]}
    if grad is not None:
        out.update({"dq": [torch.zeros_like(q), torch.zeros_like(q)], "dk": [torch.zeros_like(k), torch.zeros_like(k)],
                    "dv": [torch.zeros_like(v), torch.zeros_like(v)]})
    if nq == 0 or nk == 0:
        return {n: tuple(t) for n, t in out.items()}
    seen = torch.ones(nq, nk, dtype=torch.bool, device=q.device)
    if causal:
        seen = torch.arange(nk, device=q.device)[None] <= torch.arange(nq, device=q.device)[:, None] + nk - nq
    some = seen.any(1, keepdim=True)
    hk, hq = (nk / 4 + 40) * U, (nq * G / 4 + 40) * U
    most, weight = torch.zeros(nk, Hk, 1, dtype=q.dtype, device=q.device), torch.zeros_like(k)   # of a key's dS, and of what it meets
    for h in range(H):
        qh, kh, vh = q[:, h], k[:, h // G], v[:, h // G]
        s = (qh @ kh.t()) * scale
        e_s = (D + 2) * U * (qh.abs() @ kh.abs().t()) * scale
        top = torch.where(seen, s, -math.inf).amax(1, keepdim=True)
        top = torch.where(some, top, 0.0)
        size = torch.where(seen, s.abs(), 0.0).amax(1, keepdim=True)
        p = torch.where(seen, torch.exp(s - top), 0.0)
        total = p.sum(1, keepdim=True)
        p = p / torch.where(some, total, 1.0)
        d = e_s + 4 * U * (s.abs() + size) + 2.0 ** -22   # relative error of a probability's numerator
        mean_d = (p * d).sum(1, keepdim=True)
        y = p @ vh
        e_y = (p * (d + u + hk)) @ vh.abs() + low_p * (seen.double() @ vh.abs()) + y.abs() * (mean_d + u + hk + 4 * U)
        e_o, e_y = e_y + u * _round(y, dtype), e_y + _round(y, dtype)
        out["y"][0][:, h], out["y"][1][:, h] = y, torch.where(some, e_y, 0.0)
        if grad is None:
            continue
        g = grad[:, h]
        lse = (top + torch.log(torch.where(some, total, 1.0))).abs()
        d = e_s + 4 * U * (s.abs() + lse + size) + 2.0 ** -22 + mean_d + hk + 4 * U
        dp = g @ vh.t()
        e_dp = (D + 2) * U * (g.abs() @ vh.abs().t())
        delta = (y * g).sum(1, keepdim=True)
        e_delta = (e_o * g.abs()).sum(1, keepdim=True) + (D + 2) * U * (y * g).abs().sum(1, keepdim=True)
        ds = p * (dp - delta)
        e_ds = ds.abs() * (d + u + 3 * U) + p * (e_dp + e_delta + 2 * U * (dp.abs() + delta.abs()))
        e_ds = e_ds + seen.double() * tiny * (1 + dp.abs() + delta.abs())
        size = ds.abs() + e_ds
        low_q = low_ds * size.amax(1, keepdim=True) * seen.double()
        most[:, h // G] = torch.maximum(most[:, h // G], size.amax(0)[:, None])
        weight[:, h // G] += seen.double().t() @ qh.abs()
        out["dq"][0][:, h] = scale * (ds @ kh)
        out["dq"][1][:, h] = scale * ((e_ds + low_q + hk * ds.abs()) @ kh.abs())
        out["dk"][0][:, h // G] += scale * (ds.t() @ qh)
        out["dk"][1][:, h // G] += scale * ((e_ds + hq * ds.abs()).t() @ qh.abs())
        out["dv"][0][:, h // G] += p.t() @ g
        out["dv"][1][:, h // G] += (p * (d + u + hq)).t() @ g.abs() + low_p * (seen.double().t() @ g.abs())
    if grad is not None:
        out["dk"][1] += scale * low_ds * most * weight
    for name in ("dq", "dk", "dv"):
        if grad is not None:
            value, bound = out[name]
            out[name][1] = bound * (1 + 4 * U) + 2 * U * value.abs() + _round(value, dtype)
    return {n: tuple(t) for n, t in out.items()}


def bounds_of(start, rows):
    """The sequences' bounds: entries count as the largest of themselves and those before them, held to
    [0, rows]."""
    out, top = [], 0
    for x in start:
        top = max(top, min(max(int(x), 0), rows))
        out.append(top)
    return out


def packed(q, k, v, q_start, k_start, causal, scale, grad=None):
    """The same for packed sequences; rows of none are 0, exactly."""
    qb, kb = bounds_of(q_start, q.shape[0]), bounds_of(k_start, k.shape[0])
    out = {}
    for name, like in (("y", q), ("dq", q), ("dk", k), ("dv", v)):
        if name == "y" or grad is not None:
            out[name] = tuple(torch.zeros(like.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    for e in range(len(qb) - 1):
        at_q, at_k = slice(qb[e], qb[e + 1]), slice(kb[e], kb[e + 1])
        part = sequence(q[at_q], k[at_k], v[at_k], causal, scale, None if grad is None else grad[at_q])
        for name, at in (("y", at_q), ("dq", at_q), ("dk", at_k), ("dv", at_k)):
            if name in out:
                out[name][0][at], out[name][1][at] = part[name]
    return out


def items(q, k, v, q_len, k_len, causal, scale, grad=None):
    """The same for items [B, N, H, D] of which some rows count."""
    parts = []
    for b in range(q.shape[0]):
        nq = q.shape[1] if q_len is None else min(max(int(q_len[b]), 0), q.shape[1])
        nk = k.shape[1] if k_len is None else min(max(int(k_len[b]), 0), k.shape[1])
        parts.append(packed(q[b], k[b], v[b], [0, nq], [0, nk], causal, scale, None if grad is None else grad[b]))
    return {name: tuple(torch.stack([p[name][i] for p in parts]) for i in range(2)) for name in parts[0]}
