"""Attention over all tokens: object queries among themselves or over a volume, the tokens of a coarse
level, whole prompts, one new token over a cache.

No counterpart in the reference, whose attention samples a few places of the value; a decoder around it
also needs this one.  The heads of a group share a key head, sequences of different lengths run packed one
behind another or as items of a batch that use some of their rows, and lengths are read on the device
only, so no call waits for them.  Logits, statistics and sums are fp32; probabilities and the gradients of
logits are rounded to the tensors' dtype before they are multiplied (in float16 times powers of two, which keep
them in its range); each result is rounded once.  For the backward the forward keeps, beside the output, what rounding took from it.
Results are bitwise repeatable (csrc/attention_kernels.h).
"""
from __future__ import annotations

import math

import torch
from torch.autograd import Function

from . import _extension
from .norm import once


class AttentionFunction(Function):
    """Autograd of packed_attention for the binding without the extension module (which has its own node)."""

    @staticmethod
    def forward(ctx, q, k, v, q_start, k_start, q_len, k_len, causal, scale, native):
        out, lse, rest = native.attention_forward(q, k, v, q_start, k_start, q_len, k_len, causal, scale, True)
        ctx.save_for_backward(q, k, v, q_start, k_start, q_len, k_len, out, lse, rest)
        ctx.rest = causal, scale
        ctx.native = native
        return out

    @staticmethod
    def backward(ctx, grad_output):
        *inputs, out, lse, rest = ctx.saved_tensors
        need_q, need_k, need_v = ctx.needs_input_grad[:3]
        with torch.no_grad():
            gq, gk, gv = ctx.native.attention_backward(*inputs, *ctx.rest, out, lse, rest, grad_output, need_q, need_k or need_v)
        given = grad_output.requires_grad
        return (once(gq, True, "attention"), once(gk if need_k else None, True, "attention"),
                once(gv if need_v else None, need_q or need_k or given, "attention")) + (None,) * 7


def packed_attention(q, k, v, q_start=None, k_start=None, q_len=None, k_len=None, causal=False, scale=None):
    """``softmax(scale q k^T) v`` over the keys that a query sees.

    q [Sq, H, D] or [B, Sq, H, D]; k and v [Sk, Hk, D] or [B, Sk, Hk, D]; all of one dtype (float32, float16 or
    bfloat16) on one device.  H is a multiple of Hk: query head h reads key head ``h // (H / Hk)``.
    D is at most 128.  scale (positive) defaults to ``1 / sqrt(D)``.

    Sequences: with q_start the rows are packed sequences; q_start and k_start (None: q_start) are int64
    tensors on q's device with the first row of each sequence and the last one's end, E + 1 entries for E
    sequences.  Entries count as the largest of themselves and those before them, held to the rows.
    Without, the items of a batch, or all rows, are a sequence each; q_len and k_len, int64 [B], then say how
    many of an item's rows count (a cache's filled part, a padded batch).  Queries see the keys of their
    own sequence; causal, query i sees key j where ``j <= i + keys - queries``: the last query sees all, and
    one new token its whole cache.  A query that sees no key gives 0.  Rows that do not count or are in no
    sequence are not read; their outputs and gradients are 0.  NaN and infinities in keys and values reach
    the queries that see them, and no others.

    q, k and v may be strided between items, tokens and heads (parts of one projection, a transposed
    cache); with strided channels they are copied.  Under autocast they are cast to its dtype.
    Returns q's shape, contiguous.
    """
    if torch.is_autocast_enabled("cuda"):   # as torch's attention does; float64 is left alone (and refused)
        dt = torch.get_autocast_dtype("cuda")
        q, k, v = (t if t.dtype == torch.float64 else t.to(dt) for t in (q, k, v))
    if scale is None:
        scale = 1.0 / math.sqrt(max(1, q.shape[-1])) if q.dim() else 1.0
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite, got {scale!r}")
    if q_start is not None and k_start is None:
        k_start = q_start
    if _extension._C is None:
        raise RuntimeError("ops3d_amd native library (libops3d_fda.so) not built; packed_attention requires it.")
    return _extension._C.attention(q, k, v, q_start, k_start, q_len, k_len, bool(causal), float(scale))
