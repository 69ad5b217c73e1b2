"""Layer norm over the last axis, forward and backward.

No counterpart in the reference, whose callers put torch's norms between the ops and the linear layers.
The statistics and the sums are fp32 whatever the tensors' dtype, each result is rounded once, and
results are bitwise repeatable (csrc/norm.hip).
"""
from __future__ import annotations

import torch
from torch.autograd import Function

from . import _extension
from .linear import _Once


class LayerNormFunction(Function):
    """Autograd of layer_norm for the binding without the extension module (which has its own node)."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps, native):
        y, stats = native.layer_norm_forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        vector = weight if weight is not None else bias
        ctx.wide = vector is not None and vector.dtype == torch.float32 and x.dtype != torch.float32
        ctx.native = native
        return y

    @staticmethod
    def backward(ctx, grad_output):
        x, weight, stats = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        with torch.no_grad():
            gx, gw, gb = ctx.native.layer_norm_backward(x, weight, stats, grad_output, ctx.wide, need_x, need_w, need_b)
        given = grad_output.requires_grad
        return (once(gx, True, "a layer norm"), once(gw, need_x or given, "a layer norm"),
                once(gb, given, "a layer norm"), None, None)


def once(grad, depends, what):
    """With create_graph, a gradient that depends on something with a gradient raises when it is
    differentiated."""
    if grad is None or not depends or not torch.is_grad_enabled():
        return grad
    return _Once.apply(grad.detach().requires_grad_(True), what)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over x's last axis.

    x [..., C] of float32, float16 or bfloat16; weight and bias [C] or None, both of x's dtype or both
    float32 (beside a 16-bit x their gradients are float32 then, and nothing is cast).  eps is finite and
    not negative.  x may be strided between rows; anything else that is not contiguous is copied.
    Returns x's shape and dtype, under autocast too: the arithmetic is fp32 anyway.
    """
    if _extension._C is None:
        raise RuntimeError("ops3d_amd native library (libops3d_fda.so) not built; layer_norm requires it.")
    return _extension._C.layer_norm(x, weight, bias, float(eps))
