"""Linear layers around deformable attention, with bias, activation and residual in one pass.

No counterpart in the reference, whose callers put torch's linear layers around the ops (reference
tests/test_flash_deform_attn.py:25-60): a projection, then an activation or a residual as passes of
their own over [B, S, C].  Here they are the product's epilogue (csrc/linear_kernels.h):

    fused_linear(x, weight, bias, activation, residual)      act(x W^T + b) + residual
    grouped_linear(x, weight, group_start, ...)              the same with weights of its own for each
                                                             group of consecutive rows

The groups of ``grouped_linear`` are the levels of a flattened volume pyramid (``group_start`` is then
``level_start_index`` as it stands) or experts over rows sorted by expert.  Both run forward and
backward in fp32, fp16 and bf16 with fp32 sums, each result rounded once; the gradient behind an
activation is rounded to the tensors' dtype before it is multiplied.  Results are bitwise repeatable.
"""
from __future__ import annotations

import torch
from torch.autograd import Function

from . import _extension

ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


class LinearFunction(Function):
    """Autograd of both operators for the binding without the extension module (which has its own node);
    ``group_start`` None is the plain product, ``native`` the binding."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, group_start, act, native):
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        y, act_grad = native.linear_forward(x, weight, bias, residual, group_start, act, need_x or need_w or need_b)
        ctx.save_for_backward(x if need_w or need_b else None, weight if need_x else None, group_start, act_grad)
        ctx.in_features, ctx.groups = weight.shape[-1], weight.shape[0] if weight.dim() == 3 else 0
        ctx.native = native
        return y

    @staticmethod
    def backward(ctx, grad_output):
        x, weight, group_start, act_grad = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        grad_x = grad_w = grad_b = None
        if need_x or need_w or need_b:
            with torch.no_grad():
                grad_x, grad_w, grad_b = ctx.native.linear_backward(
                    x, weight, group_start, act_grad, grad_output, ctx.in_features, ctx.groups, need_w, need_b)
            if torch.is_grad_enabled():   # each that depends on something with a gradient
                act, given = act_grad is not None, grad_output.requires_grad
                grad_x = _once(grad_x, need_w or act or given)
                grad_w = _once(grad_w, need_x or act or given)
                grad_b = _once(grad_b, act or given)
        grad_r = None
        if need_r:   # rows of no group are 0 whatever the residual
            grad_r = grad_output if group_start is None else ctx.native.linear_keep_rows(grad_output, group_start, ctx.groups)
        return grad_x, grad_w, grad_b, grad_r, None, None, None


class _Once(Function):
    """A gradient that raises when it is differentiated."""

    @staticmethod
    def forward(ctx, t):
        return t.view_as(t)

    @staticmethod
    def backward(ctx, grad_output):
        raise RuntimeError("trying to differentiate twice a linear operator that is differentiable once")


def _once(grad, depends):
    return _Once.apply(grad.detach().requires_grad_(True)) if grad is not None and depends else grad


class KeepRowsFunction(Function):
    """Zeros in rows of no group, for the binding without the extension module; its own gradient."""

    @staticmethod
    def forward(ctx, t, group_start, groups, native):
        ctx.save_for_backward(group_start)
        ctx.groups, ctx.native = groups, native
        return native._keep_rows(t, group_start, groups)

    @staticmethod
    def backward(ctx, grad_output):
        (group_start,) = ctx.saved_tensors
        return KeepRowsFunction.apply(grad_output, group_start, ctx.groups, ctx.native), None, None, None


def _apply(x, weight, bias, residual, group_start, activation):
    try:
        act = ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)}, got {activation!r}") from None
    if torch.is_autocast_enabled("cuda"):
        # as torch's linear does: the product in the autocast dtype, float64 left alone (and refused); a
        # residual of a wider type keeps it
        dt = torch.get_autocast_dtype("cuda")
        x, weight, bias = (t if t is None or t.dtype == torch.float64 else t.to(dt) for t in (x, weight, bias))
        if residual is not None and residual.dtype != dt:
            y = _run(x, weight, bias, None, group_start, act)
            if group_start is not None:
                residual = _rows_of_groups(residual.expand(y.shape), group_start, weight.shape[0])
            return y + residual
    return _run(x, weight, bias, residual, group_start, act)


def _rows_of_groups(t, group_start, groups):
    """t with zeros in rows of no group."""
    if t.dtype in (torch.float32, torch.float16, torch.bfloat16):
        return _extension._C.linear_keep_rows(t, group_start, groups)
    ones = torch.ones((*t.shape[:-1], 1), device=t.device)
    return torch.where(_extension._C.linear_keep_rows(ones, group_start, groups) > 0, t, t.new_zeros(()))


def _run(x, weight, bias, residual, group_start, act):
    if _extension._C is None:
        raise RuntimeError("ops3d_amd native library (libops3d_fda.so) not built; the linear operators require it.")
    return _extension._C.linear(x, weight, bias, residual, group_start, act)


def fused_linear(x, weight, bias=None, activation=None, residual=None):
    """``act(x @ weight.T + bias) + residual``.

    x [..., K]; weight [N, K]; bias [N] or None; residual [..., N] or None (the output's shape);
    activation None, "relu", "gelu" (erf), "gelu_tanh" or "silu".  All of one dtype (float32, float16
    or bfloat16) on one device.  x and residual may be strided between rows (a split of a wider
    projection, an expanded tensor); anything else that is not contiguous is copied.  Returns
    [..., N].
    """
    return _apply(x, weight, bias, residual, None, activation)


def grouped_linear(x, weight, group_start, bias=None, activation=None, residual=None):
    """``act(x[r] @ weight[g(r)].T + bias[g(r)]) + residual[r]`` for rows r in groups g(r).

    x [S, K] or [B, S, K]; weight [E, N, K]; bias [E, N] or None; residual [S, N] or [B, S, N] or None.
    group_start int64 on x's device holds the first row of each group, the same in every batch item:
    E entries (the last group ends with the rows: a ``level_start_index``) or E + 1 (the last entry is
    the last group's end).  It is read on the device only, so no call waits for it; entries count as
    the largest of themselves and those before them, held to [0, S].  Groups may be empty; rows in no
    group give zeros and take no part in the gradients.  E is at most 4096.  Returns [S, N] or
    [B, S, N].
    """
    if group_start is None:
        raise ValueError("group_start must be an int64 tensor")
    return _apply(x, weight, bias, residual, group_start, activation)
