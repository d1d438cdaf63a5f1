"""Differentiable dense operators of a transformer block on node rows: the root-mean-square norm with the residual's addition and
the gated feed-forward, each one autograd node over the kernels of ``capi``.

The reference runs its models forward only (python/graphiler/utils/bench.py:10-49) and has no counterpart of these operators; they
stand next to the dense projection (``layers.project``) that a graph transformer's layer applies to the node rows
(examples/HGT/HGT.py:28-60).  Leading dimensions are flattened to rows; first derivatives only.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import capi


def _rows(t, width: int):
    return t.reshape(-1, width).contiguous()


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps, residual):
        ctx.set_materialize_grads(False)
        n = weight.shape[0]
        rows = _rows(x, n)
        res = None if residual is None else _rows(residual, n)
        out = capi.rms_norm(rows, weight, eps, residual=res, return_rstd=True)
        y, r, rstd = out if residual is not None else (out[0], rows, out[1])
        ctx.save_for_backward(r, weight, rstd)
        ctx.shape = x.shape
        return y.view(x.shape) if residual is None else (y.view(x.shape), r.view(x.shape))

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dr=None):
        r, weight, rstd = ctx.saved_tensors
        if dy is None:
            # only the sum went on: its gradient passes through
            return dr, None, None, dr if ctx.needs_input_grad[3] else None
        n = weight.shape[0]
        dx, dw = capi.rms_norm_grad(r.view(-1, n), weight, rstd, _rows(dy, n), None if dr is None else _rows(dr, n))
        dx = dx.view(ctx.shape)
        return dx, dw, None, dx if ctx.needs_input_grad[3] else None


def rms_norm(x, weight, eps: float = 1e-6, residual=None):
    """``capi.rms_norm`` on (..., n) with gradients of x, the weight and the residual.  Returns y, or (y, r) with a residual; r is
    what the block's output is added to."""
    if weight.dim() != 1 or x.dim() < 1 or x.shape[-1] != weight.shape[0]:
        raise capi.GphlError("rms_norm needs rows (..., n) and a weight of n values")
    if residual is not None and residual.shape != x.shape:
        raise capi.GphlError("rms_norm: the residual must have the rows' shape and type")
    return _RmsNorm.apply(x, weight.contiguous(), eps, residual)


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, activation):
        rows = _rows(x, x.shape[-1])
        shape = x.shape[:-1] + (w_gate.shape[1],)
        ctx.activation, ctx.shape = activation, x.shape
        if not any(ctx.needs_input_grad[:3]):
            return capi.gated_linear(rows, w_gate, w_up, activation).view(shape)
        h, g, u = capi.gated_linear(rows, w_gate, w_up, activation, return_projections=True)
        ctx.save_for_backward(rows, w_gate, w_up, g, u)
        return h.view(shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        rows, w_gate, w_up, g, u = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dwg, dwu = capi.gated_linear_grad(_rows(dh, w_gate.shape[1]), g, u, rows, w_gate, w_up, ctx.activation, want_dx=need[0],
                                              want_dw=need[1] or need[2])
        return dx.view(ctx.shape) if need[0] else None, dwg if need[1] else None, dwu if need[2] else None, None


def gated_linear(x, w_gate, w_up, activation: str = "silu"):
    """``capi.gated_linear`` on (..., k) with gradients of x and both weights.  The two projections are kept in float32 for the backward
    pass (8 bytes per element of the output) when a gradient is wanted."""
    if x.dim() < 1 or w_gate.dim() != 2 or x.shape[-1] != w_gate.shape[0]:
        raise capi.GphlError("gated_linear needs rows (..., k) and two weights (k, f)")
    return _GatedLinear.apply(x, w_gate, w_up, activation)
