"""Differentiable dense operators of a transformer block on node rows: the root-mean-square norm with the residual's addition and
the gated feed-forward, each one autograd node over the library's kernels (csrc/dense_ops.cpp).

The reference runs its models forward only (python/graphiler/utils/bench.py:10-49) and has no counterpart of these operators; they
stand next to the dense projection (``layers.project``) that a graph transformer's layer applies to the node rows
(examples/HGT/HGT.py:28-60).  Leading dimensions are flattened to rows; first derivatives only, in reverse mode.  While a CUDA graph is captured, inputs
whose gradients belong to the default stream (an eager graph of the same leaves, recorded there, still lives) are refused.
"""
from __future__ import annotations

from .capi import _call


def rms_norm(x, weight, eps: float = 1e-6, residual=None):
    """``capi.rms_norm`` on (..., n) with gradients of x, the weight and the residual.  Returns y, or (y, r) with a residual; r is
    what the block's output is added to."""
    out = _call("rms_norm", x, weight, eps, residual)
    return out[0] if residual is None else tuple(out)


def gated_linear(x, w_gate, w_up, activation: str = "silu"):
    """``capi.gated_linear`` on (..., k) with gradients of x and both weights.  Kept for the backward pass: the inputs and, for rows
    wider than 768, the two projections in float32 (8 bytes per element of the output); narrower rows make them again.  The projections'
    gradients are rounded to the rows' type on the way, with its range."""
    return _call("gated_linear", x, w_gate, w_up, activation)
