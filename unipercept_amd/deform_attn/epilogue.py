"""Operators around the attention of an encoder layer, on hand-written HIP kernels.

* ``counter_dropout``: dropout (after an optional ReLU) whose mask is computed from counters in both
  directions and never stored;
* ``dropout_add_layer_norm``: ``LayerNorm(residual + dropout(x))``, one pass a direction;
* ``level_group_norm``: group norm of the flattened pyramid, every level on its own, with an
  activation.

All take float32, float64, bfloat16 and float16 tensors on a ROCm GPU (sums and statistics are held
in 32 bits or more), use the current stream, are differentiable once, and give the same bits on every
run.  ``MSDeformAttnEncoderLayer(fused_epilogues=True)`` and ``LevelInputProjection`` call them.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _epilogue_ops as ops


def new_rng_state(device, generator: torch.Generator | None = None) -> torch.Tensor:
    """A (seed, offset) pair for the dropout operators, drawn from torch's generator of `device`
    (or `generator`), so ``torch.manual_seed`` makes runs repeatable.  One pair serves any number of
    uses that differ in ``site``."""
    return torch.randint(
        -(2**63), 2**63 - 1, (2,), dtype=torch.int64, device=device, generator=generator
    )


class CounterDropoutFunction(torch.autograd.Function):
    """``apply(x, rng_state, p, site, activation)``.  Saves the output with "relu" (the next layer
    keeps it anyway) and only the state otherwise."""

    @staticmethod
    def forward(ctx, x, rng_state, p, site, activation):
        out = ops.counter_dropout_fwd(x, rng_state, p, site, activation)
        if activation == "relu":
            ctx.save_for_backward(out, None)
        else:
            ctx.save_for_backward(None, rng_state)
        ctx.args = (p, site, activation)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        out, rng_state = ctx.saved_tensors
        p, site, activation = ctx.args
        grad = ops.counter_dropout_bwd(grad_output, out, rng_state, p, site, activation)
        return grad, None, None, None, None


class DropoutAddLayerNormFunction(torch.autograd.Function):
    """``apply(x, residual, weight, bias, rng_state, p, site, eps)``.  Saves the inputs and two values
    a row; the sum that is normalised is computed again in the backward."""

    @staticmethod
    def forward(ctx, x, residual, weight, bias, rng_state, p, site, eps):
        out, mean, rstd = ops.dropout_add_norm_fwd(
            x, residual, weight, bias, rng_state, p, site, eps, True
        )
        ctx.save_for_backward(x, residual, weight, mean, rstd, rng_state)
        ctx.args = (p, site)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        x, residual, weight, mean, rstd, rng_state = ctx.saved_tensors
        p, site = ctx.args
        need_x, need_residual, need_weight, need_bias = ctx.needs_input_grad[:4]
        # nothing dropped and one type: both gradients are the same tensor
        shared = p == 0.0 and x.dtype == residual.dtype
        grad_x, grad_residual, grad_weight, grad_bias = ops.dropout_add_norm_bwd(
            grad_output, x, residual, weight, mean, rstd, rng_state, p, site,
            need_x and not shared, need_residual or (shared and need_x), need_weight or need_bias,
        )
        if shared:
            grad_x = grad_residual
        return (
            grad_x if need_x else None, grad_residual if need_residual else None,
            grad_weight if need_weight else None, grad_bias if need_bias else None,
            None, None, None, None,
        )


class LevelGroupNormFunction(torch.autograd.Function):
    """``apply(x, weight, bias, num_groups, rows, eps, activation)``, `rows` the row count of every
    level.  Saves the inputs and two values a (sample, level, group)."""

    @staticmethod
    def forward(ctx, x, weight, bias, num_groups, rows, eps, activation):
        out, mean, rstd = ops.level_group_norm_fwd(
            x, weight, bias, num_groups, rows, eps, activation, True
        )
        ctx.save_for_backward(x, weight, bias, mean, rstd)
        ctx.args = (num_groups, rows, activation)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        x, weight, bias, mean, rstd = ctx.saved_tensors
        need_x, need_weight, need_bias = ctx.needs_input_grad[:3]
        grad_x, grad_weight, grad_bias = ops.level_group_norm_bwd(
            grad_output, x, weight, bias, mean, rstd, *ctx.args, need_x, need_weight or need_bias
        )
        return (
            grad_x if need_x else None, grad_weight if need_weight else None,
            grad_bias if need_bias else None, None, None, None, None,
        )


def _grad_wanted(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t.requires_grad for t in tensors)


def counter_dropout(
    x: torch.Tensor,
    p: float,
    rng_state: torch.Tensor | None = None,
    site: int = 0,
    activation: str = "none",
) -> torch.Tensor:
    """``keep ? act(x) / (1 - p) : 0`` with ``act`` the identity or "relu".

    The mask is a function of ``rng_state`` (int64 (seed, offset) on x's device, see
    ``new_rng_state``), ``site`` (a number that tells uses of one state apart) and the element's flat
    index: the same arguments give the same mask, in the backward too, whatever x's strides.  It
    comes from Philox4x32-7 at 16 bits an element: p is taken to the nearest multiple of 2^-16 and
    the scale belongs to that value.  A dropped element is 0 whatever x holds.  The state is read when
    the kernel runs, so a captured graph draws new masks if the caller changes it between replays;
    do not change it between a forward and its backward.  Without anything to do (p = 0, no
    activation) x itself is returned."""
    ops.check_dropout(x, p, rng_state, site, activation)
    if p == 0.0:
        if activation == "none":
            return x
        rng_state = None
    if _grad_wanted(x):
        return CounterDropoutFunction.apply(x, rng_state, p, site, activation)
    return ops.counter_dropout_fwd(x, rng_state, p, site, activation)


def dropout_add_layer_norm(
    x: torch.Tensor,
    residual: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor,
    p: float = 0.0,
    rng_state: torch.Tensor | None = None,
    site: int = 0,
    eps: float = 1e-5,
) -> torch.Tensor:
    """``LayerNorm(residual + counter_dropout(x, p, rng_state, site)) * weight + bias`` over the last
    dimension, in ``residual``'s dtype.

    ``residual`` has x's shape and dtype, or float32 next to a 16-bit x (autocast); ``weight`` and
    ``bias`` have residual's dtype or, next to a 16-bit x, float32.  Rows of up to 16 KiB in
    ``residual``'s dtype.  For the mask see ``counter_dropout``."""
    ops.check_add_norm(x, residual, weight, bias, p, rng_state, site, eps)
    if p == 0.0:
        rng_state = None
    if _grad_wanted(x, residual, weight, bias):
        return DropoutAddLayerNormFunction.apply(x, residual, weight, bias, rng_state, p, site, eps)
    return ops.dropout_add_norm_fwd(x, residual, weight, bias, rng_state, p, site, eps, False)[0]


def level_group_norm(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor,
    num_groups: int,
    spatial_shapes=None,
    eps: float = 1e-5,
    activation: str = "none",
) -> torch.Tensor:
    """Group norm, channels last, then ``activation`` ("none", "relu", "silu" or "gelu", the last by
    the error function).

    With ``spatial_shapes`` (the (H, W) pairs of up to 16 levels, as ``flatten_levels`` returns them)
    x is a flattened pyramid (N, S, C) and every level of every sample has statistics of its own;
    without, x is (N, ..., C) and a sample is normalised as a whole.  ``weight`` and ``bias`` are
    (C,) or, one set a level, (L, C), in x's dtype or float32 next to 16 bits.  The normal result for
    a level is that of ``torch.nn.functional.group_norm`` on its (N, C, H, W) map.  Rows (C channels)
    of up to 16 KiB."""
    rows = ops.level_rows(x, spatial_shapes)
    ops.check_group_norm(x, weight, bias, num_groups, rows, eps, activation)
    if _grad_wanted(x, weight, bias):
        return LevelGroupNormFunction.apply(x, weight, bias, num_groups, rows, eps, activation)
    return ops.level_group_norm_fwd(x, weight, bias, num_groups, rows, eps, activation, False)[0]
