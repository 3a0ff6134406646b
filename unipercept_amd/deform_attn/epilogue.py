"""Operators around the attention of an encoder layer, on hand-written HIP kernels.

* ``counter_dropout``: dropout (after an optional ReLU) whose mask is computed from counters in both
  directions and never stored;
* ``dropout_add_layer_norm``: ``LayerNorm(residual + dropout(x))``, one pass a direction;
* ``level_group_norm``: group norm of the flattened pyramid, every level on its own, with an
  activation.

All take float32, float64, bfloat16 and float16 tensors on a ROCm GPU (sums and statistics are held
in 32 bits or more), use the current stream, are differentiable once in reverse mode (a forward-mode
tangent raises ``NotImplementedError``), and give the same bits on every run.
``MSDeformAttnEncoderLayer(fused_epilogues=True)`` and ``LevelInputProjection`` call them.
"""

from __future__ import annotations

import torch

from .. import _lib


def new_rng_state(device, generator: torch.Generator | None = None) -> torch.Tensor:
    """A (seed, offset) pair for the dropout operators, drawn from torch's generator of `device`
    (or `generator`), so ``torch.manual_seed`` makes runs repeatable.  One pair serves any number of
    uses that differ in ``site``."""
    return torch.randint(
        -(2**63), 2**63 - 1, (2,), dtype=torch.int64, device=device, generator=generator
    )


def level_rows(spatial_shapes) -> list[int]:
    """Rows of every level from its (H, W) pairs."""
    if isinstance(spatial_shapes, torch.Tensor):
        spatial_shapes = spatial_shapes.tolist()  # a device read; pass a list to avoid it
    rows = []
    for h, w in spatial_shapes:
        if h < 1 or w < 1:
            raise ValueError(f"level_group_norm: spatial_shapes must be positive, got {list(spatial_shapes)}")
        rows.append(int(h) * int(w))
    if not rows:
        raise ValueError("level_group_norm: spatial_shapes is empty")
    return rows


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
    activation) x itself is returned.

    Under ``torch.func.vmap`` every sample counts its own elements from 0 and would drop the same ones:
    that is what ``randomness="same"`` asks for; with another mode the call is refused unless the
    states are mapped with the samples.  A call on the whole batch draws a mask for all of it."""
    return _lib.torch_ops().counter_dropout(x, p, rng_state, site, activation)


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
    return _lib.torch_ops().dropout_add_layer_norm(x, residual, weight, bias, p, rng_state, site, eps)


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
    rows = []
    if spatial_shapes is not None:
        if x.dim() != 3:
            raise ValueError(
                f"level_group_norm: with spatial_shapes x must be (N, S, C), got {tuple(x.shape)}"
            )
        rows = level_rows(spatial_shapes)
    return _lib.torch_ops().level_group_norm(x, weight, bias, num_groups, rows, eps, activation)
