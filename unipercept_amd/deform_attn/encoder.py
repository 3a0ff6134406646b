"""Pixel-decoder encoder built on ``MSDeformAttn``: the direct caller of the hot path.

The reference snapshot holds no pixel decoder (its model code that would call
``unipercept.nn.layers.deform_attn`` is absent); the stack follows the Deformable-DETR /
Mask2Former convention: per layer ``x = LN(x + MSDeformAttn(x + pos, ref, x))`` then
``x = LN(x + FFN(x))``, reference points at the pixel centres of every level, sine position
embeddings as in the reference's ``TrigonometricEmbed2d``
(sources/unipercept/nn/layers/position.py:63-83,94-122).  Everything here is PyTorch-ROCm
plumbing (hipBLASLt GEMMs, LayerNorm); the sampling itself runs in the HIP kernels, and so does all
that stands between the GEMMs with ``fused_epilogues`` and in ``LevelInputProjection``.
"""

from __future__ import annotations

import math

import torch
from torch import nn

from .epilogue import counter_dropout, dropout_add_layer_norm, level_group_norm, new_rng_state
from .layer import MSDeformAttn, token_linear


def sine_position_embedding(
    height: int,
    width: int,
    num_pos_feats: int = 128,
    temperature: float = 10000.0,
    normalize: bool = True,
    scale: float | None = None,
    device=None,
    dtype: torch.dtype = torch.float32,
) -> torch.Tensor:
    """(2 * num_pos_feats, H, W) sine/cosine embedding of the pixel grid: channels
    ``[0, F)`` encode y, ``[F, 2F)`` encode x; even channels sine, odd channels cosine of
    ``coordinate / temperature ** (2 * (c // 2) / F)``; coordinates count from 1 and, when
    ``normalize``, are divided by the last coordinate (+1e-6) and multiplied by ``scale``
    (default 2*pi).  Same arithmetic as ``trigonometric_embed_2d`` of the reference
    (sources/unipercept/nn/layers/position.py:63-83)."""
    if num_pos_feats % 2:
        raise ValueError("num_pos_feats must be even")
    if scale is not None and not normalize:
        raise ValueError("scale needs normalize=True")
    scale = 2.0 * math.pi if scale is None else scale
    y = torch.arange(1, height + 1, dtype=torch.float32, device=device)
    x = torch.arange(1, width + 1, dtype=torch.float32, device=device)
    if normalize:
        y = y / (y[-1] + 1e-6) * scale
        x = x / (x[-1] + 1e-6) * scale
    c = torch.arange(num_pos_feats, dtype=torch.float32, device=device)
    dim_t = temperature ** (2.0 * torch.div(c, 2, rounding_mode="floor") / num_pos_feats)
    ang_y = y[:, None] / dim_t[None, :]  # (H, F)
    ang_x = x[:, None] / dim_t[None, :]  # (W, F)
    even = (torch.arange(num_pos_feats, device=device) % 2 == 0)[None, :]
    pos_y = torch.where(even, ang_y.sin(), ang_y.cos())  # (H, F)
    pos_x = torch.where(even, ang_x.sin(), ang_x.cos())  # (W, F)
    out = torch.cat(
        (
            pos_y.t()[:, :, None].expand(num_pos_feats, height, width),
            pos_x.t()[:, None, :].expand(num_pos_feats, height, width),
        ),
        dim=0,
    )
    return out.to(dtype)


def encoder_reference_points(
    spatial_shapes, valid_ratios: torch.Tensor | None = None, device=None, dtype=torch.float32, batch: int = 1
) -> torch.Tensor:
    """(N, S, L, 2): every position's own pixel centre, normalised by its level's valid extent,
    then expressed on every level (multiplied by that level's valid ratio).  Without
    ``valid_ratios`` (no padding) all ratios are 1 and the point is the same on all levels."""
    levels = [(int(h), int(w)) for h, w in spatial_shapes]
    if valid_ratios is None:
        valid_ratios = torch.ones(batch, len(levels), 2, device=device, dtype=dtype)
    refs = []
    for lvl, (h, w) in enumerate(levels):
        ys = torch.arange(h, device=device, dtype=dtype) + 0.5
        xs = torch.arange(w, device=device, dtype=dtype) + 0.5
        yy, xx = torch.meshgrid(ys, xs, indexing="ij")
        ry = yy.reshape(-1)[None] / (valid_ratios[:, None, lvl, 1] * h)
        rx = xx.reshape(-1)[None] / (valid_ratios[:, None, lvl, 0] * w)
        refs.append(torch.stack((rx, ry), -1))
    ref = torch.cat(refs, 1)  # (N, S, 2)
    return ref[:, :, None, :] * valid_ratios[:, None, :, :]


def _autocast_to_fp32(t: torch.Tensor) -> torch.Tensor:
    """What autocast does to the inputs of a norm: 16 bits become fp32, so its result is fp32."""
    if torch.is_autocast_enabled("cuda") and t.dtype in (torch.bfloat16, torch.float16):
        return t.float()
    return t


def _dropout_probability(module: nn.Module) -> float:
    """What the fused route takes from a layer's dropout module: its p while the module itself trains."""
    if type(module) is nn.Dropout:
        return module.p if module.training else 0.0
    if type(module) is nn.Identity:
        return 0.0
    raise TypeError(
        f"fused_epilogues: the layer's dropout must be nn.Dropout or nn.Identity, got {type(module).__name__}"
    )


class MSDeformAttnEncoderLayer(nn.Module):
    """``fused_epilogues``: dropout, the residual sums, the layer norms and the ReLU run in the HIP
    kernels of ``epilogue`` (ROCm tensors only): ``dropout_add_layer_norm`` behind the attention and
    behind the feed-forward network, ``counter_dropout`` on its hidden tensor.  Parameters and state
    dicts are the same; dropout masks come from ``rng_state`` (see ``forward``)."""

    # uses of one rng_state in a layer: behind the attention, the hidden tensor, behind the network
    RNG_SITES = 3

    def __init__(
        self,
        d_model: int = 256,
        d_ffn: int = 1024,
        dropout: float = 0.0,
        n_levels: int = 3,
        n_heads: int = 8,
        n_points: int = 4,
        fused_epilogues: bool = False,
    ):
        super().__init__()
        self.fused_epilogues = fused_epilogues
        self.self_attn = MSDeformAttn(d_model, n_levels, n_heads, n_points)
        self.norm1 = nn.LayerNorm(d_model)
        self.linear1 = nn.Linear(d_model, d_ffn)
        self.linear2 = nn.Linear(d_ffn, d_model)
        self.norm2 = nn.LayerNorm(d_model)
        self.dropout = nn.Dropout(dropout)

    def forward(
        self,
        src: torch.Tensor,
        pos: torch.Tensor | None,
        reference_points: torch.Tensor,
        spatial_shapes: torch.Tensor,
        level_start_index: torch.Tensor,
        padding_mask: torch.Tensor | None = None,
        rng_state: torch.Tensor | None = None,
        rng_site: int = 0,
    ) -> torch.Tensor:
        """``rng_state``, ``rng_site`` (with ``fused_epilogues``): the state and the first of
        ``RNG_SITES`` sites of the dropout masks; without a state one is drawn from torch's
        generator when dropout is active."""
        query = src if pos is None else src + pos
        attn = self.self_attn(
            query, reference_points, src, spatial_shapes, level_start_index, padding_mask
        )
        if self.fused_epilogues:
            return self._fused_rest(src, attn, rng_state, rng_site)
        src = self.norm1(src + self.dropout(attn))
        hidden = torch.relu(token_linear(src, self.linear1.weight, self.linear1.bias))
        ffn = token_linear(self.dropout(hidden), self.linear2.weight, self.linear2.bias)
        return self.norm2(src + self.dropout(ffn))

    def _fused_rest(self, src, attn, rng_state, rng_site):
        p = _dropout_probability(self.dropout)
        if p > 0.0 and rng_state is None:
            rng_state = new_rng_state(src.device)
        src = _autocast_to_fp32(src)  # the normalised stream
        norm1, norm2 = self.norm1, self.norm2
        src = dropout_add_layer_norm(
            attn, src, _autocast_to_fp32(norm1.weight), _autocast_to_fp32(norm1.bias), p, rng_state,
            rng_site, norm1.eps,
        )
        hidden = token_linear(src, self.linear1.weight, self.linear1.bias)
        hidden = counter_dropout(hidden, p, rng_state, rng_site + 1, "relu")
        ffn = token_linear(hidden, self.linear2.weight, self.linear2.bias)
        return dropout_add_layer_norm(
            ffn, src, _autocast_to_fp32(norm2.weight), _autocast_to_fp32(norm2.bias), p, rng_state,
            rng_site + 2, norm2.eps,
        )


class MSDeformAttnEncoder(nn.Module):
    """``num_layers`` encoder layers over the flattened multi-level feature maps."""

    def __init__(self, num_layers: int = 6, **layer_kwargs):
        super().__init__()
        self.layers = nn.ModuleList(MSDeformAttnEncoderLayer(**layer_kwargs) for _ in range(num_layers))

    def forward(
        self,
        src: torch.Tensor,
        spatial_shapes: torch.Tensor,
        level_start_index: torch.Tensor,
        pos: torch.Tensor | None = None,
        valid_ratios: torch.Tensor | None = None,
        padding_mask: torch.Tensor | None = None,
        spatial_shapes_list=None,
    ) -> torch.Tensor:
        # the level shapes as Python ints: pass spatial_shapes_list to avoid a device read
        levels = spatial_shapes_list if spatial_shapes_list is not None else spatial_shapes.tolist()
        ref = encoder_reference_points(
            levels, valid_ratios, device=src.device, dtype=src.dtype, batch=src.shape[0]
        )
        if ref.shape[0] != src.shape[0]:
            ref = ref.expand(src.shape[0], -1, -1, -1)
        ref = ref.contiguous()
        # one state for the dropout masks of the stack, sites of its own for every fused layer
        rng_state = None
        for i, layer in enumerate(self.layers):
            args = (src, pos, ref, spatial_shapes, level_start_index, padding_mask)
            if getattr(layer, "fused_epilogues", False) and _dropout_probability(layer.dropout) > 0.0:
                if rng_state is None:
                    rng_state = new_rng_state(src.device)
                args += (rng_state, i * MSDeformAttnEncoderLayer.RNG_SITES)
            src = layer(*args)
        return src


def flatten_levels(features, position_feats: int | None = None):
    """Flattens (N, C, H_l, W_l) maps into (N, S, C) plus the level tables, and, when
    ``position_feats`` is given, the matching sine position embeddings (N, S, 2*position_feats)."""
    shapes = [(f.shape[-2], f.shape[-1]) for f in features]
    src = torch.cat([f.flatten(2).transpose(1, 2) for f in features], dim=1)
    dev = src.device
    spatial_shapes = torch.as_tensor(shapes, dtype=torch.long, device=dev)
    level_start_index = torch.cat(
        (spatial_shapes.new_zeros((1,)), spatial_shapes.prod(1).cumsum(0)[:-1])
    )
    pos = None
    if position_feats is not None:
        pos = torch.cat(
            [
                sine_position_embedding(h, w, position_feats, device=dev, dtype=src.dtype)
                .flatten(1)
                .t()
                for h, w in shapes
            ],
            dim=0,
        )[None].expand(src.shape[0], -1, -1)
    return src, spatial_shapes, level_start_index, shapes, pos


class LevelInputProjection(nn.Module):
    """Input projections of a pixel decoder: for every level a 1 x 1 convolution to ``d_model``
    channels and a group norm (with an optional activation), flattened to tokens.

    ``forward(features)`` takes the (N, C_l, H_l, W_l) maps and returns what ``flatten_levels``
    returns for the projected maps.  The convolutions run as token GEMMs on the channels-last maps,
    the norms of all levels as one ``level_group_norm`` over the flattened pyramid (parameters
    ``norm_weight`` and ``norm_bias`` (L, d_model), one set a level); ROCm tensors only.  Under autocast
    the norms and what they return are fp32, as torch's group norm is.

    A state dict of per-level ``(nn.Conv2d(c, d_model, 1), nn.GroupNorm)`` pairs does not load as it is:
    ``projections.l.weight`` is the convolution's weight with its two spatial dimensions taken off,
    ``projections.l.bias`` its bias, and ``norm_weight[l]``, ``norm_bias[l]`` are the norm's."""

    def __init__(
        self,
        in_channels,
        d_model: int = 256,
        num_groups: int = 32,
        activation: str = "none",
        eps: float = 1e-5,
    ):
        super().__init__()
        self.projections = nn.ModuleList(nn.Linear(int(c), d_model) for c in in_channels)
        if d_model % num_groups != 0:
            raise ValueError(f"d_model ({d_model}) must be divisible by num_groups ({num_groups})")
        self.norm_weight = nn.Parameter(torch.ones(len(self.projections), d_model))
        self.norm_bias = nn.Parameter(torch.zeros(len(self.projections), d_model))
        self.num_groups = num_groups
        self.activation = activation
        self.eps = eps
        for proj in self.projections:
            nn.init.xavier_uniform_(proj.weight)
            nn.init.zeros_(proj.bias)

    def forward(self, features, position_feats: int | None = None):
        if len(features) != len(self.projections):
            raise ValueError(f"expected {len(self.projections)} levels, got {len(features)}")
        maps = []
        for f, proj in zip(features, self.projections):
            tokens = token_linear(f.permute(0, 2, 3, 1), proj.weight, proj.bias)
            tokens = _autocast_to_fp32(tokens)  # before the flattening: the embeddings take its type
            maps.append(tokens.permute(0, 3, 1, 2))  # a view, as flatten_levels takes it
        src, spatial_shapes, level_start_index, shapes, pos = flatten_levels(maps, position_feats)
        src = level_group_norm(
            src, _autocast_to_fp32(self.norm_weight), _autocast_to_fp32(self.norm_bias), self.num_groups,
            shapes, self.eps, self.activation,
        )
        return src, spatial_shapes, level_start_index, shapes, pos
