"""Custom ops over the C ABI for the operators around the attention: counter-based dropout,
dropout + residual + layer norm, group norm of the flattened pyramid.

Same idiom as ``_ops``: opaque ``torch.library`` ops on ROCm tensors through ``libmsda.so``, no CPU
implementation.  Arguments are checked here, before anything is launched.
"""

from __future__ import annotations

import ctypes

import torch

from .. import _lib
from ._ops import _DTYPE_CODE, _stream_ptr

ACTIVATIONS = {
    "none": _lib.ACT_NONE,
    "relu": _lib.ACT_RELU,
    "silu": _lib.ACT_SILU,
    "gelu": _lib.ACT_GELU,
}
_HALF = (torch.bfloat16, torch.float16)
# bytes of a row (C columns) that the normalising kernels hold in one workgroup
MAX_ROW_BYTES = 16384
MAX_LEVELS = 16
MAX_DROP_ELEMENTS = 1 << 35


def _compute_dtype(dtype: torch.dtype) -> torch.dtype:
    return torch.float64 if dtype == torch.float64 else torch.float32


def _check_tensor(what: str, t: torch.Tensor) -> None:
    if t.dtype not in _DTYPE_CODE:
        raise TypeError(f"{what}: unsupported dtype {t.dtype}")
    if t.device.type not in ("cuda", "meta"):
        raise RuntimeError(f"{what} runs only on a ROCm GPU (HIP kernels); got a tensor on {t.device}")


def _check_rng(what: str, p: float, site: int, rng_state: torch.Tensor | None, x: torch.Tensor) -> None:
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"{what}: p must lie in [0, 1], got {p}")
    if not 0 <= site < 2**31:
        raise ValueError(f"{what}: site must lie in [0, 2**31), got {site}")
    if p == 0.0:
        return
    if rng_state is None:
        raise ValueError(f"{what}: p > 0 needs rng_state (see new_rng_state)")
    if rng_state.dtype != torch.int64 or tuple(rng_state.shape) != (2,):
        raise ValueError(
            f"{what}: rng_state must be an int64 tensor (seed, offset), got "
            f"{tuple(rng_state.shape)} {rng_state.dtype}"
        )
    if rng_state.device != x.device:
        raise RuntimeError(f"{what}: rng_state lives on {rng_state.device}, the input on {x.device}")
    if x.numel() > MAX_DROP_ELEMENTS:
        raise ValueError(f"{what}: at most 2**35 elements, got {x.numel()}")


def check_dropout(x, p, rng_state, site, activation) -> None:
    _check_tensor("counter_dropout", x)
    if activation not in ("none", "relu"):
        raise ValueError(f"counter_dropout: activation must be 'none' or 'relu', got {activation!r}")
    _check_rng("counter_dropout", p, site, rng_state, x)


def _check_params(what: str, weight, bias, x: torch.Tensor, dtype: torch.dtype) -> None:
    if bias.shape != weight.shape or bias.dtype != weight.dtype:
        raise ValueError(f"{what}: weight and bias must agree in shape and dtype")
    if weight.dtype != dtype and not (x.dtype in _HALF and weight.dtype == torch.float32):
        raise TypeError(
            f"{what}: parameters must be {dtype} (or float32 next to a 16-bit input), got {weight.dtype}"
        )
    if weight.device != x.device or bias.device != x.device:
        raise RuntimeError(f"{what}: all tensors must live on the same device")


def _check_row(what: str, columns: int, dtype: torch.dtype) -> None:
    if columns < 1 or columns * dtype.itemsize > MAX_ROW_BYTES:
        raise ValueError(
            f"{what}: rows of 1 to {MAX_ROW_BYTES // dtype.itemsize} columns of {dtype}, got {columns}"
        )


def check_add_norm(x, residual, weight, bias, p, rng_state, site, eps) -> None:
    what = "dropout_add_layer_norm"
    _check_tensor(what, x)
    _check_tensor(what, residual)
    if x.dim() < 1 or x.shape != residual.shape:
        raise ValueError(
            f"{what}: x and residual must agree in shape, got {tuple(x.shape)} and {tuple(residual.shape)}"
        )
    if residual.dtype != x.dtype and not (x.dtype in _HALF and residual.dtype == torch.float32):
        raise TypeError(
            f"{what}: residual must have x's dtype (or float32 next to a 16-bit x), got "
            f"{residual.dtype} next to {x.dtype}"
        )
    if residual.device != x.device:
        raise RuntimeError(f"{what}: all tensors must live on the same device")
    columns = x.shape[-1]
    _check_row(what, columns, residual.dtype)
    if tuple(weight.shape) != (columns,):
        raise ValueError(f"{what}: weight and bias must be ({columns},), got {tuple(weight.shape)}")
    _check_params(what, weight, bias, x, residual.dtype)
    if not eps >= 0.0:
        raise ValueError(f"{what}: eps must not be negative, got {eps}")
    if x.numel() // columns >= 2**31:
        raise ValueError(f"{what}: at most 2**31 - 1 rows, got {x.numel() // columns}")
    _check_rng(what, p, site, rng_state, x)


def level_rows(x: torch.Tensor, spatial_shapes) -> list[int]:
    """Rows of every level of x (N, S, C) from its (H, W) pairs; one level of all rows without."""
    what = "level_group_norm"
    if spatial_shapes is None:
        if x.dim() < 2:
            raise ValueError(f"{what}: expected (N, ..., C), got {tuple(x.shape)}")
        rows = 1
        for d in x.shape[1:-1]:
            rows *= d
        return [rows]
    if x.dim() != 3:
        raise ValueError(f"{what}: with spatial_shapes x must be (N, S, C), got {tuple(x.shape)}")
    if isinstance(spatial_shapes, torch.Tensor):
        spatial_shapes = spatial_shapes.tolist()  # a device read; pass a list to avoid it
    rows = []
    for h, w in spatial_shapes:
        if h < 1 or w < 1:
            raise ValueError(f"{what}: spatial_shapes must be positive, got {list(spatial_shapes)}")
        rows.append(int(h) * int(w))
    if not 1 <= len(rows) <= MAX_LEVELS:
        raise ValueError(f"{what}: 1 to {MAX_LEVELS} levels, got {len(rows)}")
    if sum(rows) != x.shape[1]:
        raise ValueError(
            f"{what}: x has {x.shape[1]} positions but spatial_shapes {list(spatial_shapes)} cover {sum(rows)}"
        )
    return rows


def check_group_norm(x, weight, bias, num_groups, rows, eps, activation) -> None:
    what = "level_group_norm"
    _check_tensor(what, x)
    columns = x.shape[-1]
    _check_row(what, columns, x.dtype)
    if num_groups < 1 or columns % num_groups != 0:
        raise ValueError(f"{what}: {columns} channels do not divide into {num_groups} groups")
    if tuple(weight.shape) not in ((columns,), (len(rows), columns)):
        raise ValueError(
            f"{what}: weight and bias must be ({columns},) or ({len(rows)}, {columns}), got {tuple(weight.shape)}"
        )
    _check_params(what, weight, bias, x, x.dtype)
    if not eps >= 0.0:
        raise ValueError(f"{what}: eps must not be negative, got {eps}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"{what}: activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    if x.shape[0] * sum(rows) >= 2**31:
        raise ValueError(f"{what}: at most 2**31 - 1 positions, got {x.shape[0] * sum(rows)}")


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _wanted(t: torch.Tensor, wanted: bool, make=torch.empty_like) -> torch.Tensor:
    """A gradient's buffer, or an empty tensor where it is not wanted."""
    return make(t, memory_format=torch.contiguous_format) if wanted else t.new_empty(0)


# ---- dropout ------------------------------------------------------------------------------------


@torch.library.custom_op("unipercept::counter_dropout_fwd", mutates_args=())
def counter_dropout_fwd(
    x: torch.Tensor, rng_state: torch.Tensor | None, p: float, site: int, activation: str
) -> torch.Tensor:
    check_dropout(x, p, rng_state, site, activation)
    x = x.contiguous()
    out = torch.empty_like(x)
    if x.numel() == 0:
        return out
    state = None if rng_state is None else rng_state.contiguous()
    with torch.cuda.device_of(x):
        rc = _lib.load().msda_dropout_forward(
            x.data_ptr(), out.data_ptr(), _ptr(state), x.numel(), p, site, ACTIVATIONS[activation],
            _DTYPE_CODE[x.dtype], _stream_ptr(x.device),
        )
    _lib.check(rc, "msda_dropout_forward")
    return out


@counter_dropout_fwd.register_fake
def _(x, rng_state, p, site, activation):
    return torch.empty_like(x, memory_format=torch.contiguous_format)


@torch.library.custom_op("unipercept::counter_dropout_bwd", mutates_args=())
def counter_dropout_bwd(
    grad_output: torch.Tensor, out: torch.Tensor | None, rng_state: torch.Tensor | None, p: float,
    site: int, activation: str,
) -> torch.Tensor:
    """`out` is the forward's output with activation "relu", not needed otherwise."""
    relu = activation == "relu"
    check_dropout(grad_output, 0.0 if relu else p, rng_state, site, activation)
    grad_output = grad_output.contiguous()
    if relu and (out is None or out.shape != grad_output.shape or out.dtype != grad_output.dtype):
        raise ValueError("counter_dropout: the ReLU's gradient needs the forward's output")
    if out is not None:
        out = out.contiguous()
    grad = torch.empty_like(grad_output)
    if grad.numel() == 0:
        return grad
    state = None if rng_state is None else rng_state.contiguous()
    with torch.cuda.device_of(grad_output):
        rc = _lib.load().msda_dropout_backward(
            grad_output.data_ptr(), _ptr(out), grad.data_ptr(), _ptr(state), grad.numel(), p, site,
            ACTIVATIONS[activation], _DTYPE_CODE[grad.dtype], _stream_ptr(grad.device),
        )
    _lib.check(rc, "msda_dropout_backward")
    return grad


@counter_dropout_bwd.register_fake
def _(grad_output, out, rng_state, p, site, activation):
    return torch.empty_like(grad_output, memory_format=torch.contiguous_format)


# ---- dropout + residual + layer norm ------------------------------------------------------------


@torch.library.custom_op("unipercept::dropout_add_norm_fwd", mutates_args=())
def dropout_add_norm_fwd(
    x: torch.Tensor,
    residual: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor,
    rng_state: torch.Tensor | None,
    p: float,
    site: int,
    eps: float,
    stats: bool,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Returns the output and, with `stats`, mean and 1 / standard deviation of every row (empty
    tensors otherwise)."""
    check_add_norm(x, residual, weight, bias, p, rng_state, site, eps)
    x, residual = x.contiguous(), residual.contiguous()
    weight, bias = weight.contiguous(), bias.contiguous()
    columns = x.shape[-1]
    rows = x.numel() // columns
    out = torch.empty_like(residual)
    cdt = _compute_dtype(residual.dtype)
    mean = torch.empty(rows if stats else 0, dtype=cdt, device=x.device)
    rstd = torch.empty_like(mean)
    if rows == 0:
        return out, mean, rstd
    state = None if rng_state is None else rng_state.contiguous()
    with torch.cuda.device_of(x):
        rc = _lib.load().msda_dropout_add_norm_forward(
            x.data_ptr(), residual.data_ptr(), weight.data_ptr(), bias.data_ptr(), out.data_ptr(),
            mean.data_ptr() if stats else None, rstd.data_ptr() if stats else None, _ptr(state),
            rows, columns, p, site, eps, _DTYPE_CODE[x.dtype], _DTYPE_CODE[residual.dtype],
            _DTYPE_CODE[weight.dtype], _stream_ptr(x.device),
        )
    _lib.check(rc, "msda_dropout_add_norm_forward")
    return out, mean, rstd


@dropout_add_norm_fwd.register_fake
def _(x, residual, weight, bias, rng_state, p, site, eps, stats):
    rows = x.numel() // x.shape[-1] if stats else 0
    mean = residual.new_empty((rows,), dtype=_compute_dtype(residual.dtype))
    return (
        torch.empty_like(residual, memory_format=torch.contiguous_format), mean, torch.empty_like(mean),
    )


@torch.library.custom_op("unipercept::dropout_add_norm_bwd", mutates_args=())
def dropout_add_norm_bwd(
    grad_output: torch.Tensor,
    x: torch.Tensor,
    residual: torch.Tensor,
    weight: torch.Tensor,
    mean: torch.Tensor,
    rstd: torch.Tensor,
    rng_state: torch.Tensor | None,
    p: float,
    site: int,
    want_x: bool,
    want_residual: bool,
    want_params: bool,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients of x, residual, weight and bias; empty tensors where they are not wanted."""
    check_add_norm(x, residual, weight, weight, p, rng_state, site, 0.0)
    if grad_output.shape != x.shape or grad_output.device != x.device:
        raise ValueError(f"grad_output must be {tuple(x.shape)}, got {tuple(grad_output.shape)}")
    x, residual, weight = x.contiguous(), residual.contiguous(), weight.contiguous()
    grad_output = grad_output.to(residual.dtype).contiguous()
    columns = x.shape[-1]
    rows = x.numel() // columns
    if mean.numel() != rows or rstd.numel() != rows:
        raise ValueError("dropout_add_layer_norm: the backward needs the forward's row statistics")
    make = torch.zeros_like if rows == 0 else torch.empty_like
    grad_x, grad_residual = _wanted(x, want_x), _wanted(residual, want_residual)
    grad_weight, grad_bias = _wanted(weight, want_params, make), _wanted(weight, want_params, make)
    if rows == 0:
        return grad_x, grad_residual, grad_weight, grad_bias
    lib = _lib.load()
    xcode, rcode = _DTYPE_CODE[x.dtype], _DTYPE_CODE[residual.dtype]
    nbytes = lib.msda_dropout_add_norm_workspace_bytes(rows, columns, xcode, rcode) if want_params else 0
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
    state = None if rng_state is None else rng_state.contiguous()
    with torch.cuda.device_of(x):
        rc = lib.msda_dropout_add_norm_backward(
            grad_output.data_ptr(), x.data_ptr(), residual.data_ptr(), weight.data_ptr(),
            mean.data_ptr(), rstd.data_ptr(), grad_x.data_ptr() if want_x else None,
            grad_residual.data_ptr() if want_residual else None,
            grad_weight.data_ptr() if want_params else None,
            grad_bias.data_ptr() if want_params else None, _ptr(workspace), nbytes, _ptr(state),
            rows, columns, p, site, xcode, rcode, _DTYPE_CODE[weight.dtype], _stream_ptr(x.device),
        )
    _lib.check(rc, "msda_dropout_add_norm_backward")
    return grad_x, grad_residual, grad_weight, grad_bias


@dropout_add_norm_bwd.register_fake
def _(grad_output, x, residual, weight, mean, rstd, rng_state, p, site, want_x, want_residual, want_params):
    return (
        _wanted(x, want_x), _wanted(residual, want_residual), _wanted(weight, want_params),
        _wanted(weight, want_params),
    )


# ---- group norm ---------------------------------------------------------------------------------


def _rows_host(rows):
    return (ctypes.c_int64 * len(rows))(*rows)


@torch.library.custom_op("unipercept::level_group_norm_fwd", mutates_args=())
def level_group_norm_fwd(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor,
    num_groups: int,
    rows: list[int],
    eps: float,
    activation: str,
    stats: bool,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """x (N, ..., C) whose middle dimensions hold the levels' `rows`; returns the output and, with
    `stats`, mean and 1 / standard deviation (N, levels, groups) (empty tensors otherwise)."""
    check_group_norm(x, weight, bias, num_groups, rows, eps, activation)
    x, weight, bias = x.contiguous(), weight.contiguous(), bias.contiguous()
    n, s, c, levels = x.shape[0], sum(rows), x.shape[-1], len(rows)
    out = torch.empty_like(x)
    cdt = _compute_dtype(x.dtype)
    mean = torch.empty((n, levels, num_groups) if stats else (0,), dtype=cdt, device=x.device)
    rstd = torch.empty_like(mean)
    if x.numel() == 0:
        return out, mean, rstd
    lib, host, code = _lib.load(), _rows_host(rows), _DTYPE_CODE[x.dtype]
    nbytes = lib.msda_group_norm_workspace_bytes(host, n, s, c, num_groups, levels, code, 0)
    workspace = torch.empty(max(nbytes, 8), dtype=torch.uint8, device=x.device)
    with torch.cuda.device_of(x):
        rc = lib.msda_group_norm_forward(
            x.data_ptr(), weight.data_ptr(), bias.data_ptr(), out.data_ptr(),
            mean.data_ptr() if stats else None, rstd.data_ptr() if stats else None,
            workspace.data_ptr(), nbytes, host, n, s, c, num_groups, levels,
            levels if weight.dim() == 2 else 1, eps, ACTIVATIONS[activation], code,
            _DTYPE_CODE[weight.dtype], _stream_ptr(x.device),
        )
    _lib.check(rc, "msda_group_norm_forward")
    return out, mean, rstd


@level_group_norm_fwd.register_fake
def _(x, weight, bias, num_groups, rows, eps, activation, stats):
    shape = (x.shape[0], len(rows), num_groups) if stats else (0,)
    mean = x.new_empty(shape, dtype=_compute_dtype(x.dtype))
    return torch.empty_like(x, memory_format=torch.contiguous_format), mean, torch.empty_like(mean)


@torch.library.custom_op("unipercept::level_group_norm_bwd", mutates_args=())
def level_group_norm_bwd(
    grad_output: torch.Tensor,
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor,
    mean: torch.Tensor,
    rstd: torch.Tensor,
    num_groups: int,
    rows: list[int],
    activation: str,
    want_x: bool,
    want_params: bool,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients of x, weight and bias; empty tensors where they are not wanted."""
    check_group_norm(x, weight, bias, num_groups, rows, 0.0, activation)
    if grad_output.shape != x.shape or grad_output.device != x.device:
        raise ValueError(f"grad_output must be {tuple(x.shape)}, got {tuple(grad_output.shape)}")
    x, weight, bias = x.contiguous(), weight.contiguous(), bias.contiguous()
    grad_output = grad_output.to(x.dtype).contiguous()
    n, s, c, levels = x.shape[0], sum(rows), x.shape[-1], len(rows)
    if mean.numel() != n * levels * num_groups or rstd.numel() != mean.numel():
        raise ValueError("level_group_norm: the backward needs the forward's statistics")
    make = torch.zeros_like if x.numel() == 0 else torch.empty_like
    grad_x = _wanted(x, want_x)
    grad_weight, grad_bias = _wanted(weight, want_params, make), _wanted(bias, want_params, make)
    if x.numel() == 0:
        return grad_x, grad_weight, grad_bias
    lib, host, code = _lib.load(), _rows_host(rows), _DTYPE_CODE[x.dtype]
    nbytes = lib.msda_group_norm_workspace_bytes(host, n, s, c, num_groups, levels, code, 1)
    workspace = torch.empty(max(nbytes, 8), dtype=torch.uint8, device=x.device)
    with torch.cuda.device_of(x):
        rc = lib.msda_group_norm_backward(
            grad_output.data_ptr(), x.data_ptr(), weight.data_ptr(), bias.data_ptr(),
            mean.data_ptr(), rstd.data_ptr(), grad_x.data_ptr() if want_x else None,
            grad_weight.data_ptr() if want_params else None,
            grad_bias.data_ptr() if want_params else None, workspace.data_ptr(), nbytes, host, n, s,
            c, num_groups, levels, levels if weight.dim() == 2 else 1, ACTIVATIONS[activation],
            code, _DTYPE_CODE[weight.dtype], _stream_ptr(x.device),
        )
    _lib.check(rc, "msda_group_norm_backward")
    return grad_x, grad_weight, grad_bias


@level_group_norm_bwd.register_fake
def _(grad_output, x, weight, bias, mean, rstd, num_groups, rows, activation, want_x, want_params):
    return _wanted(x, want_x), _wanted(weight, want_params), _wanted(bias, want_params)
