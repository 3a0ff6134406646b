"""The operators around the attention on the GPU, against the oracle in 64 bits.

Tolerances are sums of roundings, first order.  r is half a step of the compute type (2^-24, 2^-53
for fp64) relative to a value, half_step() that of the stored result.  A sum of n terms is off by at
most (depth of the additions) * r * (sum of magnitudes); the depths that the kernels use on these
sizes are bounded by
  DEPTH_ROW = 60    row sums: <= 32 values a lane, 6 levels of a wave, 4 waves, product with 1 / C
  DEPTH_GROUP = 300 group sums: <= 8 rows a thread, <= 256 row lanes, channels and chunks in a tree
  DEPTH_THREAD = 8  rows of one thread between merges of group statistics
  DEPTH_COLUMN = 120 + rows / 1000   column sums over workgroups
"""

from __future__ import annotations

import ctypes
import time

import pytest
import torch

from oracle import epilogue_ref as ref
from unipercept_amd import _lib
from unipercept_amd.deform_attn import (
    LevelInputProjection,
    MSDeformAttnEncoder,
    MSDeformAttnEncoderLayer,
    counter_dropout,
    dropout_add_layer_norm,
    flatten_levels,
    level_group_norm,
    new_rng_state,
)

pytestmark = pytest.mark.gpu

F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16
DEPTH_ROW, DEPTH_GROUP, DEPTH_THREAD = 60, 300, 8
STATE = (-0x1234567812345678, 0x0FEDCBA987654321)


def rng(state=STATE):
    return torch.tensor(state, dtype=torch.int64, device="cuda")


def unit(*dtypes):
    return 2.0**-53 if F64 in dtypes else 2.0**-24


def half_step(want, dtype):
    """Half a step of `dtype` at the values, and of its subnormals near zero."""
    return want.abs() * (torch.finfo(dtype).eps / 2) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def check(name, got, want, bound):
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), (
        name, int(bad.sum()), (got - want).abs()[bad].max().item(), bound.expand_as(want)[bad].max().item(),
        [int(v) for v in bad.nonzero()[0]])


def normal(shape, dtype, seed, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g, dtype=F64) * scale + shift).to(dtype)


# ---- dropout --------------------------------------------------------------------------------------


@pytest.mark.parametrize("numel", [1, 7, 8, 9, 64, 2047, 2049, 100003])
@pytest.mark.parametrize("dtype", [F32, F64, BF16, F16])
@pytest.mark.parametrize("activation", ["none", "relu"])
def test_dropout_and_gradient(numel, dtype, activation):
    x, dy = normal((numel,), dtype, numel), normal((numel,), dtype, numel + 1)
    for p, site in ((0.1, 0), (0.5, 7), (0.25, 2**31 - 1)):
        xd = x.cuda().requires_grad_(True)
        y = counter_dropout(xd, p, rng(), site, activation)
        y.backward(dy.cuda())
        want = ref.dropout(x, p, STATE, site, activation)
        grad = ref.dropout_grad(dy, x, p, STATE, site, activation)
        # two roundings in the compute type (the scale, the product) and the stored one
        assert torch.equal(y.cpu() == 0, want == 0)
        check("y", y, want, half_step(want, dtype) + 2 * unit(dtype) * want.abs())
        check("dx", xd.grad, grad, half_step(grad, dtype) + 2 * unit(dtype) * grad.abs())


@pytest.mark.parametrize("p", [0.0, 1e-9, 1 - 1e-9, 1.0])
def test_dropout_at_the_ends(p):
    x = normal((300007,), F32, 5).cuda().requires_grad_(True)
    for activation in ("none", "relu"):
        y = counter_dropout(x, p, rng(), 3, activation)
        want = ref.dropout(x.detach().cpu(), p, STATE, 3, activation)
        assert torch.equal(y.detach().cpu() == 0, want == 0)
        check("y", y, want, 3 * 2.0**-24 * want.abs())
        (g,) = torch.autograd.grad(y.sum(), x)
        grad = ref.dropout_grad(torch.ones(300007), x.detach().cpu(), p, STATE, 3, activation)
        check("dx", g, grad, 3 * 2.0**-24 * grad.abs())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_dropout_leaves_nothing_of_dropped_values(dtype):
    """NaN and infinities vanish where they are dropped and stay where they are kept."""
    n = 4096
    x = torch.ones(n, dtype=dtype)
    x[0::3], x[1::3], x[2::3] = float("nan"), float("inf"), float("-inf")
    keep = torch.from_numpy(ref.keep(0, n, 0.5, *STATE, 1))
    y = counter_dropout(x.cuda(), 0.5, rng(), 1).cpu()
    assert torch.equal(y[~keep], torch.zeros(int((~keep).sum()), dtype=dtype))
    assert torch.equal(y[keep].isnan(), x[keep].isnan()) and torch.equal(y[keep].isinf(), x[keep].isinf())
    xd = x.cuda().requires_grad_(True)
    z = counter_dropout(xd, 0.5, rng(), 1, "relu")
    z.backward(torch.ones_like(z))
    passed = keep & ~(x <= 0)
    assert torch.equal(z.detach().cpu() == 0, ~passed) and torch.equal(xd.grad.cpu() != 0, passed)


def test_dropout_mask_does_not_depend_on_strides_or_placement():
    x = normal((33, 40), F32, 9).cuda()
    want = counter_dropout(x, 0.3, rng(), 2)
    for other in (x.t().contiguous().t(), torch.cat((x, x), 1)[:, :40], x.repeat_interleave(2, 0)[::2]):
        assert not other.is_contiguous()
        assert torch.equal(counter_dropout(other, 0.3, rng(), 2), want)
    for dtype in (BF16, F16, F32, F64):
        flat = x.flatten().to(dtype)
        for shift in (1, 3):  # starts that no vector is aligned to
            moved = torch.cat((flat.new_zeros(shift), flat))[shift:]
            assert moved.data_ptr() % 16 != 0
            assert torch.equal(counter_dropout(moved, 0.3, rng(), 2), counter_dropout(flat, 0.3, rng(), 2))
    expanded = torch.ones(1, device="cuda").expand(1000)
    assert torch.equal(counter_dropout(expanded, 0.3, rng(), 0) != 0,
                       torch.from_numpy(ref.keep(0, 1000, 0.3, *STATE, 0)).cuda())


def test_dropout_of_empty_tensors():
    x = torch.empty(0, 5, device="cuda", requires_grad=True)
    y = counter_dropout(x, 0.3, rng(), 0, "relu")
    y.sum().backward()
    assert y.shape == x.grad.shape == (0, 5)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_dropout_beyond_32_bit_offsets(dtype):
    """The far end of a tensor of more than 2^31 elements has the bits of its far indices."""
    n = (1 << 31) + 1003
    x = torch.ones(n, dtype=dtype, device="cuda")
    y = counter_dropout(x, 0.5, rng(), 1)
    del x
    for first in (0, (1 << 31) - 500, n - 1000):
        want = torch.from_numpy(ref.keep(first, 1000, 0.5, *STATE, 1))
        assert torch.equal(y[first : first + 1000].cpu() != 0, want)


# ---- dropout + residual + layer norm ----------------------------------------------------------------

KINDS = {
    # x, residual, parameters
    "f32": (F32, F32, F32),
    "f64": (F64, F64, F64),
    "bf16": (BF16, BF16, BF16),
    "bf16_wide_params": (BF16, BF16, F32),
    "bf16_in_f32": (BF16, F32, F32),
    "f16": (F16, F16, F16),
    "f16_in_f32": (F16, F32, F32),
}
ROWS = [(1, 1), (1, 16), (2, 64), (3, 7), (5, 63), (300, 256), (17, 257), (1200, 24), (9, 515), (4, 1000),
        (3, 1024), (2, 2048), (5, 2047), (1, 130), (4, 4), (70, 160), (33, 297), (40, 640), (21, 1500)]
WIDE = {"f32": [(3, 4096), (2, 4095)], "bf16": [(3, 8192), (2, 8191), (2, 4104)], "f64": [(2, 2048), (2, 2047)],
        "f16_in_f32": [(3, 4096), (2, 4093)]}


def norm_bounds(x, weight, parts, dy, p, kind):
    """Bounds of (out, grad_x, grad_residual, grad_weight, grad_bias) less the stored rounding."""
    r, D = unit(*kind), DEPTH_ROW
    u, s, w = parts["u"], parts["rstd"], weight.double()
    h = parts["size"].amax(-1, keepdim=True)
    e_d = (D + 5) * r * h  # of h - mean
    e_u = e_d * s * (1 + u.abs()) + D * r * u.abs()
    e_s = e_d * s + D * r  # relative, of rstd
    g = dy.double() * w
    mg, mgu = g.abs().mean(-1, keepdim=True), (g * u).abs().mean(-1, keepdim=True)
    m2 = (g * u).mean(-1, keepdim=True).abs()
    dh = s * (g - g.mean(-1, keepdim=True) - u * (g * u).mean(-1, keepdim=True))
    e_dh = s * (
        4 * r * g.abs() + (D + 4) * r * mg + u.abs() * ((D + 4) * r * mgu + (g.abs() * e_u).mean(-1, keepdim=True))
        + e_u * m2
    ) + e_s * dh.abs() + 2 * r * dh.abs()
    f = parts["f"]
    c, rows = u.shape[-1], u.numel() // u.shape[-1]
    column = 120 + rows / 1000
    e_w = (column * r * (dy.double() * u).abs() + dy.double().abs() * e_u).reshape(-1, c).sum(0)
    e_b = (column * r * dy.double().abs()).reshape(-1, c).sum(0)
    e_out = e_u * w.abs() + 3 * r * ((u * w).abs() + 1)
    return e_out, e_dh * f + 2 * r * (dh * f).abs(), e_dh, e_w, e_b


def run_norm(kind, shape, p, seed=1, scale=1.0, shift=0.0):
    kinds = KINDS[kind]
    xt, rt, pt = kinds
    c = shape[-1]
    x, res = normal(shape, xt, seed, scale, shift), normal(shape, rt, seed + 1, scale, shift)
    w, b = normal((c,), pt, seed + 2, 0.3, 1.0), normal((c,), pt, seed + 3, 0.3)
    dy = normal(shape, rt, seed + 4)
    leaves = [t.cuda().requires_grad_(True) for t in (x, res, w, b)]
    out = dropout_add_layer_norm(*leaves, p=p, rng_state=rng(), site=5)
    assert out.dtype == rt
    out.backward(dy.cuda())
    want, parts = ref.add_norm(x, res, w, b, p, STATE, 5, 1e-5)
    grads = ref.add_norm_grad(dy, w, parts)
    bounds = norm_bounds(x, w, parts, dy, p, kinds)
    names = ("out", "dx", "dres", "dw", "db")
    for name, got, exact, bound in zip(names, [out] + [t.grad for t in leaves], (want, *grads), bounds):
        check((name, kind, shape, p), got, exact, bound + half_step(exact, got.dtype))


@pytest.mark.parametrize("shape", ROWS)
@pytest.mark.parametrize("kind", sorted(KINDS))
def test_add_norm_and_gradient(kind, shape):
    for p in (0.0, 0.1):
        run_norm(kind, shape, p)


@pytest.mark.parametrize("kind", sorted(WIDE))
def test_add_norm_widest_rows(kind):
    for shape in WIDE[kind]:
        run_norm(kind, shape, 0.25)


def test_add_norm_other_ranks_and_many_rows():
    run_norm("f32", (2, 3, 5, 32), 0.5)
    run_norm("bf16", (40000, 8), 0.1)
    run_norm("f32", (7001, 129), 0.1)
    run_norm("bf16_in_f32", (5000, 256), 0.1)


def test_add_norm_far_from_zero():
    """A common offset of 1000 standard deviations: the variance is taken about the mean."""
    run_norm("f32", (64, 256), 0.0, scale=1.0, shift=500.0)
    run_norm("f32", (64, 1023), 0.0, scale=1.0, shift=500.0)


def test_add_norm_rows_without_spread():
    """Constant rows, rows of which everything is dropped, a single column: out = bias."""
    w, b = torch.randn(64, device="cuda"), torch.randn(64, device="cuda")
    x, zero = torch.randn(5, 64, device="cuda"), torch.zeros(5, 64, device="cuda")
    ones = torch.full((5, 64), 3.0, device="cuda")
    assert torch.equal(dropout_add_layer_norm(x, ones, w, b, 1.0, rng()), b.expand(5, 64))
    assert torch.equal(dropout_add_layer_norm(zero, ones, w, b), b.expand(5, 64))
    one = dropout_add_layer_norm(x[:, :1], zero[:, :1], w[:1], b[:1])
    assert torch.equal(one, b[:1].expand(5, 1))
    assert dropout_add_layer_norm(x[:0], zero[:0], w, b).shape == (0, 64)


def test_add_norm_not_finite_rows_stay_among_themselves():
    x, res = torch.randn(6, 40, device="cuda"), torch.randn(6, 40, device="cuda")
    w, b = torch.ones(40, device="cuda"), torch.zeros(40, device="cuda")
    clean = dropout_add_layer_norm(x, res, w, b)
    x[1, 3], x[4, 0] = float("nan"), float("inf")
    got = dropout_add_layer_norm(x, res, w, b)
    assert got[[1, 4]].isnan().all() and torch.equal(got[[0, 2, 3, 5]], clean[[0, 2, 3, 5]])


def test_add_norm_mask_is_that_of_the_dropout_alone():
    x, res = normal((37, 200), F32, 1).cuda(), torch.zeros(37, 200, device="cuda")
    w, b = torch.ones(200, device="cuda"), torch.zeros(200, device="cuda")
    want = dropout_add_layer_norm(counter_dropout(x, 0.4, rng(), 6), res, w, b)
    assert torch.equal(dropout_add_layer_norm(x, res, w, b, 0.4, rng(), 6), want)


@pytest.mark.parametrize("wanted", [(1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (1, 0, 1, 0), (0, 1, 0, 1)])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_add_norm_gradients_one_by_one(wanted, p):
    args = [normal((30, 48), F32, 1), normal((30, 48), F32, 2), normal((48,), F32, 3), normal((48,), F32, 4)]
    dy = normal((30, 48), F32, 5).cuda()
    full = [t.cuda().requires_grad_(True) for t in args]
    some = [t.cuda().requires_grad_(bool(k)) for t, k in zip(args, wanted)]
    for leaves in (full, some):
        dropout_add_layer_norm(*leaves, p=p, rng_state=rng(), site=1).backward(dy)
    for a, b, k in zip(full, some, wanted):
        assert torch.equal(a.grad, b.grad) if k else b.grad is None


def test_add_norm_of_a_tensor_with_itself():
    """x and residual one tensor: both gradients arrive in it."""
    x = normal((9, 32), F64, 1)
    w, b = normal((32,), F64, 2), normal((32,), F64, 3)
    dy = normal((9, 32), F64, 4)
    for p in (0.0, 0.5):
        xd = x.cuda().requires_grad_(True)
        dropout_add_layer_norm(xd, xd, w.cuda(), b.cuda(), p, rng(), 0).backward(dy.cuda())
        _, parts = ref.add_norm(x, x, w, b, p, STATE, 0, 1e-5)
        gx, gr, _, _ = ref.add_norm_grad(dy, w, parts)
        check("dx", xd.grad, gx + gr, 1e-12 * (1 + (gx + gr).abs()))


# ---- group norm -----------------------------------------------------------------------------------------

PYRAMIDS = {
    # name: (N, level shapes or None with a plain shape, C, groups)
    "one_row": (2, [(1, 1)], 8, 4),
    "one_channel": (3, [(5, 7)], 1, 1),
    "three_levels": (2, [(8, 16), (4, 8), (2, 4)], 64, 32),
    "one_group": (2, [(9, 13), (3, 1)], 48, 1),
    "channel_groups": (2, [(6, 9), (2, 3)], 24, 24),
    "uneven": (3, [(11, 17), (6, 9), (1, 2), (1, 1)], 96, 32),
    "odd_width": (2, [(10, 15), (5, 8)], 105, 35),
    "odd_groups": (1, [(31, 33)], 21, 3),
    "wide": (2, [(3, 5), (1, 4)], 2048, 32),
    "tall": (1, [(64, 64), (32, 32), (16, 16), (8, 8)], 256, 32),
    "batch": (16, [(4, 4)], 32, 8),
    "narrow": (2, [(40, 50)], 4, 2),
    # levels that no workgroup holds, next to one row: whole vectors, parts of vectors
    "long": (2, [(96, 130), (1, 1)], 64, 8),
    "long_odd": (1, [(96, 130), (2, 1)], 22, 2),
}


def group_bounds(x, parts, dy, activation, dtype):
    """Bounds of (out, grad_x, grad_weight, grad_bias) less the stored rounding."""
    r, D = unit(dtype), DEPTH_GROUP
    outs, gxs, gws, gbs, start = [], [], [], [], 0
    for q in parts:
        rows = q["u"].shape[1]
        d = dy[:, start : start + rows].double()
        start += rows
        u, z, s, w, groups = q["u"], q["z"], q["rstd"], q["w"], q["groups"]
        n, _, c = u.shape
        e_d = D * r * 2 * q["largest"]  # of x - mean
        # spread of a group, for the sums about a thread's first value
        ug = u.reshape(n, rows, groups, c // groups)
        span = (ug.amax((1, 3), keepdim=True) - ug.amin((1, 3), keepdim=True))
        span = span.expand(n, 1, groups, c // groups).reshape(n, 1, c)
        e_s = e_d * s + D * r + DEPTH_THREAD * r * span**2
        e_u = e_d * s + u.abs() * (e_s + 2 * r)
        e_z = e_u * w.abs() + 3 * r * ((u * w).abs() + q["b"].abs())
        own = (2 * z.abs() + 8) * r * (z.abs() + 1) if activation in ("silu", "gelu") else 0 * z
        outs.append(1.2 * e_z + own)
        k = ref.slope(z, activation)
        e_k = 0.8 * e_z + own if activation in ("silu", "gelu") else 0 * z
        dz = d * k
        e_dz = d.abs() * e_k + 2 * r * dz.abs()
        g, e_g = dz * w, (e_dz + r * dz.abs()) * w.abs()
        mean = lambda v: ref.group_mean(v, groups)
        m1, m2 = mean(g), mean(g * u)
        e_m1 = D * r * mean(g.abs()) + mean(e_g)
        e_m2 = D * r * mean((g * u).abs()) + mean(e_g * u.abs() + g.abs() * e_u)
        dx = s * (g - m1 - u * m2)
        gxs.append(s * (e_g + 3 * r * g.abs() + e_m1 + 2 * r * m1.abs() + u.abs() * e_m2 + (e_u + 3 * r * u.abs()) * m2.abs())
                   + (e_s + r) * dx.abs())
        gws.append((D * r * (dz * u).abs() + e_dz * u.abs() + dz.abs() * e_u).sum((0, 1)))
        gbs.append((D * r * dz.abs() + e_dz).sum((0, 1)))
    return torch.cat(outs, 1), torch.cat(gxs, 1), torch.stack(gws), torch.stack(gbs)


def run_group(case, dtype, param, activation, per_level=True, scale=1.5, shift=0.5, seed=1):
    n, levels, c, groups = PYRAMIDS[case]
    rows = [h * w for h, w in levels]
    x = normal((n, sum(rows), c), dtype, seed, scale, shift)
    shape = (len(rows), c) if per_level else (c,)
    w, b = normal(shape, param, seed + 1, 0.3, 1.0), normal(shape, param, seed + 2, 0.3)
    dy = normal(x.shape, dtype, seed + 3)
    want, parts = ref.group_norm(x, w, b, groups, rows, 1e-5, activation)
    if activation == "relu":
        # the gradient jumps at z = 0: none there, where a rounding of z decides
        z = torch.cat([q["z"] for q in parts], 1)
        dy = torch.where(z.abs() < 1e-3, torch.zeros_like(dy), dy)
    gx, gw, gb = ref.group_norm_grad(dy, parts, activation)
    e_out, e_x, e_w, e_b = group_bounds(x, parts, dy, activation, dtype)
    if not per_level:
        gw, gb, e_w, e_b = gw.sum(0), gb.sum(0), e_w.sum(0), e_b.sum(0)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    out = level_group_norm(*leaves, groups, levels, 1e-5, activation)
    out.backward(dy.cuda())
    for name, got, exact, bound in zip(
        ("out", "dx", "dw", "db"), [out] + [t.grad for t in leaves], (want, gx, gw, gb), (e_out, e_x, e_w, e_b)
    ):
        check((name, case, dtype, activation), got, exact, bound + half_step(exact, got.dtype))


@pytest.mark.parametrize("activation", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("kind", [(F32, F32), (F64, F64), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("case", sorted(PYRAMIDS))
def test_group_norm_and_gradient(case, kind, activation):
    run_group(case, *kind, activation)


@pytest.mark.parametrize("case", ["three_levels", "uneven"])
def test_group_norm_shared_parameters(case):
    run_group(case, F32, F32, "silu", per_level=False)
    run_group(case, BF16, F32, "none", per_level=False)


def test_group_norm_far_from_zero():
    run_group("three_levels", F32, F32, "none", scale=1.0, shift=300.0)
    run_group("tall", F32, F32, "none", scale=1.0, shift=300.0)


def test_group_norm_matches_the_maps():
    """Level by level the result is torch's group norm of the (N, C, H, W) map."""
    n, levels, c, groups = PYRAMIDS["uneven"]
    maps = [normal((n, c, h, w), F64, i).cuda() for i, (h, w) in enumerate(levels)]
    src, _, _, shapes, _ = flatten_levels(maps)
    w, b = normal((len(levels), c), F64, 8).cuda(), normal((len(levels), c), F64, 9).cuda()
    got = level_group_norm(src, w, b, groups, shapes)
    want = flatten_levels([torch.nn.functional.group_norm(m, groups, w[i], b[i]) for i, m in enumerate(maps)])[0]
    assert (got - want).abs().max() < 1e-12
    one = maps[0].permute(0, 2, 3, 1)  # a channels-last view, no level table
    got = level_group_norm(one, w[0], b[0], groups)
    assert got.shape == one.shape and torch.equal(got.flatten(1, 2), level_group_norm(
        src[:, : levels[0][0] * levels[0][1]], w[0], b[0], groups))


def test_group_norm_outliers_and_not_finite_groups():
    x = normal((2, 40, 16), F32, 3)
    x[0, 0, :4] = 1e4  # the first value of a chunk far from the rest
    want, _ = ref.group_norm(x, torch.ones(16), torch.zeros(16), 4, [40], 1e-5, "none")
    one, zero = torch.ones(16, device="cuda"), torch.zeros(16, device="cuda")
    got = level_group_norm(x.cuda(), one, zero, 4)
    # the variance is off by at most DEPTH_THREAD roundings of the outlier's own share of it
    check("outlier", got, want, 2.0**-24 * (DEPTH_GROUP * 2 * 1e4 / 1e3 + DEPTH_GROUP * want.abs() + 8))
    x[1, 7, 5] = float("nan")
    x[1, 9, 14] = float("inf")
    bad = level_group_norm(x.cuda(), one, zero, 4)
    assert bad[1, :, 4:8].isnan().all() and bad[1, :, 12:16].isnan().all()
    assert torch.equal(bad[0], got[0]) and torch.equal(bad[1, :, :4], got[1, :, :4])
    assert torch.equal(bad[1, :, 8:12], got[1, :, 8:12])
    const = level_group_norm(torch.full((1, 100, 16), 7.0, device="cuda"), one, zero + 0.25, 4)
    assert torch.equal(const, torch.full_like(const, 0.25))


GATE = {
    # (samples, levels, channels, groups): one launch, whole vectors and parts of vectors a group
    "small": (2, [(8, 16), (4, 8)], 64, 8),
    "small_parts": (2, [(8, 16), (4, 8)], 64, 32),
    # the forward in one launch, the gradient in three
    "mixed": (2, [(1, 1024), (1, 3)], 256, 32),
    "long": (2, [(96, 130), (1, 9)], 64, 8),
    "long_odd": (1, [(96, 130), (2, 9)], 21, 3),
    "long_short": (1, [(130, 130)], 3, 3),
}


@pytest.mark.parametrize("case", sorted(GATE))
@pytest.mark.parametrize("dtype", [F32, BF16, F64])
def test_group_norm_relu_gate_is_one_in_every_pass(case, dtype):
    """Elements whose z is a rounding away from 0: what the output shows as open is open in dx, dw and
    db, in every kernel.  Given the gate the gradient is that of the plain norm for the gated incoming
    gradient, with its bounds."""
    n, levels, c, groups = GATE[case]
    rows = [h * w for h, w in levels]
    wide = F64 if dtype == F64 else F32
    g = torch.Generator().manual_seed(len(case))
    x = (torch.randint(-8, 9, (n, sum(rows), c), generator=g).double() * 0.25 + 0.375).to(dtype)  # few values
    w = normal((len(rows), c), wide, 5, 0.3, 1.0)
    zero = torch.zeros_like(w)
    _, mean, rstd = _lib.torch_ops().level_group_norm_fwd(
        x.cuda(), w.cuda(), zero.cuda(), groups, rows, 1e-5, "relu", True)
    mean, rstd = (t.cpu().repeat_interleave(c // groups, -1) for t in (mean, rstd))  # (n, L, c)
    b, start = torch.empty_like(w), 0
    for level, r in enumerate(rows):
        # z = 0 but for its rounding where a channel has the value of its first row of the first sample
        b[level] = -(x[0, start].to(wide) - mean[0, level]) * (rstd[0, level] * w[level])
        start += r
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    out = level_group_norm(*leaves, groups, levels, 1e-5, "relu")
    out.backward(torch.ones_like(out))
    opened = out.detach().cpu() > 0
    dz = opened.to(dtype)
    _, parts = ref.group_norm(x, w, b, groups, rows, 1e-5, "none")
    z = torch.cat([q["z"] for q in parts], 1)
    assert (z.abs() < 1e-5).any(1).any(0).sum() > c // 2  # the case holds what it is about
    bounds = group_bounds(x, parts, dz, "none", dtype)[1:]
    assert torch.equal(leaves[2].grad.cpu().double(), torch.stack(
        [v.double().sum((0, 1)) for v in dz.split(rows, 1)]))  # whole numbers
    for name, t, want, bound in zip(("dx", "dw"), leaves, ref.group_norm_grad(dz, parts, "none"), bounds):
        check((name, case, dtype), t.grad, want, bound + half_step(want, t.grad.dtype))


@pytest.mark.parametrize("dtype,c,groups", [(F32, 1024, 32), (F32, 1023, 33), (BF16, 2048, 64), (BF16, 2047, 23), (F64, 512, 16)])
def test_group_norm_statistics_with_outliers(dtype, c, groups):
    """170 rows a thread, which the small levels of the other tests never give, with values far from the
    rest at the first rows of threads and in between.  A step of four rows adds five terms to a thread's
    M2, none larger than M2 after it; lanes, chunks and groups join in fewer than 100 additions more."""
    n, rows = 2, 170 * 1024
    depth = 5 * (170 // 4 + 3) + 100
    g = torch.Generator(device="cuda").manual_seed(3)
    clean = torch.empty(n, rows, c, dtype=dtype, device="cuda").normal_(generator=g)
    w = torch.ones(c, dtype=F64 if dtype == F64 else F32, device="cuda")
    for far in (1e4, -3e6):
        x = clean.clone()
        x[0, 0] = x[1, 172 * 9] = x[1, 172 * 700 + 3] = x[1, 172 * 700 + 77] = far
        _, mean, rstd = _lib.torch_ops().level_group_norm_fwd(x, w, w, groups, [rows], 1e-5, "none", True)
        for i in range(n):
            wide = x[i].double().view(rows, groups, c // groups)
            exact_mean = wide.mean((0, 2))
            exact = ((wide - exact_mean[:, None]).square().mean((0, 2)) + 1e-5).rsqrt()
            size = wide.abs().mean((0, 2))
            # (chunks of 172 rows join about the mean of the first, which an outlying row moves by far / 172)
            check(("mean", i, far), mean[i, 0], exact_mean.cpu(), (depth * unit(dtype) * (size + abs(far) / 172)).cpu())
            # half of the variance's relative error, two roundings of the root and the quotient
            check(("rstd", i, far), rstd[i, 0], exact.cpu(), ((depth / 2 + 4) * unit(dtype) * exact).cpu())


@pytest.mark.parametrize("c,groups", [(32, 4), (21, 3)])
def test_group_norm_not_finite_groups_of_long_levels(c, groups):
    """NaN and infinities stay in their (sample, level, group); a group without spread gives the bias."""
    rows, per = [96 * 130, 5000], c // groups
    x = normal((2, sum(rows), c), F32, 4).cuda()
    one, zero = torch.ones(c, device="cuda"), torch.zeros(c, device="cuda")
    shapes = [(96, 130), (50, 100)]
    clean = level_group_norm(x, one, zero, groups, shapes)
    for at, value in ((0, float("nan")), (rows[0] + 4321, float("inf")), (rows[0] - 1, float("-inf"))):
        bad = x.clone()
        bad[1, at, per + 1] = value
        got = level_group_norm(bad, one, zero, groups, shapes)
        hit = torch.zeros_like(got, dtype=torch.bool)
        hit[1, (slice(0, rows[0]) if at < rows[0] else slice(rows[0], None)), per : 2 * per] = True
        assert got[hit].isnan().all() and torch.equal(got[~hit], clean[~hit]), (at, value)
    const = level_group_norm(torch.full_like(x, 7.0), one, zero + 0.25, groups, shapes)
    assert torch.equal(const, torch.full_like(const, 0.25))


def test_group_norm_empty_and_partial_gradients():
    w, b = torch.ones(8, device="cuda", requires_grad=True), torch.zeros(8, device="cuda", requires_grad=True)
    for shape in ((0, 5, 8), (3, 0, 8)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        y = level_group_norm(x, w, b, 4)
        gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
        assert y.shape == gx.shape == shape and not gw.any() and not gb.any()
    x = normal((2, 30, 8), F32, 1).cuda()
    full = x.clone().requires_grad_(True)
    grads = torch.autograd.grad(level_group_norm(full, w, b, 4).square().sum(), (full, w, b))
    y = level_group_norm(x, w.detach(), b, 4)
    assert torch.equal(torch.autograd.grad(y.square().sum(), b)[0], grads[2])
    y = level_group_norm(full, w.detach(), b.detach(), 4)
    assert torch.equal(torch.autograd.grad(y.square().sum(), full)[0], grads[0])


# ---- all of them ------------------------------------------------------------------------------------------


def _calls(dtype=F32, seed=0):
    """name -> function of no arguments: outputs and gradients of one training step of each operator."""
    x, res = normal((2, 150, 64), dtype, seed).cuda(), normal((2, 150, 64), dtype, seed + 1).cuda()
    w, b = normal((64,), dtype, seed + 2).cuda(), normal((64,), dtype, seed + 3).cuda()
    dy = normal((2, 150, 64), dtype, seed + 4).cuda()
    state = rng()

    def step(f, *tensors):
        leaves = [t.detach().clone().requires_grad_(True) for t in tensors]
        out = f(*leaves)
        return [out.detach(), *torch.autograd.grad(out, leaves, dy)]

    calls = {
        "dropout": lambda: step(lambda x: counter_dropout(x, 0.2, state, 1), x),
        "relu_dropout": lambda: step(lambda x: counter_dropout(x, 0.2, state, 2, "relu"), x),
        "add_norm": lambda: step(lambda x, r, w, b: dropout_add_layer_norm(x, r, w, b, 0.2, state, 3), x, res, w, b),
        "group_norm": lambda: step(lambda x, w, b: level_group_norm(x, w, b, 8, [(10, 13), (4, 5)], activation="silu"), x, w, b),
    }
    return calls, state


@pytest.mark.parametrize("dtype", [F32, F64, BF16, F16])
def test_runs_agree_bit_for_bit(dtype):
    calls, _ = _calls(dtype)
    for name, call in calls.items():
        first = call()
        for _ in range(2):
            assert all(torch.equal(a, b) for a, b in zip(first, call())), name


def test_gradients_against_differences():
    """torch's gradcheck in fp64: every operator against differences of its own forward."""
    x, res = normal((2, 6, 6), F64, 1).cuda(), normal((2, 6, 6), F64, 2).cuda()
    w, b = normal((6,), F64, 3).cuda(), normal((6,), F64, 4).cuda()
    state = rng()
    x, res, w, b = (t.requires_grad_(True) for t in (x, res, w, b))
    check_ = torch.autograd.gradcheck
    assert check_(lambda x: counter_dropout(x, 0.4, state, 1), (x,))
    assert check_(lambda x: counter_dropout(x, 0.4, state, 1, "relu"), (x,))
    assert check_(lambda *a: dropout_add_layer_norm(*a, 0.4, state, 2), (x, res, w, b))
    assert check_(lambda *a: dropout_add_layer_norm(*a), (x, res, w, b))
    for act in ("none", "relu", "silu", "gelu"):
        assert check_(lambda x, w, b: level_group_norm(x, w, b, 3, [(2, 2), (1, 2)], activation=act), (x, w, b))


def test_second_differentiation_is_refused():
    x = torch.randn(4, 8, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(counter_dropout(x, 0.5, rng(), 0).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


def test_state_changed_before_the_backward_is_noticed():
    state = rng()
    x = torch.randn(4, 8, device="cuda", requires_grad=True)
    y = counter_dropout(x, 0.5, state, 0)
    state.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_other_streams():
    """Work on a stream of its own, inputs made on another one that it waits for."""
    calls, _ = _calls()
    want = {name: call() for name, call in calls.items()}
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = {name: call() for name, call in calls.items()}
    torch.cuda.current_stream().wait_stream(stream)
    for name in want:
        assert all(torch.equal(a, b) for a, b in zip(want[name], got[name])), name


def test_captured_steps_replay_with_new_masks():
    """Forward and backward of every operator in two graphs, replayed in turn with eager work between
    them and the generator state changed: every replay equals the eager result."""
    calls, state = _calls()
    for call in calls.values():
        call()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for call in calls.values():
            call()
    torch.cuda.current_stream().wait_stream(stream)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = {name: call() for name, call in calls.items()}
        graphs.append((graph, outs))
    for turn in range(4):
        state.copy_(torch.tensor((turn * 77 - 3, turn), dtype=torch.int64))
        want = {name: call() for name, call in calls.items()}
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, outs in graphs:
            for name in want:
                assert all(torch.equal(a, b) for a, b in zip(want[name], outs[name])), (turn, name)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_other_device_than_the_current_one():
    x = torch.randn(8, 64, device="cuda:1")
    w, b = torch.ones(64, device="cuda:1"), torch.zeros(64, device="cuda:1")
    with torch.cuda.device(0):
        assert dropout_add_layer_norm(x, x, w, b).device == x.device
        assert level_group_norm(x, w, b, 4).device == x.device


def test_outputs_stay_inside_their_buffers():
    """Through the C ABI with buffers of odd sizes inside larger ones: nothing else is written."""
    lib = _lib.load()
    st = torch.cuda.current_stream().cuda_stream
    code = {F32: 0, BF16: 2, F16: 3}
    for dtype in (F32, BF16, F16):
        for rows, c in ((1, 1), (3, 7), (11, 13), (5, 257), (2, 64)):
            n = rows * c

            def buffer(count, dt=dtype):
                whole = torch.full((count + 64,), 7.0, dtype=dt, device="cuda")
                return whole, whole[33 : 33 + count]

            x, dy = normal((n,), dtype, 1).cuda(), normal((n,), dtype, 2).cuda()
            w, b = normal((c,), F32, 3).cuda(), normal((c,), F32, 4).cuda()
            state = rng()
            bufs = {k: buffer(n) for k in ("drop", "out", "gx", "gr", "gn", "gnx")}
            stats = {k: buffer(rows, F32) for k in ("mean", "rstd")}
            gstats = {k: buffer(1, F32) for k in ("mean", "rstd")}
            params = {k: buffer(c, F32) for k in ("gw", "gb", "ggw", "ggb")}
            host = (ctypes.c_int64 * 1)(rows)
            need = lib.msda_group_norm_workspace_bytes(host, 1, rows, c, 1, 1, code[dtype], 1)
            need2 = lib.msda_dropout_add_norm_workspace_bytes(rows, c, code[dtype], code[dtype])
            work, work2 = (torch.full((k // 4 + 64,), 7.0, device="cuda") for k in (need, need2))
            p = lambda pair: pair[1].data_ptr()
            wsp, wsp2 = work[32:].data_ptr(), work2[32:].data_ptr()
            k = code[dtype]
            rcs = [
                lib.msda_dropout_forward(x.data_ptr(), p(bufs["drop"]), state.data_ptr(), n, 0.5, 0, 0, k, st),
                lib.msda_dropout_add_norm_forward(
                    x.data_ptr(), dy.data_ptr(), w.data_ptr(), b.data_ptr(), p(bufs["out"]), p(stats["mean"]),
                    p(stats["rstd"]), state.data_ptr(), rows, c, 0.5, 0, 1e-5, k, k, 0, st),
                lib.msda_dropout_add_norm_backward(
                    dy.data_ptr(), x.data_ptr(), dy.data_ptr(), w.data_ptr(), p(stats["mean"]), p(stats["rstd"]),
                    p(bufs["gx"]), p(bufs["gr"]), p(params["gw"]), p(params["gb"]), wsp2, need2,
                    state.data_ptr(), rows, c, 0.5, 0, k, k, 0, st),
                lib.msda_group_norm_forward(
                    x.data_ptr(), w.data_ptr(), b.data_ptr(), p(bufs["gn"]), p(gstats["mean"]), p(gstats["rstd"]),
                    wsp, need, host, 1, rows, c, 1, 1, 1, 1e-5, 2, k, 0, st),
                lib.msda_group_norm_backward(
                    dy.data_ptr(), x.data_ptr(), w.data_ptr(), b.data_ptr(), p(gstats["mean"]), p(gstats["rstd"]),
                    p(bufs["gnx"]), p(params["ggw"]), p(params["ggb"]), wsp, need, host, 1, rows, c, 1, 1, 1, 2,
                    k, 0, st),
            ]
            assert rcs == [0] * 5, rcs
            for whole, inner in (*bufs.values(), *stats.values(), *gstats.values(), *params.values()):
                assert (whole[:33] == 7).all() and (whole[33 + inner.numel() :] == 7).all(), (dtype, rows, c)
                assert not (inner == 7).any()
            for whole, count in ((work, need // 4), (work2, need2 // 4)):
                assert (whole[:32] == 7).all() and (whole[32 + count :] == 7).all()


def test_group_norm_beyond_32_bit_offsets():
    """More than 2^31 elements: the last sample alone gives the same bits."""
    n, s, c = 3, 1 << 18, 4096
    x = torch.empty(n, s, c, dtype=BF16, device="cuda")
    for i in range(n):
        x[i].normal_(generator=torch.Generator(device="cuda").manual_seed(i))
    w, b = torch.ones(c, device="cuda"), torch.zeros(c, device="cuda")
    y = level_group_norm(x, w, b, 32, activation="silu")
    # chunks differ with the batch, so the statistics may differ in the last bits of fp32: a step of bf16
    one = level_group_norm(x[2:], w, b, 32, activation="silu")
    assert ((y[2:].float() - one.float()).abs() <= 2.0**-7 * one.float().abs() + 1e-6).all()
    z = dropout_add_layer_norm(x.view(-1, c), x.view(-1, c), w, b, 0.5, rng(), 1)
    tail = x.view(-1, c)[-3:]
    f = ref.keep(x.numel() - 3 * c, 3 * c, 0.5, *STATE, 1)
    h = tail.float().cpu() * (1 + 2 * torch.from_numpy(f).view(3, c).float())
    want = torch.nn.functional.layer_norm(h, (c,))
    assert ((z[-3:].float().cpu() - want).abs() <= 2.0**-8 * want.abs() + 1e-4).all()


def test_gradients_beyond_32_bit_offsets():
    """The last rows of gradients of more than 2^31 elements have the bits of the rows alone."""
    c, rows = 4096, (1 << 19) + 64
    g = torch.Generator(device="cuda").manual_seed(1)
    tail = 64  # (a multiple of every team's step: the last rows fall into workgroups of their own)
    x = torch.empty(rows, c, dtype=BF16, device="cuda").normal_(generator=g)
    dy = torch.empty(rows, c, dtype=BF16, device="cuda").normal_(generator=g)
    w = torch.ones(c, device="cuda")
    op = torch.ops.unipercept
    _, mean, rstd = op.dropout_add_norm_fwd(x, x, w, w, None, 0.0, 0, 1e-5, True)
    gx, gr, gw, gb = op.dropout_add_norm_bwd(dy, x, x, w, mean, rstd, rng(), 0.5, 1, True, True, True)
    one = op.dropout_add_norm_bwd(
        dy[-tail:], x[-tail:], x[-tail:], w, mean[-tail:], rstd[-tail:], None, 0.0, 0, True, True, True)
    keep = torch.from_numpy(ref.keep((rows - tail) * c, tail * c, 0.5, *STATE, 1)).view(tail, c).cuda()
    assert torch.equal(gx[-tail:] != 0, keep & (gr[-tail:] != 0)) and torch.isfinite(gw).all()
    del gx, gr
    _, gr, _, _ = op.dropout_add_norm_bwd(dy, x, x, w, mean, rstd, None, 0.0, 0, False, True, False)
    assert torch.equal(gr[-tail:], one[1])
    want = dy.float().sum(0)
    assert (gb - want).norm() <= 1e-4 * want.norm()
    del gr, gb
    y = op.counter_dropout_fwd(x, rng(), 0.5, 2, "relu")
    gx = op.counter_dropout_bwd(dy, y, None, 0.5, 2, "relu")
    assert torch.equal(gx[-tail:], torch.where(y[-tail:] > 0, dy[-tail:] * 2, torch.zeros_like(dy[-tail:])))
    del y, gx
    # group norm: the last sample of several against the sample alone
    n = 4
    x, dy = x[: rows // n * n].view(n, rows // n, c), dy[: rows // n * n].view(n, rows // n, c)
    _, mean, rstd = op.level_group_norm_fwd(x, w, w, 32, [], 1e-5, "silu", True)
    gx, gw, gb = op.level_group_norm_bwd(dy, x, w, w, mean, rstd, 32, [], "silu", True, True)
    last = op.level_group_norm_bwd(dy[-1:], x[-1:], w, w, mean[-1:], rstd[-1:], 32, [], "silu", True, True)
    # (chunks differ with the batch: fp32 sums in another order, one step of bf16)
    assert ((gx[-1:].float() - last[0].float()).abs() <= 2.0**-7 * last[0].float().abs() + 1e-6).all()


def test_parameter_gradients_beyond_32_bit_offsets():
    """Sums over more than 2^31 elements against sums of blocks in fp64, from the forward's statistics.
    A workgroup adds up to 256 rows a thread and the rest is joined by lanes: fewer than 400 additions deep."""
    n, s, c, groups = 4, 1 << 17, 4112, 16
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.empty(n, s, c, dtype=BF16, device="cuda").normal_(generator=g)
    dy = torch.empty(n, s, c, dtype=BF16, device="cuda").normal_(generator=g)
    assert x.numel() > 2**31
    w = torch.ones(c, device="cuda").normal_(1.0, 0.3, generator=g)
    b = torch.zeros(c, device="cuda").normal_(0.0, 0.3, generator=g)
    op, r, depth = _lib.torch_ops(), 2.0**-24, 400

    def compare(name, got, terms):
        """terms(i, rows) -> the summands of (dw, db) for rows of sample i, and the error of a summand."""
        sums = [torch.zeros(c, dtype=F64, device="cuda") for _ in range(4)]
        for i in range(n):
            for at in range(0, s, 1 << 13):
                a, d, ea, ed = terms(i, slice(at, at + (1 << 13)))
                for total, part in zip(sums, (a, d, depth * r * a.abs() + ea, depth * r * d.abs() + ed)):
                    total += part.sum(0)
        for k, what in enumerate(("dw", "db")):
            check((name, what), got[k], sums[k].cpu(), sums[2 + k].cpu() + half_step(sums[k].cpu(), F32))

    _, mean, rstd = op.level_group_norm_fwd(x, w, b, groups, [], 1e-5, "silu", True)
    _, gw, gb = op.level_group_norm_bwd(dy, x, w, b, mean, rstd, groups, [], "silu", False, True)

    def group_terms(i, rows):
        mu, s_ = (t[i, 0].double().repeat_interleave(c // groups) for t in (mean, rstd))
        u, d = (x[i, rows].double() - mu) * s_, dy[i, rows].double()
        z = u * w.double() + b.double()
        sig = torch.sigmoid(z)
        dz = d * sig * (1 + z * (1 - sig))
        # the slope: its own roundings, and those of z (|slope'| <= 0.5)
        e = d.abs() * r * ((2 * z.abs() + 8) * (z.abs() + 1) + 0.5 * 5 * (u * w).abs() + 2 * b.abs()) + 2 * r * dz.abs()
        return dz * u, dz, e * u.abs() + 4 * r * (dz * u).abs(), e

    compare("group norm", (gw, gb), group_terms)
    flat = x.view(-1, c)
    _, mean, rstd = op.dropout_add_norm_fwd(flat, flat, w, b, None, 0.0, 0, 1e-5, True)
    _, _, gw, gb = op.dropout_add_norm_bwd(dy.view(-1, c), flat, flat, w, mean, rstd, None, 0.0, 0, False, False, True)

    def norm_terms(i, rows):
        at = slice(i * s + rows.start, i * s + rows.stop)
        u = (2 * flat[at].double() - mean[at, None].double()) * rstd[at, None].double()
        d = dy[i, rows].double()
        return d * u, d, 4 * r * (d * u).abs(), 0 * d

    compare("residual norm", (gw, gb), norm_terms)


@pytest.mark.parametrize("dtype,c,groups", [(BF16, 8192, 1), (F16, 8191, 1), (F32, 4096, 1), (F32, 4095, 3), (F64, 2047, 1),
                                            (BF16, 8192, 8192), (F32, 4096, 32)])
def test_group_norm_widest_rows(dtype, c, groups):
    PYRAMIDS["_widest"] = (2, [(3, 3), (1, 2)], c, groups)
    try:
        run_group("_widest", dtype, F64 if dtype == F64 else F32, "silu")
    finally:
        del PYRAMIDS["_widest"]


@pytest.mark.parametrize("dtype,c,groups,full", [
    (F32, 256, 1, 64), (F32, 256, 2, 128), (BF16, 256, 1, 128), (BF16, 256, 32, 1024), (F32, 256, 32, 1024),
    (F16, 64, 2, 1024), (F32, 48, 2, 340), (BF16, 96, 32, 340), (F32, 4, 1, 4096), (BF16, 8, 2, 4096)])
@pytest.mark.parametrize("extra", [0, 1])
def test_group_norm_full_workgroups(dtype, c, groups, full, extra):
    """Levels of as many rows as a workgroup of 1024 threads holds (four vectors a thread), and of one
    row more, beside a level of half and one of a single row."""
    PYRAMIDS["_full"] = (2, [(1, full + extra), (1, full // 2), (1, 1)], c, groups)
    try:
        run_group("_full", dtype, F32, "silu")
    finally:
        del PYRAMIDS["_full"]


def test_group_norm_many_samples():
    """More (sample, level) pairs than rows in each, through the one-launch and the general kernels."""
    for n, levels, c, groups in ((5000, [(1, 2), (1, 1)], 16, 4), (3000, [(1, 3)], 6, 3), (4000, [(4, 4)], 256, 32)):
        x = normal((n, sum(h * w for h, w in levels), c), F32, n)
        w, b = normal((len(levels), c), F32, 2), normal((len(levels), c), F32, 3)
        rows = [h * v for h, v in levels]
        want, _ = ref.group_norm(x, w, b, groups, rows, 1e-5, "none")
        got = level_group_norm(x.cuda(), w.cuda(), b.cuda(), groups, levels).cpu().double()
        # groups of a few elements: a step of fp32 in x - mean against spreads down to 1e-3
        assert ((got - want).abs() <= 2.0**-24 * 1e4 * (1 + want.abs())).all()


def test_no_memory_is_kept_between_steps():
    calls, _ = _calls()
    for call in calls.values():
        call()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for _ in range(5):
        for call in calls.values():
            call()
    torch.cuda.synchronize()
    # (the engine's thread lets go of the last call's gradients a moment after it has woken the caller)
    for _ in range(100):
        if torch.cuda.memory_allocated() == before:
            break
        time.sleep(0.01)
    assert torch.cuda.memory_allocated() == before


def test_inference_mode_and_detached_results():
    x, w, b = normal((2, 20, 64), F32, 1).cuda(), torch.ones(64, device="cuda"), torch.zeros(64, device="cuda")
    w.requires_grad_(True)
    want = [counter_dropout(x, 0.3, rng(), 0, "relu"), dropout_add_layer_norm(x, x, w, b, 0.3, rng()),
            level_group_norm(x, w, b, 8)]
    assert [t.requires_grad for t in want] == [False, True, True]
    for mode in (torch.inference_mode, torch.no_grad):
        with mode():
            got = [counter_dropout(x, 0.3, rng(), 0, "relu"), dropout_add_layer_norm(x, x, w, b, 0.3, rng()),
                   level_group_norm(x, w, b, 8)]
        assert all(torch.equal(a, c) for a, c in zip(got, want)) and not any(t.requires_grad for t in got)


def test_function_transforms_are_right_or_refused():
    """torch.func.grad either gives the gradient or raises: never a silent zero."""
    x = normal((4, 64), F32, 1).cuda()
    w, b = torch.ones(64, device="cuda"), torch.zeros(64, device="cuda")
    state = rng()
    for f in (lambda t: counter_dropout(t, 0.3, state, 0), lambda t: dropout_add_layer_norm(t, t, w, b),
              lambda t: level_group_norm(t[:, None], w, b, 8)):
        leaf = x.clone().requires_grad_(True)
        (want,) = torch.autograd.grad(f(leaf).square().sum(), leaf)
        try:
            got = torch.func.grad(lambda t: f(t).square().sum())(x)
        except RuntimeError:
            continue
        assert torch.equal(got, want)


def test_vmap_draws_the_masks_of_its_states():
    x = normal((3, 10, 24), F32, 1).cuda().requires_grad_(True)
    states = torch.stack([rng((k, 7 - k)) for k in range(3)])
    w, b = normal((24,), F32, 2).cuda(), normal((24,), F32, 3).cuda()
    dy = normal((3, 10, 24), F32, 4).cuda()
    for f in (lambda t, state: counter_dropout(t, 0.4, state, 1, "relu"),
              lambda t, state: dropout_add_layer_norm(t, t, w, b, 0.4, state, 2)):
        for mode, in_dims, state in (("different", (0, 0), states), ("error", (0, 0), states), ("same", (0, None), states[0])):
            got = torch.func.vmap(f, in_dims=in_dims, randomness=mode)(x, state)
            want = torch.stack([f(x[k], state if in_dims[1] is None else state[k]) for k in range(3)])
            assert torch.equal(got, want)
            assert torch.equal(*(torch.autograd.grad(t, x, dy)[0] for t in (got, want)))
        with pytest.raises(RuntimeError, match="same mask"):
            torch.func.vmap(lambda t: f(t, states[0]), randomness="different")(x)


def test_two_threads_at_once():
    """Calls of two host threads on streams of their own."""
    import threading

    calls, _ = _calls()
    want = {name: call() for name, call in calls.items()}
    torch.cuda.synchronize()
    results, errors = [], []

    def work():
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(10):
                    results.append({name: call() for name, call in calls.items()})
            stream.synchronize()
        except BaseException as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work) for _ in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors and len(results) == 20
    for got in results:
        for name in want:
            assert all(torch.equal(a, c) for a, c in zip(want[name], got[name])), name


# ---- the path they were made for ---------------------------------------------------------------------


def _layer_pair(dropout, **kw):
    torch.manual_seed(11)
    plain = MSDeformAttnEncoderLayer(64, 96, dropout, n_levels=2, n_heads=4, n_points=2, **kw).cuda()
    fused = MSDeformAttnEncoderLayer(64, 96, dropout, n_levels=2, n_heads=4, n_points=2, fused_epilogues=True, **kw).cuda()
    for p in plain.parameters():
        torch.nn.init.normal_(p, std=0.1)
    fused.load_state_dict(plain.state_dict())
    return plain, fused


def _layer_inputs():
    levels = [(8, 12), (4, 6)]
    shapes = torch.as_tensor(levels, device="cuda")
    lsi = torch.tensor([0, 96], device="cuda")
    src = normal((2, 120, 64), F32, 1).cuda()
    pos = normal((2, 120, 64), F32, 2).cuda()
    ref_points = torch.rand(2, 120, 2, 2, generator=torch.Generator().manual_seed(3)).cuda()
    dy = normal((2, 120, 64), F32, 4).cuda()
    return src, pos, ref_points, shapes, lsi, dy


def _train(layer, src, pos, ref_points, shapes, lsi, dy, **kw):
    layer.zero_grad()
    x = src.clone().requires_grad_(True)
    out = layer(x, pos, ref_points, shapes, lsi, **kw)
    out.backward(dy.to(out.dtype))
    return [out.detach(), x.grad] + [p.grad for p in layer.parameters()]


def _close(a, b, rel):
    for x, y in zip(a, b):
        assert x.dtype == y.dtype
        assert (x - y).float().norm() <= rel * y.float().norm() + 1e-6


def test_encoder_layer_without_dropout_equals_the_plain_layer():
    """The same sums in another order: fp32 noise of the GEMMs' size (2-norm 1e-4 after two norms)."""
    plain, fused = _layer_pair(0.0)
    inputs = _layer_inputs()
    _close(_train(fused, *inputs), _train(plain, *inputs), 1e-4)
    plain, fused = _layer_pair(0.3)
    plain.eval(), fused.eval()
    _close(_train(fused, *inputs), _train(plain, *inputs), 1e-4)


def test_encoder_layer_with_dropout_equals_the_masked_layer():
    """The plain layer with the oracle's masks in place of its dropout, forward and backward."""
    plain, fused = _layer_pair(0.3)
    inputs = _layer_inputs()
    sites = iter((10, 11, 12))

    class Masked(torch.nn.Module):
        def forward(self, x):
            f = ref.factor(tuple(x.shape), 0.3, STATE, next(sites))
            return x * f.to(x.device, x.dtype)

    plain.dropout = Masked()
    got = _train(fused, *inputs, rng_state=rng(), rng_site=10)
    _close(got, _train(plain, *inputs), 1e-4)


def test_encoder_layer_under_autocast():
    plain, fused = _layer_pair(0.0)
    inputs = _layer_inputs()
    with torch.autocast("cuda", torch.bfloat16):
        a, b = _train(fused, *inputs), _train(plain, *inputs)
    # both routes round the same tensors to bf16; sums kept in fp32 here may land on another side
    _close(a, b, 3e-2)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("stream", [F32, "same"])
def test_encoder_layer_with_16_bit_parameters_under_autocast(dtype, stream, monkeypatch):
    monkeypatch.setenv("MSDA_DETERMINISTIC", "1")  # the attention's gradients with the same bits every time
    plain, fused = (layer.to(dtype) for layer in _layer_pair(0.0))
    src, pos, ref_points, shapes, lsi, dy = _layer_inputs()
    if stream == "same":
        src, pos = src.to(dtype), pos.to(dtype)
    inputs = (src, pos, ref_points, shapes, lsi, dy)
    with torch.autocast("cuda", dtype):
        a, b = _train(fused, *inputs), _train(plain, *inputs)
    assert a[0].dtype == F32
    # The same values as fp32 parameters: every product runs in 16 bits and every norm in fp32 either way,
    # so the results agree to the bit but for the parameters' own rounding of their gradients.
    lifted = _layer_pair(0.0)[1]
    lifted.load_state_dict({k: v.float() for k, v in fused.state_dict().items()})
    with torch.autocast("cuda", dtype):
        c = _train(lifted, *inputs)
    assert all(torch.equal(x, y.to(x.dtype)) for x, y in zip(a, c))
    # Against the plain layer.  Both routes round the same tensors, and sums kept in fp32 may land a whole
    # step (eps of the value) apart at each; the longest path, to the gradient of the sampling offsets'
    # weight, has 14 of them (query, its projection, value, attention, output projection, linear1, linear2;
    # the gradients of linear2's output, hidden tensor, linear1's input, attention branch, output
    # projection's input, sampling points, weight).  The ReLU's input differs by up to 2.5 steps (the sum
    # that the plain route rounds, linear1's input, its output), which moves a share of 2.5 * 2 * eps *
    # (density 0.4 of a normal variable at 0) = 2 eps of the units over 0, where half of them are open:
    # sqrt(2 eps / 0.5) of the gradient's norm.
    eps = torch.finfo(dtype).eps
    _close(a[:1], b[:1], 14 * eps)
    _close(a, b, 14 * eps + 2 * eps**0.5)


def test_projection_and_encoder_train_together():
    """Input projections, then a stack with dropout: repeatable under one seed, new masks otherwise."""
    torch.manual_seed(5)
    proj = LevelInputProjection([24, 40], 64, 16, "relu").cuda()
    enc = MSDeformAttnEncoder(2, d_model=64, d_ffn=96, dropout=0.2, n_levels=2, n_heads=4, n_points=2,
                              fused_epilogues=True).cuda()
    maps = [normal((2, 24, 8, 12), F32, 1).cuda(), normal((2, 40, 4, 6), F32, 2).cuda()]

    def step(seed):
        torch.manual_seed(seed)
        params = [*proj.parameters(), *enc.parameters()]
        src, shapes, lsi, levels, pos = proj(maps, position_feats=32)
        out = enc(src, shapes, lsi, pos=pos, spatial_shapes_list=levels)
        return [out.detach(), *torch.autograd.grad(out.square().sum(), params)]

    first, again, other = step(1), step(1), step(2)
    assert torch.equal(first[0], again[0]) and not torch.equal(first[0], other[0])
    assert all(torch.isfinite(t).all() for t in first)
    # the projection against 1 x 1 convolutions and torch's group norm
    want = flatten_levels([
        torch.relu(torch.nn.functional.group_norm(
            torch.nn.functional.conv2d(m.double(), p.weight.double()[:, :, None, None], p.bias.double()), 16,
            proj.norm_weight[i].double(), proj.norm_bias[i].double()))
        for i, (m, p) in enumerate(zip(maps, proj.projections))])[0]
    got = proj(maps)[0]
    assert (got - want).abs().max() <= 1e-4
    with torch.no_grad():
        enc.eval()
        src, shapes, lsi, levels, pos = proj(maps, position_feats=32)
        assert torch.equal(enc(src, shapes, lsi, pos=pos, spatial_shapes_list=levels),
                           enc(src, shapes, lsi, pos=pos, spatial_shapes_list=levels))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_projection_under_autocast(dtype):
    """As a convolution and torch's group norm under autocast: 16-bit products, the norm's result and the
    position embeddings in fp32."""
    torch.manual_seed(7)
    proj = LevelInputProjection([24, 40], 64, 16, "relu").cuda()
    maps = [normal((2, 24, 8, 12), F32, 1).cuda(), normal((2, 40, 4, 6), F32, 2).cuda()]
    with torch.autocast("cuda", dtype):
        got, _, _, _, pos = proj(maps, position_feats=32)
        want = flatten_levels([
            torch.relu(torch.nn.functional.group_norm(
                torch.nn.functional.conv2d(m, p.weight[:, :, None, None], p.bias), 16,
                proj.norm_weight[i], proj.norm_bias[i]))
            for i, (m, p) in enumerate(zip(maps, proj.projections))])[0]
    assert got.dtype == want.dtype == pos.dtype == F32
    assert (got - want).norm() <= 3 * torch.finfo(dtype).eps * want.norm()
    # the norm's result is not rounded to 16 bits: most values lie between two of them
    assert (got.to(dtype).float() != got)[got > 0].double().mean() > 0.9
    (grad,) = torch.autograd.grad(got.square().sum(), proj.norm_weight)
    assert grad.dtype == F32 and torch.isfinite(grad).all()
    # 16-bit parameters: the bits of the same values in fp32
    proj.to(dtype)
    wide = LevelInputProjection([24, 40], 64, 16, "relu").cuda()
    wide.load_state_dict({k: v.float() for k, v in proj.state_dict().items()})
    with torch.autocast("cuda", dtype):
        assert torch.equal(proj(maps)[0], wide(maps)[0])
    assert torch.equal(pos, flatten_levels([m[:, :24] for m in maps], 32)[4])


def test_projection_gradients_match_convolutions():
    """Many tokens (the projections' weight gradients by slices), channels-last and plain maps:
    outputs and gradients against 1 x 1 convolutions and torch's group norm in fp64."""
    torch.manual_seed(6)
    proj = LevelInputProjection([24, 40], 64, 16, "silu").cuda()
    maps = [normal((2, 24, 128, 136), F32, 1).cuda().contiguous(memory_format=torch.channels_last),
            normal((2, 40, 31, 17), F32, 2).cuda()]
    dy = normal((2, 128 * 136 + 31 * 17, 64), F32, 3).cuda()
    params = [*proj.parameters()]
    leaves = [m.requires_grad_(True) for m in maps]
    got = torch.autograd.grad(proj(leaves)[0], [*params, *leaves], dy)
    twin = LevelInputProjection([24, 40], 64, 16).double().cuda()
    twin.load_state_dict(proj.state_dict())
    wide = [m.detach().double().requires_grad_(True) for m in maps]
    out = flatten_levels([
        torch.nn.functional.silu(torch.nn.functional.group_norm(
            torch.nn.functional.conv2d(m, p.weight[:, :, None, None], p.bias), 16, twin.norm_weight[i],
            twin.norm_bias[i]))
        for i, (m, p) in enumerate(zip(wide, twin.projections))])[0]
    want = torch.autograd.grad(out, [*twin.parameters(), *wide], dy.double())
    for a, b in zip(got, want):
        # fp32 GEMMs over up to 34816 tokens; a bias before a norm has a gradient of rounding alone
        assert (a - b).norm() <= 1e-4 * b.norm() + 1e-2


def test_masks_of_a_state_from_torchs_generator():
    a = new_rng_state("cuda", torch.Generator(device="cuda").manual_seed(3))
    b = new_rng_state("cuda", torch.Generator(device="cuda").manual_seed(3))
    assert torch.equal(a, b)
    x = torch.ones(1 << 20, device="cuda")
    y = counter_dropout(x, 0.1, a, 0)
    kept = (y != 0).double().mean().item()
    # five standard deviations of a binomial share
    assert abs(kept - (1 - round(6553.6) / 65536)) < 5 * (0.09 / (1 << 20)) ** 0.5


def test_compiled_graphs_hold_the_operators():
    """torch.compile (tracing only, eager kernels): forward and backward as in eager mode."""
    calls, state = _calls()
    w, b = torch.ones(64, device="cuda", requires_grad=True), torch.zeros(64, device="cuda", requires_grad=True)
    x, res = normal((2, 20, 64), F32, 1).cuda(), normal((2, 20, 64), F32, 2).cuda()

    def net(x, res, w, b, state):
        h = counter_dropout(x, 0.2, state, 1, "relu")
        h = dropout_add_layer_norm(h, res, w, b, 0.2, state, 2)
        return level_group_norm(h, w, b, 8, [(4, 4), (2, 2)], activation="silu")

    def grads(f):
        xs = x.clone().requires_grad_(True)
        out = f(xs, res, w, b, state)
        return [out.detach(), *torch.autograd.grad(out.square().sum(), (xs, w, b))]

    want = grads(net)
    for dynamic in (False, True):
        torch._dynamo.reset()
        got = grads(torch.compile(net, backend="aot_eager", fullgraph=True, dynamic=dynamic))
        for a, c in zip(got, want):
            assert torch.equal(a, c)
