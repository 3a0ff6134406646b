"""The operators around the attention where no GPU is needed: the oracle's generator against its
published vectors, the oracle's gradients against differences, argument checks of the Python surface
and of the C ABI (nothing is launched), shapes under torch's fake tensors."""

from __future__ import annotations

import ctypes

import numpy as np
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
from unipercept_amd.deform_attn import epilogue

FAKE = 0x1000  # never dereferenced: every call below fails validation first


# ---- the oracle itself ----------------------------------------------------------------------------


def test_generator_known_answers():
    """Vectors published with the generator (zeros; 10 rounds also with all bits set)."""
    z, f = 0, 0xFFFFFFFF
    assert [int(v) for v in ref.philox4x32((z,) * 4, (z,) * 2, 7)] == [
        0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48]
    assert [int(v) for v in ref.philox4x32((z,) * 4, (z,) * 2, 10)] == [
        0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert [int(v) for v in ref.philox4x32((f,) * 4, (f,) * 2, 10)] == [
        0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_keep_bits_statistics_and_windows():
    n, p = 1 << 16, 0.1
    k = ref.keep(0, n, p, -5, 3, 2)
    # 5 standard deviations of a binomial count
    assert abs(k.sum() - n * (1 - round(p * 65536) / 65536)) < 5 * (n * p * (1 - p)) ** 0.5
    assert np.array_equal(ref.keep(1003, 77, p, -5, 3, 2), k[1003:1080])
    for other in (ref.keep(0, n, p, -5, 3, 1), ref.keep(0, n, p, -5, 4, 2), ref.keep(0, n, p, -6, 3, 2)):
        agree = (other == k).mean()
        assert abs(agree - (p * p + (1 - p) ** 2)) < 0.01  # as independent masks do


@pytest.mark.parametrize("p,t", [(0.0, 0), (1e-9, 1), (0.1, 6554), (0.5, 32768), (1 - 1e-9, 65535), (1.0, 65536)])
def test_probability_steps(p, t):
    assert ref.threshold(p) == t


def _difference(f, x, d):
    h = 1e-6
    return ((f(x + h * d) - f(x - h * d)) / (2 * h)).item()


@pytest.mark.parametrize("activation", ["none", "relu", "silu", "gelu"])
def test_oracle_gradients_against_differences(activation):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 7, 6, generator=g, dtype=torch.float64)
    dy = torch.randn(2, 7, 6, generator=g, dtype=torch.float64)
    w = torch.randn(2, 6, generator=g, dtype=torch.float64)
    b = torch.randn(2, 6, generator=g, dtype=torch.float64)
    rows = [4, 3]

    def value(x, w, b):
        return (ref.group_norm(x, w, b, 3, rows, 1e-5, activation)[0] * dy).sum()

    grads = ref.group_norm_grad(dy, ref.group_norm(x, w, b, 3, rows, 1e-5, activation)[1], activation)
    for k, t in enumerate((x, w, b)):
        d = torch.randn(t.shape, generator=g, dtype=torch.float64)
        got = _difference(lambda v: value(*[v if i == k else a for i, a in enumerate((x, w, b))]), t, d)
        assert abs(got - (grads[k] * d).sum().item()) < 1e-6 * (1 + abs(got))
    if activation in ("silu", "gelu"):
        return
    state = (123456789, -7)
    got = _difference(lambda v: (ref.dropout(v, 0.3, state, 4, activation) * dy).sum(), x, dy)
    assert abs(got - (ref.dropout_grad(dy, x, 0.3, state, 4, activation) * dy).sum().item()) < 1e-6 * (1 + abs(got))
    if activation == "none":
        args = [x, x.flip(0).contiguous(), w[0], b[0]]

        def norm(args):
            return (ref.add_norm(*args, 0.3, state, 1, 1e-5)[0] * dy).sum()

        grads = ref.add_norm_grad(dy, w[0], ref.add_norm(*args, 0.3, state, 1, 1e-5)[1])
        for k, t in enumerate(args):
            d = torch.randn(t.shape, generator=g, dtype=torch.float64)
            got = _difference(lambda v: norm([v if i == k else a for i, a in enumerate(args)]), t, d)
            assert abs(got - (grads[k] * d).sum().item()) < 1e-6 * (1 + abs(got))


def test_normal_distribution_fit():
    """The constants of gn_phi, as fp32 holds them, against the complementary error function: the error
    that the kernel's comment states, without the kernel's own roundings."""
    import re
    from pathlib import Path

    from scipy.special import erfc

    source = (Path(_lib.__file__).parent / "csrc" / "msda_groupnorm.h").read_text()
    body = source[source.index("float gn_phi(float z, float& e)") :]
    body = body[: body.index("\n}")]
    step = float(np.float32(re.search(r"1\.f \+ ([0-9.]+)f \* a", body).group(1)))
    first = re.search(r"float r = (-?[0-9.]+)f;", body).group(1)
    rest = re.findall(r"r = r \* t ([+-]) ([0-9.]+)f;", body)
    coefficients = [float(np.float32(v)) for v in (first, *(sign + value for sign, value in rest))]
    assert len(coefficients) == 7
    a = np.linspace(0.0, 8.0, 400001)
    t = 1 / (1 + step * a)
    upper = np.polyval([*coefficients, 0.0], t) * np.exp(-0.5 * a * a)
    assert np.abs(upper - 0.5 * erfc(a * 0.5**0.5)).max() <= 8.4e-9


# ---- refusals of the Python surface -----------------------------------------------------------------


def meta(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta")


STATE = torch.empty(2, dtype=torch.int64, device="meta")


@pytest.mark.parametrize(
    "args,kw,exc",
    [
        ((torch.zeros(4), 0.1, torch.zeros(2, dtype=torch.int64)), {}, RuntimeError),  # CPU tensor
        ((meta(4, dtype=torch.int32), 0.1, STATE), {}, TypeError),
        ((meta(4), -0.1, STATE), {}, ValueError),
        ((meta(4), 1.1, STATE), {}, ValueError),
        ((meta(4), float("nan"), STATE), {}, ValueError),
        ((meta(4), 0.1), {}, ValueError),  # no state
        ((meta(4), 0.1, meta(3, dtype=torch.int64)), {}, ValueError),
        ((meta(4), 0.1, meta(2)), {}, ValueError),
        ((meta(4), 0.1, torch.zeros(2, dtype=torch.int64)), {}, RuntimeError),  # another device
        ((meta(4), 0.1, STATE), {"site": -1}, ValueError),
        ((meta(4), 0.1, STATE), {"site": 2**31}, ValueError),
        ((meta(4), 0.1, STATE), {"activation": "silu"}, ValueError),
        ((meta(2**18, 2**18, dtype=torch.bfloat16), 0.1, STATE), {}, ValueError),  # 2^36 elements
    ],
)
def test_dropout_refusals(args, kw, exc):
    with pytest.raises(exc):
        counter_dropout(*args, **kw)


def test_dropout_of_nothing_is_the_input():
    x = meta(4)
    assert counter_dropout(x, 0.0) is x


NORM = dict(x=meta(3, 8), residual=meta(3, 8), weight=meta(8), bias=meta(8))
BF = torch.bfloat16


@pytest.mark.parametrize(
    "change,exc",
    [
        (dict(x=torch.zeros(3, 8)), RuntimeError),
        (dict(residual=meta(3, 9)), ValueError),
        (dict(residual=meta(3, 8, dtype=BF)), TypeError),  # a residual narrower than x
        (dict(x=meta(3, 8, dtype=torch.float64)), TypeError),
        (dict(x=meta(3, 8, dtype=BF), residual=meta(3, 8, dtype=torch.float16)), TypeError),
        (dict(weight=meta(9), bias=meta(9)), ValueError),
        (dict(weight=meta(8, dtype=BF)), ValueError),  # weight and bias differ
        (dict(weight=meta(8, dtype=BF), bias=meta(8, dtype=BF)), TypeError),  # narrower than x
        (dict(weight=torch.zeros(8), bias=torch.zeros(8)), RuntimeError),
        (dict(eps=-1e-5), ValueError),
        (dict(eps=float("nan")), ValueError),
        (dict(p=0.1), ValueError),
        (dict(p=2.0, rng_state=STATE), ValueError),
        (dict(x=meta(2, 4100), residual=meta(2, 4100), weight=meta(4100), bias=meta(4100)), ValueError),
        (dict(x=meta(3, 0), residual=meta(3, 0), weight=meta(0), bias=meta(0)), ValueError),
        (dict(x=meta(), residual=meta()), ValueError),
    ],
)
def test_add_norm_refusals(change, exc):
    with pytest.raises(exc):
        dropout_add_layer_norm(**{**NORM, **change})


GROUP = dict(x=meta(2, 20, 8), weight=meta(8), bias=meta(8), num_groups=4)


@pytest.mark.parametrize(
    "change,exc",
    [
        (dict(x=torch.zeros(2, 20, 8)), RuntimeError),
        (dict(x=meta(8)), ValueError),
        (dict(num_groups=3), ValueError),
        (dict(num_groups=0), ValueError),
        (dict(spatial_shapes=[(4, 4)]), ValueError),  # 16 of 20 positions
        (dict(spatial_shapes=[(4, 4), (0, 9), (2, 2)]), ValueError),
        (dict(spatial_shapes=[(1, 1)] * 20), ValueError),  # more than 16 levels
        (dict(x=meta(2, 4, 5, 8), spatial_shapes=[(4, 5)]), ValueError),
        (dict(weight=meta(3, 8), bias=meta(3, 8), spatial_shapes=[(4, 4), (2, 2)]), ValueError),
        (dict(weight=meta(8, dtype=BF), bias=meta(8, dtype=BF)), TypeError),
        (dict(bias=meta(2, 8)), ValueError),
        (dict(activation="tanh"), ValueError),
        (dict(eps=-1.0), ValueError),
        (dict(x=meta(1, 2, 8200, dtype=BF), weight=meta(8200), bias=meta(8200)), ValueError),
        (dict(x=meta(2, 20, 8, dtype=torch.int64)), TypeError),
        (dict(x=meta(2**21 + 1, 1, 8)), ValueError),
        (dict(x=meta(2**20 + 1, 2, 8), spatial_shapes=[(1, 1), (1, 1)]), ValueError),
    ],
)
def test_group_norm_refusals(change, exc):
    with pytest.raises(exc):
        level_group_norm(**{**GROUP, **change})


def test_shapes_and_types_without_running():
    x = meta(2, 20, 8, dtype=BF)
    shapes = [(4, 4), (2, 2)]
    assert counter_dropout(x, 0.1, STATE).shape == x.shape
    y = level_group_norm(x, meta(2, 8), meta(2, 8), 4, shapes)
    assert y.shape == x.shape and y.dtype == BF
    z = dropout_add_layer_norm(x, meta(2, 20, 8), meta(8), meta(8))
    assert z.shape == x.shape and z.dtype == torch.float32
    out, mean, rstd = torch.ops.unipercept.level_group_norm_fwd(x, meta(8), meta(8), 4, [16, 4], 1e-5, "none", True)
    assert mean.shape == rstd.shape == (2, 2, 4) and mean.dtype == torch.float32
    gx, gr, gw, gb = torch.ops.unipercept.dropout_add_norm_bwd(
        z, x, z, meta(8), meta(40), meta(40), None, 0.0, 0, True, False, True)
    assert gx.dtype == BF and gr.numel() == 0 and gw.shape == gb.shape == (8,)
    assert new_rng_state("cpu").shape == (2,) and new_rng_state("cpu").dtype == torch.int64


def test_level_rows_come_from_lists_and_tensors():
    assert epilogue.level_rows([(4, 4), (2, 2)]) == [16, 4]
    assert epilogue.level_rows(torch.tensor([[4, 4], [2, 2]])) == [16, 4]
    assert level_group_norm(meta(2, 4, 5, 8), meta(8), meta(8), 4).shape == (2, 4, 5, 8)
    assert level_group_norm(meta(2, 8), meta(8), meta(8), 4).shape == (2, 8)
    with pytest.raises(ValueError):
        level_group_norm(meta(2, 4, 8), meta(8), meta(8), 4, [])


def test_gradients_have_shapes_without_running():
    """The operators' graphs on the meta device: types and shapes of every gradient."""
    x = meta(2, 20, 8, dtype=BF).requires_grad_(True)
    res, w, b = (t.requires_grad_(True) for t in (meta(2, 20, 8), meta(8), meta(8)))
    y = dropout_add_layer_norm(counter_dropout(x, 0.1, STATE, 1, "relu"), res, w, b, 0.1, STATE)
    y = level_group_norm(y, w, b, 4, [(4, 4), (2, 2)], activation="gelu")
    grads = torch.autograd.grad(y, (x, res, w, b), torch.empty_like(y))
    assert [g.dtype for g in grads] == [BF, torch.float32, torch.float32, torch.float32]
    assert [g.shape for g in grads] == [t.shape for t in (x, res, w, b)]


def _calls_by_input():
    """(operator, input) -> a function of that input alone, on the meta device."""
    big, one = (2, 20, 8), (8,)
    drop = lambda x, act: counter_dropout(x, 0.0 if act == "relu" else 0.1, STATE, 1, act)
    norm = lambda **kw: dropout_add_layer_norm(
        **{**dict(x=meta(*big), residual=meta(*big), weight=meta(*one), bias=meta(*one)), **kw})
    group = lambda **kw: level_group_norm(
        **{**dict(x=meta(*big), weight=meta(*one), bias=meta(*one), num_groups=4), **kw})
    calls = {("dropout", act): (big, lambda t, act=act: drop(t, act)) for act in ("none", "relu")}
    for name in ("x", "residual", "weight", "bias"):
        shape = big if name in ("x", "residual") else one
        calls["norm", name] = (shape, lambda t, name=name: norm(**{name: t}))
        if name != "residual":
            calls["group", name] = (shape, lambda t, name=name: group(**{name: t}))
    return calls


@pytest.mark.parametrize("call", sorted(_calls_by_input()))
def test_forward_mode_derivatives_are_refused(call):
    """A tangent on any input raises, whether or not the input requires a gradient as well: an output
    without a tangent would count as a derivative of zero."""
    from torch.autograd import forward_ad

    shape, f = _calls_by_input()[call]
    for requires_grad in (False, True):
        with forward_ad.dual_level():
            t = forward_ad.make_dual(meta(*shape).requires_grad_(requires_grad), meta(*shape))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f(t)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                f(t)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(f, (meta(*shape),), (meta(*shape),))
    # without a tangent, inside a dual level, everything runs
    with forward_ad.dual_level():
        f(meta(*shape))


@pytest.mark.parametrize("call", sorted(_calls_by_input()))
def test_a_tangent_of_the_incoming_gradient_is_refused(call):
    from torch.autograd import forward_ad

    shape, f = _calls_by_input()[call]
    t = meta(*shape).requires_grad_(True)
    y = f(t)
    with forward_ad.dual_level():
        dy = forward_ad.make_dual(meta(*y.shape), meta(*y.shape))
        for create_graph in (False, True):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(y, t, dy, retain_graph=True, create_graph=create_graph)
    assert torch.autograd.grad(y, t, meta(*y.shape))[0].shape == shape


def test_dropout_of_nothing_keeps_its_tangent():
    from torch.autograd import forward_ad

    with forward_ad.dual_level():
        t = forward_ad.make_dual(meta(4), meta(4))
        assert forward_ad.unpack_dual(counter_dropout(t, 0.0)).tangent is not None


@pytest.mark.parametrize("name", ["dropout", "norm"])
def test_vmap_does_not_repeat_a_mask_unasked(name):
    """Samples of a vmap count their elements from 0 each: refused unless the caller asks for equal
    masks or maps the states with the samples."""
    w = meta(8)
    f = {"dropout": lambda x, state, p=0.1: counter_dropout(x, p, state, 1, "relu"),
         "norm": lambda x, state, p=0.1: dropout_add_layer_norm(x, x, w, w, p, state)}[name]
    x, states = meta(3, 5, 8), meta(3, 2, dtype=torch.int64)
    vmap = torch.func.vmap
    for mode in ("error", "different"):
        refused = "randomness error mode" if mode == "error" else "same mask"
        with pytest.raises(RuntimeError, match=refused):
            vmap(lambda t: f(t, STATE), randomness=mode)(x)
        assert vmap(f, randomness=mode)(x, states).shape == x.shape
        assert vmap(lambda t: f(t, STATE, 0.0), randomness=mode)(x).shape == x.shape
        # an outer map without states of its own
        with pytest.raises(RuntimeError, match=refused):
            vmap(lambda a: vmap(f, randomness=mode)(a, states), randomness=mode)(meta(4, 3, 5, 8))
        both = vmap(vmap(f, randomness=mode), randomness=mode)
        assert both(meta(4, 3, 5, 8), meta(4, 3, 2, dtype=torch.int64)).shape == (4, 3, 5, 8)
    assert vmap(lambda t: f(t, STATE), randomness="same")(x).shape == x.shape
    outer = meta(3, 5, 8).requires_grad_(True)
    y = vmap(lambda t: f(t, STATE), randomness="same")(outer)
    assert torch.autograd.grad(y, outer, meta(3, 5, 8))[0].shape == x.shape
    # gradients of a batch of incoming gradients: one forward, one mask
    leaf = meta(5, 8).requires_grad_(True)
    y = f(leaf, STATE)
    assert torch.autograd.grad(y, leaf, meta(3, 5, 8), is_grads_batched=True)[0].shape == (3, 5, 8)


def test_torch_operators_are_built_and_loud_when_missing(monkeypatch, tmp_path):
    assert _lib.torch_ops() is torch.ops.unipercept
    monkeypatch.setattr(_lib, "_torch_ops", None)
    monkeypatch.setattr(_lib, "TORCH_LIB_PATH", tmp_path / "libmsda_torch.so")
    with pytest.raises(_lib.MsdaLibraryError):
        counter_dropout(meta(4), 0.1, STATE)


def test_packaging_builds_the_same_torch_operators():
    import importlib.util
    from pathlib import Path

    import __graft_entry__ as entry

    root = Path(entry.__file__).resolve().parent
    spec = importlib.util.spec_from_file_location("_setup_under_test", root / "setup.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    out = root / "unipercept_amd" / "libmsda_torch.so"
    assert mod.torch_ops_command(out) == entry.torch_ops_command(out)
    assert entry.build_torch_ops() == out


def _packaging(tmp_path, **env):
    """`setup.py build_hip` in a copy of the sources, the compilers replaced by scripts that write their
    output file."""
    import os
    import shutil
    import subprocess
    import sys
    from pathlib import Path

    import __graft_entry__ as entry

    root, tree = Path(entry.__file__).resolve().parent, tmp_path / "tree"
    if not tree.exists():
        for part in ("unipercept_amd/csrc", "unipercept_amd/torch_ops", "include"):
            shutil.copytree(root / part, tree / part)
        for part in ("setup.py", "pyproject.toml", "README.md", "unipercept_amd/__init__.py"):
            shutil.copy(root / part, tree / part)
    compiler = tmp_path / "compiler"
    compiler.write_text(
        "#!/bin/bash\nwhile [ $# -gt 1 ]; do [ \"$1\" = -o ] && echo built >> \"$2\"; shift; done\n")
    compiler.chmod(0o755)
    done = subprocess.run(
        [sys.executable, "setup.py", "build_hip"], cwd=tree, capture_output=True, text=True, timeout=120,
        env={**os.environ, "HIPCC": str(compiler), "CXX": str(compiler), **env})
    return tree / "unipercept_amd", done


def test_packaging_without_torch_leaves_out_its_operators_alone(tmp_path):
    """A build environment of its own (pip's isolation) holds no torch: the C library is built as ever."""
    block = tmp_path / "block"
    block.mkdir()
    (block / "torch.py").write_text("raise ModuleNotFoundError(\"No module named 'torch'\", name='torch')\n")
    package, done = _packaging(tmp_path, PYTHONPATH=str(block))
    assert done.returncode == 0, done.stderr
    assert (package / "libmsda.so").exists() and not (package / "libmsda_torch.so").exists()
    assert "--no-build-isolation" in done.stderr


def test_packaging_compiles_the_torch_operators_for_the_torch_at_hand(tmp_path):
    """Whatever is there may be another torch's: file times do not tell."""
    package, done = _packaging(tmp_path)
    assert done.returncode == 0, done.stderr
    first = (package / "libmsda_torch.so").read_text(), (package / "libmsda.so").read_text()
    package, done = _packaging(tmp_path)
    assert done.returncode == 0, done.stderr
    assert first == ("built\n", "built\n")
    assert (package / "libmsda_torch.so").read_text() == "built\nbuilt\n"
    assert (package / "libmsda.so").read_text() == "built\n"


# ---- argument errors of the C ABI -------------------------------------------------------------------


def test_abi_dropout_errors():
    lib = _lib.load()

    def fwd(x=FAKE, out=FAKE, state=FAKE, numel=8, p=0.1, site=0, act=0, dtype=0):
        return lib.msda_dropout_forward(x, out, state, numel, p, site, act, dtype, None)

    def bwd(g=FAKE, out=FAKE, gx=FAKE, state=FAKE, numel=8, p=0.1, site=0, act=1, dtype=0):
        return lib.msda_dropout_backward(g, out, gx, state, numel, p, site, act, dtype, None)

    assert fwd(x=None) == -1 and fwd(out=None) == -1 and fwd(state=None) == -1
    assert bwd(g=None) == -1 and bwd(gx=None) == -1 and bwd(out=None) == -1
    assert bwd(act=0, state=None) == -1
    assert fwd(numel=0) == -2 and fwd(p=-0.1) == -2 and fwd(p=1.5) == -2 and fwd(p=float("nan")) == -2
    assert fwd(site=-1) == -2 and fwd(numel=(1 << 35) + 1) == -2
    assert fwd(dtype=9) == -3 and fwd(act=2) == -3 and bwd(act=3) == -3 and bwd(dtype=-1) == -3
    assert fwd(x=FAKE + 2) == -4 and fwd(state=FAKE + 4) == -4 and bwd(gx=FAKE + 1, dtype=2) == -4


def test_abi_add_norm_errors():
    lib = _lib.load()
    need = lib.msda_dropout_add_norm_workspace_bytes

    def fwd(x=FAKE, res=FAKE, w=FAKE, b=FAKE, out=FAKE, mean=FAKE, rstd=FAKE, state=FAKE, rows=4, c=8,
            p=0.1, site=0, eps=1e-5, dx=0, dr=0, dp=0):
        return lib.msda_dropout_add_norm_forward(
            x, res, w, b, out, mean, rstd, state, rows, c, p, site, eps, dx, dr, dp, None)

    def bwd(g=FAKE, x=FAKE, res=FAKE, w=FAKE, mean=FAKE, rstd=FAKE, gx=FAKE, gr=FAKE, gw=FAKE, gb=FAKE,
            ws=FAKE, nbytes=1 << 20, state=FAKE, rows=4, c=8, p=0.1, site=0, dx=0, dr=0, dp=0):
        return lib.msda_dropout_add_norm_backward(
            g, x, res, w, mean, rstd, gx, gr, gw, gb, ws, nbytes, state, rows, c, p, site, dx, dr, dp, None)

    for name in ("x", "res", "w", "b", "out", "state"):
        assert fwd(**{name: None}) == -1
    assert fwd(mean=None) == -1 and fwd(rstd=None) == -1  # both or neither
    for name in ("g", "x", "res", "w", "mean", "rstd", "state"):
        assert bwd(**{name: None}) == -1
    assert bwd(gw=None) == -1 and bwd(gb=None) == -1
    for call in (fwd, bwd):
        assert call(rows=0) == -2 and call(c=0) == -2 and call(rows=1 << 31) == -2 and call(c=4097) == -2
        assert call(p=1.01) == -2 and call(site=-3) == -2
        assert call(dx=9) == -3 and call(dx=0, dr=2) == -3 and call(dx=2, dr=3, dp=3) == -3
        assert call(dx=2, dr=0, dp=2) == -3 and call(dx=1, dr=1, dp=0) == -3
        assert call(x=FAKE + 2) == -4 and call(rstd=FAKE + 2) == -4 and call(state=FAKE + 4) == -4
        assert call(dx=1, dr=1, dp=1, c=2049) == -2  # 16 KiB of the residual's type
    assert fwd(eps=-1.0) == -2 and fwd(eps=float("nan")) == -2
    assert bwd(ws=None) == -5 and bwd(ws=FAKE + 4) == -5 and bwd(nbytes=need(4, 8, 0, 0) - 1) == -5
    # two sums per column and workgroup (512 threads take 32 rows of 256 fp32 columns), and 16 rows
    # of them for the second step where there are many workgroups
    assert need(4, 8, 0, 0) == 2 * 8 * 4 and need(10**6, 256, 2, 0) == (31250 + 16) * 2 * 256 * 4
    assert need(4, 8, 1, 1) == 2 * 8 * 8 and need(0, 8, 0, 0) == 0 and need(4, 8, 0, 2) == 0


def test_abi_group_norm_errors():
    lib = _lib.load()
    need = lib.msda_group_norm_workspace_bytes

    def host(rows):
        return (ctypes.c_int64 * len(rows))(*rows)

    def fwd(x=FAKE, w=FAKE, b=FAKE, out=FAKE, mean=FAKE, rstd=FAKE, ws=FAKE, nbytes=1 << 24, rows=(16, 4),
            n=2, s=20, c=8, g=4, l=2, pl=1, eps=1e-5, act=0, dtype=0, dp=0):
        return lib.msda_group_norm_forward(
            x, w, b, out, mean, rstd, ws, nbytes, rows and host(rows), n, s, c, g, l, pl, eps, act, dtype, dp, None)

    def bwd(gy=FAKE, x=FAKE, w=FAKE, b=FAKE, mean=FAKE, rstd=FAKE, gx=FAKE, gw=FAKE, gb=FAKE, ws=FAKE,
            nbytes=1 << 24, rows=(16, 4), n=2, s=20, c=8, g=4, l=2, pl=1, act=0, dtype=0, dp=0):
        return lib.msda_group_norm_backward(
            gy, x, w, b, mean, rstd, gx, gw, gb, ws, nbytes, rows and host(rows), n, s, c, g, l, pl, act,
            dtype, dp, None)

    for name in ("x", "w", "b", "out", "mean", "rstd", "rows"):
        assert fwd(**{name: None}) == -1
    for name in ("gy", "x", "w", "b", "mean", "rstd", "gw", "gb", "rows"):
        assert bwd(**{name: None}) == -1
    for call in (fwd, bwd):
        assert call(n=0) == -2 and call(s=0) == -2 and call(c=0) == -2 and call(g=0) == -2 and call(l=0) == -2
        assert call(g=3) == -2 and call(pl=3) == -2 and call(pl=0) == -2
        assert call(rows=(16, 5)) == -2 and call(rows=(21, -1)) == -2 and call(rows=(20, 0)) == -2
        assert call(rows=(1,) * 17, l=17, s=17) == -7
        assert call(c=4100) == -2 and call(n=1 << 30) == -2 and call(n=(1 << 20) + 1) == -2
        assert call(dtype=9) == -3 and call(act=4) == -3 and call(act=-1) == -3 and call(dp=2) == -3
        assert call(dtype=1, dp=0) == -3 and call(dtype=2, dp=3) == -3
        assert call(x=FAKE + 2) == -4 and call(mean=FAKE + 2) == -4
        assert call(ws=None) == -5 and call(ws=FAKE + 4) == -5 and call(nbytes=0) == -5
    assert fwd(eps=float("nan")) == -2
    rows = host((16, 4))
    assert need(rows, 2, 20, 8, 4, 2, 0, 0) > 0 and need(rows, 2, 20, 8, 4, 2, 0, 1) > need(rows, 2, 20, 8, 4, 2, 0, 0)
    assert need(rows, 2, 21, 8, 4, 2, 0, 0) == 0 and need(None, 2, 20, 8, 4, 2, 0, 0) == 0


# ---- the modules --------------------------------------------------------------------------------------


def test_encoder_layers_keep_their_parameters_and_default_route():
    plain = MSDeformAttnEncoderLayer(32, 48, 0.1, n_levels=2, n_heads=4, n_points=2)
    fused = MSDeformAttnEncoderLayer(32, 48, 0.1, n_levels=2, n_heads=4, n_points=2, fused_epilogues=True)
    assert not plain.fused_epilogues
    fused.load_state_dict(plain.state_dict())
    enc = MSDeformAttnEncoder(2, d_model=32, d_ffn=48, n_levels=2, n_heads=4, n_points=2, fused_epilogues=True)
    assert all(layer.fused_epilogues for layer in enc.layers)


def test_encoder_passes_its_old_arguments_to_foreign_layers():
    """Layers put in place of the stack's own are called with the arguments they always were."""

    class Foreign(torch.nn.Module):
        def forward(self, src, pos, ref, shapes, lsi, mask):
            return src + 1

    enc = MSDeformAttnEncoder(1, d_model=16, d_ffn=32, n_levels=1, n_heads=2, n_points=2)
    enc.layers[0] = Foreign()
    src, shapes, lsi, levels, _ = flatten_levels([torch.zeros(1, 16, 2, 3)])
    assert torch.equal(enc(src, shapes, lsi, spatial_shapes_list=levels), src + 1)

def _watched(monkeypatch):
    """The fused route's operators replaced by recorders: (p, whether a state was given) of every call."""
    from unipercept_amd.deform_attn import encoder

    seen = []

    def norm(x, residual, weight, bias, p=0.0, rng_state=None, site=0, eps=1e-5):
        seen.append((p, rng_state is not None))
        return residual

    def drop(x, p, rng_state=None, site=0, activation="none"):
        seen.append((p, rng_state is not None))
        return x

    monkeypatch.setattr(encoder, "dropout_add_layer_norm", norm)
    monkeypatch.setattr(encoder, "counter_dropout", drop)
    return seen


@pytest.mark.parametrize("layer_trains", [False, True])
@pytest.mark.parametrize("dropout_trains", [False, True])
def test_fused_dropout_obeys_the_dropout_module(monkeypatch, layer_trains, dropout_trains):
    """As in the plain route the mode of the dropout module decides, not that of the layer: frozen dropout
    in a training layer, dropout that stays active in a layer that evaluates."""
    seen = _watched(monkeypatch)
    enc = MSDeformAttnEncoder(2, d_model=16, d_ffn=32, dropout=0.25, n_levels=1, n_heads=2, n_points=2,
                              fused_epilogues=True)
    src, shapes, lsi, levels, _ = flatten_levels([torch.zeros(1, 16, 2, 3)])
    for layer in enc.layers:
        layer.train(layer_trains)
        layer.dropout.train(dropout_trains)
        layer.self_attn.forward = lambda query, *args: query
    want = (0.25, True) if dropout_trains else (0.0, False)
    enc(src, shapes, lsi, spatial_shapes_list=levels)
    assert seen == [want] * 6
    seen.clear()
    enc.layers[0]._fused_rest(src, src, None, 0)  # a state of its own where one is needed
    assert seen == [want] * 3


def test_fused_route_takes_no_dropout_it_does_not_know(monkeypatch):
    seen = _watched(monkeypatch)
    layer = MSDeformAttnEncoderLayer(16, 32, 0.25, n_levels=1, n_heads=2, n_points=2, fused_epilogues=True)
    src = torch.zeros(1, 6, 16)
    layer.dropout = torch.nn.Identity()
    layer._fused_rest(src, src, None, 0)
    assert seen == [(0.0, False)] * 3
    for other in (torch.nn.AlphaDropout(0.25), torch.nn.ReLU()):
        layer.dropout = other
        with pytest.raises(TypeError, match="nn.Dropout"):
            layer._fused_rest(src, src, None, 0)


def test_fused_routes_refuse_cpu_tensors():
    src, shapes, lsi, levels, _ = flatten_levels([torch.zeros(1, 16, 2, 3)])
    layer = MSDeformAttnEncoderLayer(16, 32, 0.0, n_levels=1, n_heads=2, n_points=2, fused_epilogues=True)
    with pytest.raises(RuntimeError, match="only on a ROCm GPU"):
        layer._fused_rest(src, src, None, 0)
    with pytest.raises(RuntimeError, match="only on a ROCm GPU"):
        LevelInputProjection([16], 16, 4)([torch.zeros(1, 16, 2, 3)])


def test_input_projection_checks():
    with pytest.raises(ValueError, match="divisible"):
        LevelInputProjection([16], 20, 8)
    with pytest.raises(ValueError, match="levels"):
        LevelInputProjection([16, 32], 16, 4)([torch.zeros(1, 16, 2, 3)])


def test_input_projection_takes_the_weights_of_convolutions_and_norms():
    """The conversion that the documentation gives, from a state dict of (Conv2d, GroupNorm) pairs."""
    nn = torch.nn
    pairs = nn.ModuleList(nn.Sequential(nn.Conv2d(c, 16, 1), nn.GroupNorm(4, 16)) for c in (8, 24))
    sd, levels = pairs.state_dict(), 2
    proj = LevelInputProjection([8, 24], 16, 4)
    proj.load_state_dict({
        **{f"projections.{l}.weight": sd[f"{l}.0.weight"].flatten(1) for l in range(levels)},
        **{f"projections.{l}.bias": sd[f"{l}.0.bias"] for l in range(levels)},
        "norm_weight": torch.stack([sd[f"{l}.1.weight"] for l in range(levels)]),
        "norm_bias": torch.stack([sd[f"{l}.1.bias"] for l in range(levels)]),
    })
    assert torch.equal(proj.projections[1].weight, pairs[1][0].weight[:, :, 0, 0])
    assert torch.equal(proj.norm_bias[1], pairs[1][1].bias)
