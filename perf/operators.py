"""Measured cases of the operators around the attention of an encoder layer.

Three operators of ``unipercept_amd.deform_attn``:

* ``level_group_norm``: group normalisation of the flattened pyramid (N, S, C), every level on its
  own, with an activation (the input projections of a pixel decoder);
* ``counter_dropout``: dropout from a counter-based generator, after an optional ReLU (the hidden
  tensor of the feed-forward network);
* ``dropout_add_layer_norm``: ``LayerNorm(residual + dropout(x))`` (behind the attention and behind
  the feed-forward network).

``own`` chooses what ``run`` calls: the operators of the package, or their plain form below.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}

# position counts are heights x widths of a pyramid's levels, largest first
_CITYSCAPES = "128x256 64x128 32x64"  # 1024 x 2048 images, strides 8 / 16 / 32
_HALF_CITYSCAPES = "64x128 32x64 16x32"  # 512 x 1024 images
_COCO = "128x128 64x64 32x32 16x16"  # 1024 x 1024 images, strides 8 / 16 / 32 / 64


def _group_norm(name, batch, levels, channels, groups, act, dtype, param, train):
    return dict(
        name=name, op="group_norm", batch=batch, levels=levels, channels=channels, groups=groups,
        act=act, dtype=dtype, param=param, train=train,
    )


def _dropout(name, batch, tokens, channels, act, p, dtype, train):
    return dict(
        name=name, op="dropout", batch=batch, tokens=tokens, channels=channels, act=act, p=p,
        dtype=dtype, train=train,
    )


def _add_norm(name, batch, tokens, channels, p, dtype, residual, param, train):
    return dict(
        name=name, op="add_norm", batch=batch, tokens=tokens, channels=channels, p=p, dtype=dtype,
        residual=residual, param=param, train=train,
    )


def listed():
    return [
        # the coarsest level of one 512 x 1024 image, inference: latency counts
        _group_norm("gn_one_level_infer_bf16", 1, "16x32", 256, 32, "relu", "bf16", "bf16", False),
        # the three levels of one 512 x 1024 image, inference
        _group_norm("gn_pyramid_infer_bf16", 1, _HALF_CITYSCAPES, 256, 32, "relu", "bf16", "bf16", False),
        # training step of the input projections, Cityscapes crops, batch 8 of a GPU, fp32
        _group_norm("gn_cityscapes_train_f32", 8, _CITYSCAPES, 256, 32, "none", "f32", "f32", True),
        # the same for COCO crops in bf16 with fp32 parameters and a smooth activation, batch 16
        _group_norm("gn_coco_train_bf16", 16, _COCO, 256, 32, "silu", "bf16", "f32", True),
        # uneven maps and three channels a group, as images of any size and narrow models give
        _group_norm("gn_uneven_train_f16", 3, "51x77 26x39 13x20", 96, 32, "gelu", "f16", "f32", True),
        # training step of a short decoder-style sequence: latency counts
        _dropout("drop_queries_train_bf16", 2, 300, 256, "none", 0.1, "bf16", True),
        # odd everything, fp32
        _dropout("drop_odd_train_f32", 5, 21001, 129, "none", 0.25, "f32", True),
        # the hidden tensor of the feed-forward network, Cityscapes crops, batch 8: the largest
        _dropout("drop_hidden_train_bf16", 8, 43008, 1024, "relu", 0.1, "bf16", True),
        # training step behind the attention of a short decoder-style sequence: latency counts
        _add_norm("norm_queries_train_bf16", 2, 300, 256, 0.1, "bf16", "bf16", "bf16", True),
        # training step, Cityscapes crops, batch 8, fp32
        _add_norm("norm_cityscapes_train_f32", 8, 43008, 256, 0.1, "f32", "f32", "f32", True),
        # the same under autocast, COCO crops, batch 16: bf16 branch, fp32 residual stream
        _add_norm("norm_coco_autocast_train", 16, 21760, 256, 0.1, "bf16", "f32", "f32", True),
        # inference, odd token count and a width that no vector load divides
        _add_norm("norm_odd_infer_f16", 2, 10751, 515, 0.0, "f16", "f16", "f16", False),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("group_norm", "dropout", "add_norm"))
    dtype = rng.choice(("f32", "bf16", "f16"))
    train = rng.random() < 0.7
    limit = 80_000_000  # elements
    if op == "group_norm":
        groups = rng.choice((1, 4, 8, 16, 32))
        channels = groups * _spread(rng, 1 if groups > 1 else 4, min(32, 1024 // groups))
        h, w = _spread(rng, 3, 160), _spread(rng, 3, 256)
        levels = []
        for _ in range(rng.randint(1, 4)):
            levels.append((h, w))
            h, w = (h + 1) // 2, (w + 1) // 2
        positions = sum(a * b for a, b in levels)
        batch = _spread(rng, 1, 16)
        while batch > 1 and batch * positions * channels > limit:
            batch -= 1
        # training cases take smooth activations: a ReLU's gradient jumps at zero
        act = rng.choice(("none", "silu", "gelu") if train else ("none", "relu", "silu", "gelu"))
        text = " ".join("%dx%d" % level for level in levels)
        return _group_norm(None, batch, text, channels, groups, act, dtype, rng.choice((dtype, "f32")), train)
    channels = _spread(rng, 16, 2048)
    if rng.random() < 0.6:
        channels = (channels + 15) // 16 * 16
    batch = _spread(rng, 1, 16)
    tokens = max(1, min(_spread(rng, 1, 44000), limit // (batch * channels)))
    p = rng.choice((0.05, 0.1, 0.25, 0.5))
    if op == "dropout":
        return _dropout(None, batch, tokens, channels, rng.choice(("none", "relu")), p, dtype, train)
    residual = rng.choice((dtype, "f32"))
    param = "f32" if residual == "f32" else rng.choice((dtype, "f32"))
    return _add_norm(
        None, batch, tokens, channels, p if train else 0.0, dtype, residual, param, train
    )


def _shapes(case):
    return [tuple(int(v) for v in level.split("x")) for level in case["levels"].split()]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(shape, dtype, scale=1.0, shift=0.0):
        t = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
        return t.mul_(scale).add_(shift).to(_DTYPE[dtype])

    c = case["channels"]
    state = {"case": case}
    leaves = []
    if case["op"] == "group_norm":
        shapes = _shapes(case)
        positions = sum(h * w for h, w in shapes)
        x = torch.randn((case["batch"], positions, c), generator=g, device="cuda")
        # a projection's channels have means of their own
        x = x.mul_(1.5).add_(torch.randn((c,), generator=g, device="cuda")).to(_DTYPE[case["dtype"]])
        state["shapes"] = shapes
        state["weight"] = normal((len(shapes), c), case["param"], 0.1, 1.0)
        state["bias"] = normal((len(shapes), c), case["param"], 0.1)
        out_dtype = case["dtype"]
        leaves = ["x", "weight", "bias"]
    else:
        x = normal((case["batch"], case["tokens"], c), case["dtype"])
        state["rng_state"] = torch.randint(
            -(2**63), 2**63 - 1, (2,), generator=g, device="cuda", dtype=torch.int64
        )
        out_dtype = case["dtype"]
        leaves = ["x"]
        if case["op"] == "add_norm":
            state["residual"] = normal(tuple(x.shape), case["residual"])
            state["weight"] = normal((c,), case["param"], 0.1, 1.0)
            state["bias"] = normal((c,), case["param"], 0.1)
            out_dtype = case["residual"]
            leaves = ["x", "residual", "weight", "bias"]
    state["x"] = x
    if case["train"]:
        state["grad_out"] = normal(tuple(x.shape), out_dtype)
        for name in leaves:
            state[name].requires_grad_(True)
    state["leaves"] = leaves
    return state


# ---- the plain form ------------------------------------------------------------------------------

_M32 = 0xFFFFFFFF


def _random_bits(rng_state, site, numel):
    """16 random bits for each of `numel` elements: Philox4x32 with 7 rounds (Salmon, Moraes, Dror
    and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011).  Elements 8 j .. 8 j + 7 share
    the counter (j, site, offset low, offset high) under the key (seed low, seed high); element
    8 j + e takes the low (even e) or high half of word e // 2."""
    seed, offset = rng_state[0], rng_state[1]
    blocks = (numel + 7) // 8
    c0 = torch.arange(blocks, device=rng_state.device, dtype=torch.int64)
    c1 = torch.full_like(c0, site)
    c2 = (offset & _M32).expand_as(c0)
    c3 = ((offset >> 32) & _M32).expand_as(c0)
    k0, k1 = seed & _M32, (seed >> 32) & _M32
    for _ in range(7):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # 64 bits, wrapping
        c0, c1, c2, c3 = (
            ((p1 >> 32) & _M32) ^ c1 ^ k0, p1 & _M32, ((p0 >> 32) & _M32) ^ c3 ^ k1, p0 & _M32,
        )
        k0, k1 = (k0 + 0x9E3779B9) & _M32, (k1 + 0xBB67AE85) & _M32
    words = torch.stack((c0, c1, c2, c3), -1)
    return torch.stack((words & 0xFFFF, words >> 16), -1).reshape(-1)[:numel]


def _plain_dropout(x, p, rng_state, site):
    threshold = round(p * 65536)
    if threshold == 0:
        return x
    keep = _random_bits(rng_state, site, x.numel()).reshape(x.shape) >= threshold
    return torch.where(keep, x * (65536.0 / (65536 - threshold)), torch.zeros_like(x))


def _plain_activation(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _plain(state):
    case = state["case"]
    x = state["x"].float()
    if case["op"] == "group_norm":
        n, _, c = x.shape
        groups = case["groups"]
        parts, start = [], 0
        for level, (h, w) in enumerate(state["shapes"]):
            part = x[:, start : start + h * w].reshape(n, h * w, groups, c // groups)
            centred = part - part.mean((1, 3), keepdim=True)
            variance = (centred * centred).mean((1, 3), keepdim=True)
            z = (centred / torch.sqrt(variance + 1e-5)).reshape(n, h * w, c)
            z = z * state["weight"][level].float() + state["bias"][level].float()
            parts.append(_plain_activation(z, case["act"]))
            start += h * w
        return torch.cat(parts, 1).to(_DTYPE[case["dtype"]])
    if case["op"] == "dropout":
        y = _plain_activation(x, case["act"])
        return _plain_dropout(y, case["p"], state["rng_state"], 1).to(_DTYPE[case["dtype"]])
    h = state["residual"].float() + _plain_dropout(x, case["p"], state["rng_state"], 2)
    centred = h - h.mean(-1, keepdim=True)
    variance = (centred * centred).mean(-1, keepdim=True)
    z = centred / torch.sqrt(variance + 1e-5)
    z = z * state["weight"].float() + state["bias"].float()
    return z.to(_DTYPE[case["residual"]])


def _own(state):
    from unipercept_amd import deform_attn

    case = state["case"]
    if case["op"] == "group_norm":
        return deform_attn.level_group_norm(
            state["x"], state["weight"], state["bias"], case["groups"],
            spatial_shapes=state["shapes"], eps=1e-5, activation=case["act"],
        )
    if case["op"] == "dropout":
        return deform_attn.counter_dropout(
            state["x"], case["p"], state["rng_state"], site=1, activation=case["act"]
        )
    return deform_attn.dropout_add_layer_norm(
        state["x"], state["residual"], state["weight"], state["bias"], p=case["p"],
        rng_state=state["rng_state"], site=2, eps=1e-5,
    )


def run(state):
    forward = _own if own else _plain
    if not state["case"]["train"]:
        with torch.no_grad():
            return [forward(state)]
    out = forward(state)
    grads = torch.autograd.grad(out, [state[name] for name in state["leaves"]], state["grad_out"])
    return [out.detach(), *grads]


def work(case):
    size = _SIZE[case["dtype"]]
    c = case["channels"]
    if case["op"] == "group_norm":
        shapes = _shapes(case)
        elements = case["batch"] * sum(h * w for h, w in shapes) * c
        params = 2 * len(shapes) * c * _SIZE[case["param"]]
        moved, flops = 2 * elements * size + params, 8 * elements
        if case["train"]:  # the gradient comes in, those of x and of the parameters go out
            moved, flops = moved + 2 * elements * size + params, flops + 16 * elements
        return {"bytes": moved, "flops": flops}
    elements = case["batch"] * case["tokens"] * c
    if case["op"] == "dropout":
        passes = 2 if case["train"] else 1
        return {"bytes": passes * 2 * elements * size, "flops": passes * 2 * elements}
    stream = _SIZE[case["residual"]]
    params = 2 * c * _SIZE[case["param"]]
    moved, flops = elements * (size + 2 * stream) + params, 10 * elements
    if case["train"]:
        moved, flops = moved + elements * (size + 2 * stream) + params, flops + 18 * elements
    return {"bytes": moved, "flops": flops}


# ---- the definition in 64 bits -------------------------------------------------------------------


def _wide_product(a, m):
    """High and low 32 bits of a * m, by 16-bit halves (no product passes 2^33)."""
    al, ah, ml, mh = a & 0xFFFF, a >> 16, m & 0xFFFF, m >> 16
    ll, lh, hl, hh = al * ml, al * mh, ah * ml, ah * mh
    middle = (ll >> 16) + (lh & 0xFFFF) + (hl & 0xFFFF)
    return hh + (lh >> 16) + (hl >> 16) + (middle >> 16), ((middle & 0xFFFF) << 16) | (ll & 0xFFFF)


def _kept(state, site):
    """1 / (1 - p) where an element is kept and 0 where it is dropped, in 64 bits; None at p = 0."""
    case = state["case"]
    threshold = round(case["p"] * 65536)
    if threshold == 0:
        return None
    x = state["x"]
    seed, offset = (int(v) & (2**64 - 1) for v in state["rng_state"].tolist())
    blocks = -(-x.numel() // 8)
    a = torch.arange(blocks, device=x.device, dtype=torch.int64)
    b = torch.full_like(a, site)
    c = torch.full_like(a, offset % 2**32)
    d = torch.full_like(a, offset // 2**32)
    key = [seed % 2**32, seed // 2**32]
    for step in range(7):
        k0 = (key[0] + step * 0x9E3779B9) % 2**32
        k1 = (key[1] + step * 0xBB67AE85) % 2**32
        high_a, low_a = _wide_product(a, 0xD2511F53)
        high_c, low_c = _wide_product(c, 0xCD9E8D57)
        a, b, c, d = high_c ^ b ^ k0, low_c, high_a ^ d ^ k1, low_a
    kept = torch.empty((blocks, 8), device=x.device, dtype=torch.bool)
    for w, word in enumerate((a, b, c, d)):
        kept[:, 2 * w] = word % 65536 >= threshold
        kept[:, 2 * w + 1] = word // 65536 >= threshold
    return kept.flatten()[: x.numel()].view(x.shape).double() * (65536 / (65536 - threshold))


def _normal_parts(z):
    """Distribution function and density of the normal distribution."""
    return 0.5 * torch.special.erfc(-z / math.sqrt(2)), torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


def _exact_group_norm(case, state):
    x = state["x"].detach()
    n, _, c = x.shape
    g = case["groups"]
    out = torch.empty_like(x, dtype=torch.float64)
    weight, bias = state["weight"].detach().double(), state["bias"].detach().double()
    grads = None
    if case["train"]:
        grads = [torch.empty_like(out), torch.empty_like(weight), torch.empty_like(bias)]
    start = 0
    for level, (h, w) in enumerate(state["shapes"]):
        rows = slice(start, start + h * w)
        start += h * w
        part = x[:, rows].double().unflatten(2, (g, c // g))
        variance, mean = torch.var_mean(part, dim=(1, 3), correction=0, keepdim=True)
        scale = (variance + 1e-5) ** -0.5
        unit = (part - mean) * scale
        wl, bl = weight[level].view(g, c // g), bias[level].view(g, c // g)
        z = unit * wl + bl
        if case["act"] == "relu":
            y = z.clamp(min=0)
        elif case["act"] == "silu":
            s = torch.sigmoid(z)
            y, slope = z * s, s * (1 + z * (1 - s))
        elif case["act"] == "gelu":
            below, density = _normal_parts(z)
            y, slope = z * below, below + z * density
        else:
            y, slope = z, torch.ones_like(z)
        out[:, rows] = y.flatten(2)
        if grads is None:
            continue
        dz = state["grad_out"][:, rows].double().unflatten(2, (g, c // g)) * slope
        grads[1][level] = (dz * unit).sum((0, 1)).flatten()
        grads[2][level] = dz.sum((0, 1)).flatten()
        dunit = dz * wl
        along = dunit.mean((1, 3), keepdim=True)
        across = (dunit * unit).mean((1, 3), keepdim=True)
        grads[0][:, rows] = (scale * (dunit - along - unit * across)).flatten(2)
    return [out] if grads is None else [out, *grads]


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "group_norm":
            return _exact_group_norm(case, state)
        if case["op"] == "dropout":
            x = state["x"].detach()
            factor = _kept(state, 1)
            passed = (x > 0).double() if case["act"] == "relu" else 1.0
            slope = passed if factor is None else factor * passed
            out = [x.double() * slope]
            if case["train"]:
                out.append(state["grad_out"].double() * slope)
            return out
        factor = _kept(state, 2)
        x, residual = state["x"].detach().double(), state["residual"].detach().double()
        h = residual + (x if factor is None else x * factor)
        variance, mean = torch.var_mean(h, dim=-1, correction=0, keepdim=True)
        scale = (variance + 1e-5) ** -0.5
        unit = (h - mean) * scale
        weight, bias = state["weight"].detach().double(), state["bias"].detach().double()
        out = [unit * weight + bias]
        if case["train"]:
            dy = state["grad_out"].double()
            dunit = dy * weight
            dh = scale * (
                dunit - dunit.mean(-1, keepdim=True) - unit * (dunit * unit).mean(-1, keepdim=True)
            )
            out += [dh if factor is None else dh * factor, dh]
            out += [(dy * unit).sum((0, 1)), dy.sum((0, 1))]
        return out
