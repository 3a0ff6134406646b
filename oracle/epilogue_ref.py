"""TEST INFRASTRUCTURE: the operators around the attention in 64 bits, from their definitions.

Plain numpy / torch on the CPU; gradients are written out, not taken by autograd.
"""

from __future__ import annotations

import math

import numpy as np
import torch


def philox4x32(counter, key, rounds: int):
    """Salmon, Moraes, Dror, Shaw 2011, on uint64 arrays that hold 32-bit words."""
    m32 = np.uint64(0xFFFFFFFF)
    c = [np.asarray(v, dtype=np.uint64) for v in counter]
    k = [int(v) for v in key]
    for _ in range(rounds):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [
            (p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), p1 & m32,
            (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), p0 & m32,
        ]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def threshold(p: float) -> int:
    t = round(p * 65536)
    if 0 < p < 1:
        t = min(max(t, 1), 65535)
    return t


def keep(first: int, count: int, p: float, seed: int, offset: int, site: int) -> np.ndarray:
    """Keep bits of the elements [first, first + count)."""
    i = np.arange(first, first + count, dtype=np.uint64)
    blocks = i >> np.uint64(3)
    start = int(blocks[0]) if count else 0
    span = np.arange(start, (int(blocks[-1]) if count else -1) + 1, dtype=np.uint64)
    full = np.full_like(span, 1)
    words = philox4x32(
        (span, full * np.uint64(site), full * np.uint64(offset & 0xFFFFFFFF),
         full * np.uint64((offset >> 32) & 0xFFFFFFFF)),
        (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF), 7,
    )
    bits = np.stack([half for w in words for half in (w & np.uint64(0xFFFF), w >> np.uint64(16))], -1)
    return bits.reshape(-1)[first - 8 * start :][:count] >= np.uint64(threshold(p))


def factor(shape, p: float, rng_state, site: int) -> torch.Tensor:
    """1 / (1 - p) where an element is kept, 0 where it is dropped."""
    t = threshold(p) if p > 0 else 0
    if t == 0:
        return torch.ones(shape, dtype=torch.float64)
    if t == 65536:
        return torch.zeros(shape, dtype=torch.float64)
    count = math.prod(shape)
    k = keep(0, count, p, int(rng_state[0]), int(rng_state[1]), site)
    return torch.from_numpy(k.astype(np.float64)).reshape(shape) * (65536 / (65536 - t))


def _masked(x: torch.Tensor, f: torch.Tensor) -> torch.Tensor:
    return torch.where(f > 0, x * f, torch.zeros_like(x))


def dropout(x, p, rng_state, site, activation="none"):
    x = x.double()
    if activation == "relu":
        x = torch.where(x <= 0, torch.zeros_like(x), x)
    return _masked(x, factor(tuple(x.shape), p, rng_state, site))


def dropout_grad(grad, x, p, rng_state, site, activation="none"):
    g = _masked(grad.double(), factor(tuple(x.shape), p, rng_state, site))
    if activation == "relu":
        g = torch.where(x.double() <= 0, torch.zeros_like(g), g)
    return g


def add_norm(x, residual, weight, bias, p, rng_state, site, eps):
    """(out, parts) with parts for the gradient and for error bounds."""
    f = factor(tuple(x.shape), p, rng_state, site)
    h = residual.double() + _masked(x.double(), f)
    mean = h.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((h - mean) ** 2).mean(-1, keepdim=True) + eps)
    u = (h - mean) * rstd
    out = u * weight.double() + bias.double()
    size = residual.double().abs() + _masked(x.double(), f).abs()
    return out, {"f": f, "u": u, "mean": mean, "rstd": rstd, "size": size}


def add_norm_grad(grad, weight, parts):
    """(grad_x, grad_residual, grad_weight, grad_bias)"""
    dy, u = grad.double(), parts["u"]
    g = dy * weight.double()
    dh = parts["rstd"] * (g - g.mean(-1, keepdim=True) - u * (g * u).mean(-1, keepdim=True))
    c = u.shape[-1]
    return _masked(dh, parts["f"]), dh, (dy * u).reshape(-1, c).sum(0), dy.reshape(-1, c).sum(0)


def activate(z, activation):
    if activation == "relu":
        return torch.where(z <= 0, torch.zeros_like(z), z)
    if activation == "silu":
        return z / (1 + torch.exp(-z))
    if activation == "gelu":
        return 0.5 * z * torch.special.erfc(-z * math.sqrt(0.5))
    return z


def slope(z, activation):
    if activation == "relu":
        return (z > 0).double()
    if activation == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s + z * s * (1 - s)
    if activation == "gelu":
        return 0.5 * torch.special.erfc(-z * math.sqrt(0.5)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def group_norm(x, weight, bias, groups, rows, eps, activation):
    """x (N, S, C); (out, parts), parts one dict a level."""
    n, _, c = x.shape
    weight, bias = weight.double().expand(len(rows), c), bias.double().expand(len(rows), c)
    out, parts, start = [], [], 0
    for l, r in enumerate(rows):
        part = x[:, start : start + r].double().reshape(n, r, groups, c // groups)
        start += r
        mean = part.mean((1, 3), keepdim=True)
        rstd = 1 / torch.sqrt(((part - mean) ** 2).mean((1, 3), keepdim=True) + eps)
        u = ((part - mean) * rstd).reshape(n, r, c)
        z = u * weight[l] + bias[l]
        out.append(activate(z, activation))
        parts.append({
            "u": u, "z": z, "w": weight[l], "b": bias[l], "mean": mean.flatten(1), "groups": groups,
            "rstd": rstd.expand(n, 1, groups, c // groups).reshape(n, 1, c),
            "largest": part.abs().amax((1, 3), keepdim=True).expand(n, 1, groups, c // groups).reshape(n, 1, c),
        })
    return torch.cat(out, 1), parts


def group_mean(v, groups):
    """Mean over rows and the channels of a group, at every channel: (N, R, C) -> (N, 1, C)."""
    n, r, c = v.shape
    m = v.reshape(n, r, groups, c // groups).mean((1, 3), keepdim=True)
    return m.expand(n, 1, groups, c // groups).reshape(n, 1, c)


def group_norm_grad(grad, parts, activation):
    """(grad_x, grad_weight (L, C), grad_bias (L, C))"""
    gx, gw, gb, start = [], [], [], 0
    for q in parts:
        r = q["u"].shape[1]
        dz = grad[:, start : start + r].double() * slope(q["z"], activation)
        start += r
        wdz = dz * q["w"]
        m1, m2 = group_mean(wdz, q["groups"]), group_mean(wdz * q["u"], q["groups"])
        gx.append(q["rstd"] * (wdz - m1 - q["u"] * m2))
        gw.append((dz * q["u"]).sum((0, 1)))
        gb.append(dz.sum((0, 1)))
    return torch.cat(gx, 1), torch.stack(gw), torch.stack(gb)
