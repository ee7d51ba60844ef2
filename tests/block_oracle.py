"""Plain implementations in 64 bits of layer norm, rotary positions on several axes, dropout and gated projections.

Bounds are made of token_oracle's U (a rounding to the type) and F32 (what 32-bit functions and short sums lose), and of
gamma(n) for sums of n products in 32 bits in any order: n + 8 roundings of 2^-24 at most, times the sum of the products'
absolute values.
"""
import math

import numpy as np
import torch

from token_oracle import DTYPES, F32, TINY, U, within  # noqa: F401


def gamma(n):
    return (n + 8) * 2.0 ** -24


# -------------------------------------------------------------------------------------------------------- layer norm

def layer_norm(x, residual, weight, bias, eps):
    """(y, h, mean, rstd, bound on y without its rounding)."""
    h = x.double() + (0 if residual is None else residual.double())
    mean = h.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((h - mean).square().mean(-1, keepdim=True) + eps)
    n = (h - mean) * rstd
    w = torch.ones(h.shape[-1], dtype=torch.float64) if weight is None else weight.double()
    b = torch.zeros(h.shape[-1], dtype=torch.float64) if bias is None else bias.double()
    size = h.abs().mean(-1, keepdim=True)
    # h and its mean are rounded in 32 bits before they are subtracted: that much of their size, against the spread
    off = F32 * ((1 + size * rstd) * n.abs() + (h.abs() + size) * rstd) * w.abs() + F32 * b.abs()
    return n * w + b, h, mean[..., 0], rstd[..., 0], off


def layer_norm_grad(grad_y, grad_sum, h, weight, mean, rstd):
    """((gx, gw, gb), bounds on them without their rounding)."""
    r = rstd.double()[..., None]
    n, gy = (h.double() - mean.double()[..., None]) * r, grad_y.double()
    w = torch.ones(h.shape[-1], dtype=torch.float64) if weight is None else weight.double()
    g = gy * w
    gx = (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True)) * r
    s = torch.zeros_like(gx) if grad_sum is None else grad_sum.double()
    big = (h.double().abs() + mean.double().abs()[..., None]) * r  # of n, before its subtraction
    off = F32 * ((g.abs() + g.abs().mean(-1, keepdim=True) + big * (g.abs() * big).mean(-1, keepdim=True)) * r + s.abs())
    rows = (gy * n).flatten(0, -2), gy.flatten(0, -2)
    sums = tuple(t.sum(0) for t in rows)
    return (gx + s, *sums), (off, (F32 + gamma(len(rows[0]) / 8)) * (gy.abs() * big).flatten(0, -2).sum(0),
                             (F32 + gamma(len(rows[0]) / 8)) * gy.abs().flatten(0, -2).sum(0))


# ------------------------------------------------------------------------------------------------------- rotary axes

def pairs_of(sections, layout):
    """(axis, column) of every pair."""
    left, out = list(sections), []
    while any(left):
        for a, n in enumerate(left):
            for _ in range(min(n, 1) if layout == 2 else n):
                out.append((a, sections[a] - left[a] if layout == 1 else len(out)))
                left[a] -= 1
    return out


def rotary_axes(x, table, positions, sections, layout, interleaved, inverse):
    """(result, bound without its rounding)."""
    pairs, y, off = pairs_of(sections, layout), x.double().clone(), torch.zeros(x.shape, dtype=torch.float64)
    columns = table.shape[1] // 2
    for i, (axis, column) in enumerate(pairs):
        u, v = (2 * i, 2 * i + 1) if interleaved else (i, len(pairs) + i)
        at = positions[axis].long()
        inside = (at >= 0) & (at < len(table))
        row = table.double()[at.clamp(0, max(0, len(table) - 1))]
        cos = torch.where(inside, row[..., column], math.nan)[..., None]
        sin = torch.where(inside, row[..., columns + column], math.nan)[..., None] * (-1 if inverse else 1)
        a, b = x.double()[..., u], x.double()[..., v]
        y[..., u], y[..., v] = a * cos - b * sin, b * cos + a * sin
        off[..., u] = off[..., v] = 2.0 ** -22 * (a.abs() + b.abs())
    return y, off


# ----------------------------------------------------------------------------------------------------------- dropout

def philox(counter, offset, seed):
    """Words of Philox 4x32-10 for an array of 64-bit counters: (n, 4) uint32."""
    low = np.uint64(0xffffffff)
    c = np.asarray(counter, dtype=np.uint64)
    word = [c & low, c >> np.uint64(32), np.full_like(c, offset & 0xffffffff), np.full_like(c, (offset >> 32) & 0xffffffff)]
    key = [seed & 0xffffffff, (seed >> 32) & 0xffffffff]
    for _ in range(10):
        p, q = word[0] * np.uint64(0xd2511f53), word[2] * np.uint64(0xcd9e8d57)
        word = [(q >> np.uint64(32)) ^ word[1] ^ np.uint64(key[0]), q & low,
                (p >> np.uint64(32)) ^ word[3] ^ np.uint64(key[1]), p & low]
        key = [(key[0] + 0x9e3779b9) & 0xffffffff, (key[1] + 0xbb67ae85) & 0xffffffff]
    return np.stack(word, -1).astype(np.uint32)


def numbers(n, seed, offset):
    words = philox(np.arange((n + 7) // 8), offset % 2 ** 64, seed % 2 ** 64)
    return np.stack([words & 0xffff, words >> 16], -1).reshape(-1)[:n]


def dropout(x, residual, state, p):
    """Every step is one rounded 32-bit operation, so the result is exact."""
    threshold = int(np.rint(p * 65536))
    keep = torch.from_numpy((numbers(x.numel(), *state) >= threshold).reshape(tuple(x.shape)))
    scale = np.float32(65536 / (65536 - threshold)) if threshold < 65536 else np.float32(0)
    y = torch.where(keep, x.float() * float(scale), torch.zeros((), dtype=torch.float32))
    return (y if residual is None else y + residual.float()).to(x.dtype), keep


# ------------------------------------------------------------------------------------------------- gated projections

def activation(g, kind):
    """Value and derivative."""
    if kind == 0:
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if kind == 1:
        below = torch.special.ndtr(g)
        return g * below, below + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g ** 3))
    return g * (1 + t) / 2, (1 + t) / 2 + g * (1 - t * t) / 2 * c * (1 + 3 * 0.044715 * g * g)


def gated(x, wg, wu, bg, bu, kind):
    """((y, gate, up), bounds on them without their rounding)."""
    def product(w, b):
        s, size = x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t()
        if b is not None:
            s, size = s + b.double(), size + b.double().abs()
        return s, gamma(x.shape[-1]) * size
    (gate, eg), (up, eu) = product(wg, bg), product(wu, bu)
    act = activation(gate, kind)[0]
    # slopes are under 1.2; the activations' 32-bit functions lose F32 of the gate at most
    ea = 1.2 * eg + F32 * gate.abs()
    return (act * up, gate, up), (ea * up.abs() + act.abs() * eu + ea * eu + F32 * (act * up).abs(), eg, eu)


def gated_grad(grad_y, x, wg, wu, gate, up, kind, dtype):
    """((gx, gwg, gwu, gbg, gbu), bounds on them without their rounding): dGate and dUp are rounded to the type before the
    products, FLOAT16 no finer than 2^-25 of 2^-14 of the largest of a row or column."""
    rows = x.flatten(0, -2).double()
    gy, g, u = (t.flatten(0, -2).double() for t in (grad_y, gate, up))
    act, slope = activation(g, kind)
    dg, du = gy * u * slope, gy * act
    # what the functions lose, before the rounding
    eg, eu = F32 * (gy * u).abs() * (1 + g.abs()), F32 * gy.abs() * g.abs()
    half = 0 if dtype == "fp32" else U[dtype]
    both, off = torch.cat([dg, du], 1), torch.cat([eg, eu], 1)
    coarse = both.abs().max() * 2.0 ** -39 if dtype == "fp16" and both.numel() else 0.0
    w = torch.cat([wg, wu]).double()
    gx, ex = both @ w, (off + (half + gamma(2 * g.shape[1])) * both.abs() + coarse) @ w.abs()
    gw = both.t() @ rows
    ew = (off + (half + gamma(len(rows))) * both.abs() + coarse).t() @ rows.abs()
    gb, eb = both.sum(0), (off + gamma(len(rows)) * both.abs()).sum(0)
    n = g.shape[1]
    return (gx.view(x.shape), gw[:n], gw[n:], gb[:n], gb[n:]), (ex.view(x.shape), ew[:n], ew[n:], eb[:n], eb[n:])
