"""Plain implementations in 64 bits of the operators on token sequences, and bounds on how far a kernel may be from them.

U is a type's unit roundoff (half a step relative to 1), F32 a bound on what 32-bit sums and exponentials lose here: their
relative errors are a few 2^-24 per operation, and the sums of these tests have at most a few thousand terms in 32 or
more partial sums.
"""
import math

import numpy as np
import torch

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
U = {"fp32": 2.0 ** -24, "fp16": 2.0 ** -11, "bf16": 2.0 ** -8}
F32 = 1e-5
TINY = {"fp32": 1e-37, "fp16": 2.0 ** -25, "bf16": 1e-37}  # half the smallest step of the type, or less than any result


def within(got, want, bound, what):
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= bound) & ~((got == want) | (got.isnan() & want.isnan()))
    if bad.any():
        at = tuple(int(i) for i in bad.nonzero()[0])
        b = bound if not torch.is_tensor(bound) else bound.expand_as(want)[at].item()
        raise AssertionError("%s: %d of %d off, first at %s: %r, expected %r within %g" % (
            what, int(bad.sum()), bad.numel(), at, got[at].item(), want[at].item(), b))


# ------------------------------------------------------------------------------------------------------------- norm

def norm(x, residual, weight, eps):
    h = x.double() + (0 if residual is None else residual.double())
    rstd = 1 / torch.sqrt(h.square().mean(-1) + eps)
    return h * rstd[..., None] * weight.double(), h, rstd


def norm_int8(x, residual, weight):
    """The 8-bit numbers from the operator's definition: every step is one rounded 32-bit operation, so they are exact."""
    f = np.float32
    h = x.float().numpy() + (f(0) if residual is None else residual.float().numpy())
    t = h * weight.float().numpy()
    most = np.abs(t).max(-1, keepdims=True)
    with np.errstate(all="ignore"):
        step = np.where(most > 0, f(127) / most, f(0)).astype(f)
    return np.rint(t * step).astype(np.int8), most[..., 0]


def norm_grad(grad_y, grad_sum, h, weight, rstd):
    n = h.double() * rstd.double()[..., None]
    gn = grad_y.double() * weight.double()
    gx = (gn - n * (gn * n).mean(-1, keepdim=True)) * rstd.double()[..., None]
    if grad_sum is not None:
        gx = gx + grad_sum.double()
    return gx, (grad_y.double() * n).flatten(0, -2).sum(0)


# ----------------------------------------------------------------------------------------------------------- rotary

def rotary_table(positions, rot, base=10000.0, scaling=0, factor=1.0, original_length=0, magnitude=1.0):
    i = torch.arange(rot // 2, dtype=torch.float64)
    if scaling == 2:
        base = base * factor ** (rot / (rot - 2))
    f = base ** (-2 * i / rot)
    if scaling == 1:
        f = f / factor
    if scaling == 3:
        keep = ((original_length * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * f
    return torch.cat([angle.cos(), angle.sin()], -1) * magnitude


def rotary(x, table, positions, interleaved, inverse):
    rot = table.shape[1]
    half = rot // 2
    at = table.double()[positions]
    cos, sin = at[..., None, :half], at[..., None, half:]
    sin = -sin if inverse else sin
    x = x.double()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :half], x[..., half:rot])
    y = x.clone()
    p, q = a * cos - b * sin, b * cos + a * sin
    if interleaved:
        y[..., 0:rot:2], y[..., 1:rot:2] = p, q
    else:
        y[..., :half], y[..., half:rot] = p, q
    return y


def rotary_size(x, table, positions, interleaved):
    """|a cos| + |b sin| and |b cos| + |a sin| in the places of the results."""
    return rotary(x.abs(), table.abs(), positions, interleaved, False).maximum(
        rotary(x.abs(), table.abs(), positions, interleaved, True))


# -------------------------------------------------------------------------------------------------------- attention

def seen(sq, skv, left, right, sinks, q_len, kv_len):
    left, right = min(left, 2 ** 40), min(right, 2 ** 40)
    i = torch.arange(sq)[:, None]
    j = torch.arange(skv)[None]
    p = kv_len - q_len + i
    return (i < q_len) & (j < kv_len) & (j <= p + right) & ((j >= p - left) | (j < sinks))


def attention(q, k, v, scale, left, right, sinks, q_lens=None, kv_lens=None, grad_out=None):
    """Results of all sequences: out, lse, and with grad_out the gradients; "weights" and "scores_grad" (b, heads, sq, skv)
    for the bounds.  Keys and values that nobody sees are taken as zeros, whatever they hold."""
    b, sq, heads, d = q.shape
    skv, group = k.shape[1], heads // k.shape[2]
    r = {"out": torch.zeros(b, sq, heads, d, dtype=torch.float64),
         "lse": torch.full((b, heads, sq), -math.inf, dtype=torch.float64),
         "weights": torch.zeros(b, heads, sq, skv, dtype=torch.float64)}
    if grad_out is not None:
        r.update(gq=torch.zeros(q.shape, dtype=torch.float64), gk=torch.zeros(k.shape, dtype=torch.float64),
                 gv=torch.zeros(v.shape, dtype=torch.float64),
                 gs=torch.zeros(b, heads, sq, skv, dtype=torch.float64))
    for n in range(b):
        q_len = sq if q_lens is None else min(max(int(q_lens[n]), 0), sq)
        kv_len = skv if kv_lens is None else min(max(int(kv_lens[n]), 0), skv)
        see = seen(sq, skv, left, right, sinks, q_len, kv_len)
        rows, keys = see.any(1), see.any(0)
        for h in range(heads):
            kd = torch.where(keys[:, None], k[n, :, h // group].double(), 0)
            vd = torch.where(keys[:, None], v[n, :, h // group].double(), 0)
            qd = torch.where(rows[:, None], q[n, :, h].double(), 0)
            if skv == 0:
                continue
            s = (qd @ kd.T * scale).masked_fill(~see, -math.inf)
            r["lse"][n, h] = torch.logsumexp(s, 1)
            w = torch.where(rows[:, None], torch.softmax(s, 1), 0)
            r["weights"][n, h] = w
            r["out"][n, :, h] = w @ vd
            if grad_out is not None:
                go = torch.where(rows[:, None], grad_out[n, :, h].double(), 0)
                gw = go @ vd.T
                gs = w * (gw - (w * gw).sum(1, keepdim=True))
                r["gs"][n, h] = gs
                r["gq"][n, :, h] = gs @ kd * scale
                r["gk"][n, :, h // group] += gs.T @ qd * scale
                r["gv"][n, :, h // group] += w.T @ go
    return r


def attention_bounds(r, q, k, v, scale, dtype, grad_out=None):
    """How far out and the gradients may be.  The weights are rounded to the type before they meet the values (relative U,
    and in FLOAT16 absolute 2^-25 for the smallest), the gradients of the scores before they meet queries and keys; the
    rows' sums of grad_out times out carry out's rounding; results are rounded once more."""
    u, tiny = U[dtype], TINY[dtype]
    b, sq, heads, d = q.shape
    group = heads // k.shape[2]
    spread = lambda x: x.double().nan_to_num(0, 0, 0).abs().repeat_interleave(group, 2).transpose(1, 2)  # noqa: E731
    gather = lambda x: x.transpose(1, 2).unflatten(2, (k.shape[2], group)).sum(3)  # noqa: E731
    w = r["weights"]
    vs, ks, qs = spread(v), spread(k), q.double().nan_to_num(0, 0, 0).abs().transpose(1, 2)
    live = (w > 0).double()
    bounds = {"out": (w * (u + F32) + tiny * live) @ vs}
    bounds["out"] = bounds["out"].transpose(1, 2) + u * r["out"].abs() + tiny
    if grad_out is not None:
        go = grad_out.double().nan_to_num(0, 0, 0).abs().transpose(1, 2)
        o = r["out"].abs().transpose(1, 2)
        most = go.amax() if dtype == "fp16" else 1.0
        products = go @ vs.transpose(2, 3) + (go * o).sum(-1, keepdim=True)
        off = r["gs"].abs() * (u + F32) + w * products * F32 + w * (go * o).sum(-1, keepdim=True) * u
        off = off + tiny * most * live
        bounds["gq"] = (off @ ks * scale).transpose(1, 2) + u * r["gq"].abs() + tiny
        bounds["gk"] = gather(off.transpose(2, 3) @ qs) * scale + u * r["gk"].abs() + tiny
        bounds["gv"] = gather((w * (u + F32) + tiny * live).transpose(2, 3) @ go) + u * r["gv"].abs() + tiny
    return bounds
