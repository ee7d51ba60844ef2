"""More operators on token sequences, as workloads: what the blocks of a picture or video transformer call besides attention.

A case is a dict of plain values.  `op` names the entry point (helpers of ops_cv_amd.aclnn):

    norm        layer_norm                 layer norm of x, or of x + residual, which comes back too
    norm_grad   layer_norm_backward        gradients of x (and of the residual, which is the same), weight and bias
    axes        rotary_axes                queries and keys turned by positions on several axes; inverse: the gradient's way
    dropout     dropout                    elements zeroed by a counter-based generator, and the residual's addition; without
                                           a residual it is also the gradient's way
    gated       gated_projection           act(x Wg^T + bg) * (x Wu^T + bu), with both factors' sums for training
    gated_grad  gated_projection_backward  gradients of x, of both weights and of both biases

With `own` false run() computes the same in elementary torch operations in 32 bits, rounded once at the end.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
EPS = 1e-5
ROTARY_BASE = 10000.0
LAYOUTS = ["consecutive", "restart", "dealt"]
ACTIVATIONS = ["silu", "gelu", "gelu_tanh"]

# no drawn case asks for more than the largest listed one
MOST_TENSOR = 10 ** 8  # bytes
MOST_WEIGHTS = 25 * 10 ** 7  # bytes
MOST_FLOPS = {"bf16": 9e11, "fp16": 9e11, "fp32": 5e10}


def _norm(name, op, dtype, rows, width, residual=True, bias=True, stats=False):
    return {"name": name, "op": op, "dtype": dtype, "rows": rows, "width": width, "residual": residual, "bias": bias,
            "stats": stats}


def _axes(name, dtype, b, extents, heads, kv_heads, d, sections, layout, interleaved=False, inverse=False):
    return {"name": name, "op": "axes", "dtype": dtype, "b": b, "extents": " ".join(map(str, extents)), "heads": heads,
            "kv_heads": kv_heads, "d": d, "sections": " ".join(map(str, sections)), "layout": layout,
            "interleaved": interleaved, "inverse": inverse}


def _dropout(name, dtype, rows, width, p, residual=True):
    return {"name": name, "op": "dropout", "dtype": dtype, "rows": rows, "width": width, "p": p, "residual": residual}


def _gated(name, op, dtype, rows, width, inner, activation, bias=False, sums=False):
    return {"name": name, "op": op, "dtype": dtype, "rows": rows, "width": width, "inner": inner, "activation": activation,
            "bias": bias, "sums": sums}


def listed():
    return [
        # eight sequences that grow by one token: the call whose cost is the call itself
        _norm("norm_token", "norm", "bf16", 8, 4096),
        # a vision encoder's layer: eight pictures of 37 x 37 patches
        _norm("norm_image", "norm", "fp16", 10952, 1280),
        # a training step's way back through a norm
        _norm("norm_train", "norm_grad", "bf16", 16384, 2048),
        # a clip of 8 x 32 x 32 patches on its way into attention
        _axes("axes_video", "bf16", 1, (8, 32, 32), 32, 8, 128, (16, 24, 24), "consecutive"),
        # gradients of the tokens of 37 x 37 patches in single precision, frequencies of its own for each axis
        _axes("axes_train", "fp32", 4, (37, 37), 16, 16, 80, (20, 20), "restart", interleaved=True, inverse=True),
        # a training step's tokens after a product, added to the residual stream
        _dropout("dropout_train", "bf16", 16384, 4096, 0.1),
        # the same gradient's way back in single precision, odd rows
        _dropout("dropout_odd", "fp32", 5477, 1283, 0.25, residual=False),
        # one new token of each of eight sequences
        _gated("gated_token", "gated", "bf16", 8, 4096, 14336, "silu"),
        # a prompt
        _gated("gated_prompt", "gated", "bf16", 4096, 4096, 14336, "silu"),
        # a vision encoder's layer in training, odd inner width
        _gated("gated_image", "gated", "fp16", 10952, 1280, 3413, "gelu", bias=True, sums=True),
        # a training step's way back
        _gated("gated_train", "gated_grad", "bf16", 4096, 2048, 8192, "silu"),
        # the same in single precision, odd sizes
        _gated("gated_train_odd", "gated_grad", "fp32", 777, 1001, 2731, "gelu_tanh", bias=True),
    ]


def _spread(rng, low, high):
    """A whole number of the range by its logarithm, odd or a power of two."""
    n = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(low, min(high, 1 << round(math.log2(n)) if rng.random() < 0.5 else int(n) | 1))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "axes", "dropout", "gated", "gated", "gated_grad", "gated_grad"])
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    if op.startswith("norm"):
        width = rng.choice([768, 1024, 1280, 2048, 4096, 5120, 8192, 2 * rng.randint(50, 700) + 1])
        rows = _spread(rng, 1, min(16384, MOST_TENSOR // BYTES[dtype] // width))
        c = _norm("", op, dtype, rows, width, rng.random() < 0.7, rng.random() < 0.7, op == "norm" and rng.random() < 0.5)
    elif op == "dropout":
        width = rng.choice([768, 1024, 1280, 2048, 4096, 2 * rng.randint(50, 700) + 1])
        c = _dropout("", dtype, _spread(rng, 1, min(16384, MOST_TENSOR // BYTES[dtype] // width)), width,
                     rng.choice([0.0, 0.05, 0.1, 0.2, 0.5, 0.9]), rng.random() < 0.6)
    elif op == "axes":
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 4])
        d = rng.choice([32, 64, 72, 80, 96, 128, 256])
        layout = rng.choice(LAYOUTS)
        turned = rng.choice([d, d, d // 2]) // 2
        axes = rng.choice([2, 3])
        first = turned // axes if layout == "restart" or rng.random() < 0.5 else turned // axes // 4 * 4
        sections = [turned - (axes - 1) * first] + [first] * (axes - 1)
        extents = [_spread(rng, 1, 16)] * (axes - 2) + [rng.randint(1, 48), rng.randint(1, 48)]
        tokens = math.prod(extents)
        b = _spread(rng, 1, max(1, min(64, MOST_TENSOR // (2 * BYTES[dtype]) // (tokens * heads * d))))
        c = _axes("", dtype, b, extents, heads, kv_heads, d, sections, layout, rng.random() < 0.5, rng.random() < 0.3)
    else:
        width = rng.choice([512, 1024, 1280, 2048, 4096, 2 * rng.randint(50, 700) + 1])
        inner = rng.choice([4 * width, 7 * width // 2, 8 * width // 3, 2 * rng.randint(200, 2000) + 1])
        each = 4 if op == "gated_grad" else 2  # weights and their gradients; products
        inner = min(inner, MOST_WEIGHTS // (each * BYTES[dtype] * width))
        rows = _spread(rng, 1, max(1, min(16384, int(MOST_FLOPS[dtype] / (2 * each * width * inner)),
                                          MOST_TENSOR // BYTES[dtype] // inner)))
        c = _gated("", op, dtype, rows, width, inner, rng.choice(ACTIVATIONS), rng.random() < 0.5,
                   op == "gated" and rng.random() < 0.5)
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------------- inputs

def _normal(g, *size, dtype, scale=1.0):
    return (torch.randn(*size, generator=g, device="cuda") * scale).to(dtype)


def _numbers(text):
    return [int(n) for n in text.split()]


def prepare(case, seed):
    c = dict(case)
    dtype = DTYPES[c["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(seed)
    if c["op"] in ("norm", "norm_grad"):
        rows, width = c["rows"], c["width"]
        c["weight"] = (1 + _normal(g, width, dtype=torch.float32, scale=0.1)).to(dtype)
        c["shift"] = _normal(g, width, dtype=dtype, scale=0.1) if c["bias"] else None
        x = _normal(g, rows, width, dtype=dtype)
        r = (0.5 + _normal(g, rows, width, dtype=torch.float32, scale=2.0)).to(dtype) if c["residual"] else None
        if c["op"] == "norm_grad":
            c["sum"] = x if r is None else x + r
            var, mean = torch.var_mean(c["sum"].float(), -1, correction=0)
            c["mean_in"], c["rstd_in"] = mean, torch.rsqrt(var + EPS)
            c["grad_y"] = _normal(g, rows, width, dtype=dtype, scale=0.01)
            c["grad_sum"] = _normal(g, rows, width, dtype=dtype, scale=0.01) if r is not None else None
        else:
            c["x"], c["r"] = x, r
    elif c["op"] == "axes":
        extents, c["parts"] = _numbers(c["extents"]), _numbers(c["sections"])
        tokens = math.prod(extents)
        c["q"] = _normal(g, c["b"], tokens, c["heads"], c["d"], dtype=dtype)
        c["k"] = _normal(g, c["b"], tokens, c["kv_heads"], c["d"], dtype=dtype)
        columns = max(c["parts"]) if c["layout"] == "restart" else sum(c["parts"])
        first = torch.randint(0, 64, (len(extents), c["b"], 1), generator=g, device="cuda")
        at = torch.stack([p.flatten() for p in torch.meshgrid(*[torch.arange(n, device="cuda") for n in extents], indexing="ij")])
        c["positions"] = first + at[:, None]
        turn = ROTARY_BASE ** (-torch.arange(columns, device="cuda", dtype=torch.float64) / columns)
        angle = torch.arange(64 + max(extents), device="cuda", dtype=torch.float64)[:, None] * turn
        c["angles"] = torch.cat([angle.cos(), angle.sin()], -1).float()
    elif c["op"] == "dropout":
        c["x"] = _normal(g, c["rows"], c["width"], dtype=dtype)
        c["r"] = _normal(g, c["rows"], c["width"], dtype=dtype, scale=2.0) if c["residual"] else None
        # key and offset of the generator: numbers of 64 bits
        c["state"] = torch.randint(-2 ** 63, 2 ** 63 - 1, (2,), generator=g, device="cuda")
    else:
        rows, width, inner = c["rows"], c["width"], c["inner"]
        c["x"] = _normal(g, rows, width, dtype=dtype)
        c["wg"] = _normal(g, inner, width, dtype=dtype, scale=width ** -0.5)
        c["wu"] = _normal(g, inner, width, dtype=dtype, scale=width ** -0.5)
        c["bg"] = _normal(g, inner, dtype=dtype, scale=0.1) if c["bias"] else None
        c["bu"] = _normal(g, inner, dtype=dtype, scale=0.1) if c["bias"] else None
        if c["op"] == "gated_grad":
            c["gate"], c["up"] = (t.to(dtype) for t in _plain_sums(c))
            c["grad_y"] = _normal(g, rows, inner, dtype=dtype, scale=0.01)
    return c


# ---------------------------------------------------------------------------------------------------- plain forms

def _plain_norm(s):
    h = s["x"].float() if s["r"] is None else s["x"].float() + s["r"].float()
    mean = h.mean(-1, keepdim=True)
    rstd = torch.rsqrt((h - mean).square().mean(-1, keepdim=True) + EPS)
    y = (h - mean) * rstd * s["weight"].float()
    if s["shift"] is not None:
        y = y + s["shift"].float()
    dtype = s["x"].dtype
    return (y.to(dtype), None if s["r"] is None else h.to(dtype), mean[:, 0] if s["stats"] else None,
            rstd[:, 0] if s["stats"] else None)


def _plain_norm_grad(s):
    rstd = s["rstd_in"][:, None]
    n = (s["sum"].float() - s["mean_in"][:, None]) * rstd
    gy = s["grad_y"].float()
    gn = gy * s["weight"].float()
    gx = (gn - gn.mean(-1, keepdim=True) - n * (gn * n).mean(-1, keepdim=True)) * rstd
    if s["grad_sum"] is not None:
        gx = gx + s["grad_sum"].float()
    dtype = s["sum"].dtype
    return gx.to(dtype), (gy * n).sum(0).to(dtype), gy.sum(0).to(dtype) if s["bias"] else None


def _axis_of_pairs(parts, layout):
    """The axis of every pair and its column in the table."""
    if layout == "dealt":  # one pair to each axis in turn, as long as it has any left
        axis = [a for turn in range(max(parts)) for a, n in enumerate(parts) if turn < n]
        return axis, list(range(len(axis)))
    axis = [a for a, n in enumerate(parts) for _ in range(n)]
    return axis, [i for n in parts for i in range(n)] if layout == "restart" else list(range(len(axis)))


def _plain_rotate(x, cos, sin, interleaved):
    rot = 2 * cos.shape[-1]
    x = x.float()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    p, q = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([p, q], -1).flatten(-2) if interleaved else torch.cat([p, q], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _plain_axes(s):
    axis, column = (torch.tensor(n, device="cuda") for n in _axis_of_pairs(s["parts"], s["layout"]))
    at = s["positions"].permute(1, 2, 0)[..., axis]  # (b, tokens, pairs)
    columns = s["angles"].shape[1] // 2
    cos, sin = s["angles"][at, column][:, :, None], s["angles"][at, columns + column][:, :, None]
    sin = -sin if s["inverse"] else sin
    return tuple(_plain_rotate(x, cos, sin, s["interleaved"]).to(x.dtype) for x in (s["q"], s["k"]))


def _plain_bits(state, n):
    """Numbers of 16 bits for elements 0 to n - 1: Philox 4x32 with ten rounds (Salmon, Moraes, Dror and Shaw, 2011) on the
    counter (element / 8, offset) under the key; an element's number is half a word, the low one first."""
    low = 0xffffffff
    at = torch.arange((n + 7) // 8, device="cuda")
    key, offset = state[0], state[1]
    c0, c1 = at, torch.zeros_like(at)
    c2, c3 = (offset & low).expand_as(at), ((offset >> 32) & low).expand_as(at)
    k0, k1 = key & low, (key >> 32) & low
    for _ in range(10):
        p, q = c0 * 0xd2511f53, c2 * 0xcd9e8d57
        c0, c1, c2, c3 = ((q >> 32) & low) ^ c1 ^ k0, q & low, ((p >> 32) & low) ^ c3 ^ k1, p & low
        k0, k1 = (k0 + 0x9e3779b9) & low, (k1 + 0xbb67ae85) & low
    words = torch.stack([c0, c1, c2, c3], -1)
    return torch.stack([words & 0xffff, words >> 16], -1).flatten()[:n]


def _plain_dropout(s):
    threshold = round(s["p"] * 65536)
    keep = (_plain_bits(s["state"], s["x"].numel()) >= threshold).view_as(s["x"])
    y = torch.where(keep, s["x"].float() * (65536 / (65536 - threshold)), 0.0)
    if s["r"] is not None:
        y = y + s["r"].float()
    return y.to(s["x"].dtype)


def _plain_sums(s):
    x = s["x"].float()
    gate, up = x @ s["wg"].float().t(), x @ s["wu"].float().t()
    return (gate, up) if s["bg"] is None else (gate + s["bg"].float(), up + s["bu"].float())


def _plain_activation(gate, kind):
    """The activation and its derivative."""
    if kind == "silu":
        s = 1 / (1 + torch.exp(-gate))
        return gate * s, s * (1 + gate * (1 - s))
    if kind == "gelu":
        below = 0.5 * torch.erfc(-gate * math.sqrt(0.5))
        return gate * below, below + gate * torch.exp(-0.5 * gate * gate) / math.sqrt(2 * math.pi)
    c, cubic = math.sqrt(2 / math.pi), 0.044715
    t = torch.tanh(c * (gate + cubic * gate ** 3))
    return 0.5 * gate * (1 + t), 0.5 * (1 + t) + 0.5 * gate * (1 - t * t) * c * (1 + 3 * cubic * gate * gate)


def _plain_gated(s):
    gate, up = _plain_sums(s)
    y, dtype = _plain_activation(gate, s["activation"])[0] * up, s["x"].dtype
    return (y.to(dtype), gate.to(dtype), up.to(dtype)) if s["sums"] else (y.to(dtype), None, None)


def _plain_gated_grad(s):
    act, slope = _plain_activation(s["gate"].float(), s["activation"])
    gy, x, dtype = s["grad_y"].float(), s["x"].float(), s["x"].dtype
    dg, du = gy * s["up"].float() * slope, gy * act
    gx = dg @ s["wg"].float() + du @ s["wu"].float()
    biases = (dg.sum(0).to(dtype), du.sum(0).to(dtype)) if s["bias"] else (None, None)
    return gx.to(dtype), (dg.t() @ x).to(dtype), (du.t() @ x).to(dtype), *biases


# ---------------------------------------------------------------------------------------------------- one pass

def run(state):
    s = state
    if not own:
        plain = {"norm": _plain_norm, "norm_grad": _plain_norm_grad, "axes": _plain_axes, "dropout": _plain_dropout,
                 "gated": _plain_gated, "gated_grad": _plain_gated_grad}
        return plain[s["op"]](s)
    from ops_cv_amd import aclnn
    if s["op"] == "norm":
        return aclnn.layer_norm(s["x"], s["weight"], s["shift"], residual=s["r"], eps=EPS, need_stats=s["stats"])
    if s["op"] == "norm_grad":
        return aclnn.layer_norm_backward(s["grad_y"], s["sum"], s["weight"], s["mean_in"], s["rstd_in"],
                                         grad_sum=s["grad_sum"], need_bias=s["bias"])
    if s["op"] == "axes":
        layout = {"consecutive": aclnn.AXES_CONSECUTIVE, "restart": aclnn.AXES_RESTART, "dealt": aclnn.AXES_DEALT}
        return aclnn.rotary_axes(s["q"], s["k"], s["angles"], s["positions"], s["parts"], layout=layout[s["layout"]],
                                 interleaved=s["interleaved"], inverse=s["inverse"])
    if s["op"] == "dropout":
        return aclnn.dropout(s["x"], s["state"], s["p"], residual=s["r"])
    kind = {"silu": aclnn.GATE_SILU, "gelu": aclnn.GATE_GELU, "gelu_tanh": aclnn.GATE_GELU_TANH}[s["activation"]]
    if s["op"] == "gated":
        return aclnn.gated_projection(s["x"], s["wg"], s["wu"], s["bg"], s["bu"], activation=kind, need_sums=s["sums"])
    return aclnn.gated_projection_backward(s["grad_y"], s["x"], s["wg"], s["wu"], s["gate"], s["up"], activation=kind,
                                           need_bias=s["bias"])


# ---------------------------------------------------------------------------------------------------- work

def work(case):
    c = case
    e = BYTES[c["dtype"]]
    if c["op"].startswith("norm"):
        n = c["rows"] * c["width"]
        if c["op"] == "norm_grad":  # grad_y, sum and, with a residual, grad_sum; the gradients; mean and rstd
            return {"bytes": n * e * (4 if c["residual"] else 3) + (3 if c["bias"] else 2) * c["width"] * e + 8 * c["rows"],
                    "flops": 12 * n}
        return {"bytes": n * e * (4 if c["residual"] else 2) + (2 if c["bias"] else 1) * c["width"] * e +
                (8 * c["rows"] if c["stats"] else 0), "flops": 7 * n}
    if c["op"] == "axes":
        extents, pairs = _numbers(c["extents"]), sum(_numbers(c["sections"]))
        tokens = c["b"] * math.prod(extents)
        n = tokens * (c["heads"] + c["kv_heads"])
        return {"bytes": 2 * n * c["d"] * e + 8 * tokens * len(extents) + 8 * pairs * (64 + max(extents)),
                "flops": 6 * n * pairs}
    if c["op"] == "dropout":
        n = c["rows"] * c["width"]
        return {"bytes": n * e * (3 if c["residual"] else 2), "flops": 2 * n}
    x, y, w = c["rows"] * c["width"], c["rows"] * c["inner"], c["width"] * c["inner"]
    biases = 2 * c["inner"] if c["bias"] else 0
    if c["op"] == "gated":  # two products
        return {"bytes": e * (x + 2 * w + biases + y * (3 if c["sums"] else 1)), "flops": 4 * c["rows"] * w}
    # four products; x, weights and their gradients; the outputs' gradient and both sums
    return {"bytes": e * (2 * x + 4 * w + biases + 3 * y), "flops": 8 * c["rows"] * w}


# ---------------------------------------------------------------------------------------------------- 64 bits

def _exact_norm(s):
    h = s["x"].double()
    if s["r"] is not None:
        h = h + s["r"].double()
    var, mean = torch.var_mean(h, 1, correction=0)
    root = (var + EPS).sqrt()
    y = torch.addcmul(s["shift"].double() if s["bias"] else torch.zeros((), dtype=torch.float64, device="cuda"),
                      (h - mean[:, None]) / root[:, None], s["weight"].double())
    return y, None if s["r"] is None else h, mean if s["stats"] else None, 1 / root if s["stats"] else None


def _exact_norm_grad(s):
    h, r = s["sum"].double() - s["mean_in"].double()[:, None], s["rstd_in"].double()[:, None]
    gy = s["grad_y"].double()
    g = gy * s["weight"].double()
    width = h.shape[1]
    gx = r * g - r * (g.sum(1, keepdim=True) / width) - r.pow(3) * h * ((g * h).sum(1, keepdim=True) / width)
    if s["grad_sum"] is not None:
        gx += s["grad_sum"].double()
    return gx, torch.einsum("ij,ij->j", gy, h * r), torch.einsum("ij->j", gy) if s["bias"] else None


def _exact_axes(s):
    """One pair at a time."""
    left, pairs = list(s["parts"]), []
    while any(left):  # (axis, column of the table) of every pair
        for a in range(len(left)):
            for _ in range(min(left[a], 1) if s["layout"] == "dealt" else left[a]):
                pairs.append((a, s["parts"][a] - left[a] if s["layout"] == "restart" else len(pairs)))
                left[a] -= 1
    half, columns = len(pairs), s["angles"].shape[1] // 2
    out = [x.double() for x in (s["q"], s["k"])]
    for i, (a, column) in enumerate(pairs):
        u, v = (2 * i, 2 * i + 1) if s["interleaved"] else (i, half + i)
        at = s["angles"].double()[s["positions"][a]]
        turn = torch.complex(at[..., column], at[..., columns + column])[..., None]
        turn = turn.conj() if s["inverse"] else turn
        for x in out:
            z = torch.complex(x[..., u].clone(), x[..., v].clone()) * turn
            x[..., u], x[..., v] = z.real, z.imag
    return tuple(out)


def _exact_dropout(s):
    """Products of 32 bits from halves of 16."""
    def product(a, m):
        lo, hi = a % 65536, a // 65536
        ml, mh = m % 65536, m // 65536
        mid = lo * mh + hi * ml + lo * ml // 65536
        return hi * mh + mid // 65536, (mid % 65536) * 65536 + lo * ml % 65536

    key, offset = (int(n) % 2 ** 64 for n in s["state"].tolist())
    n = s["x"].numel()
    words = [torch.arange(-(-n // 8), device="cuda")]
    words += [torch.full_like(words[0], v) for v in (0, offset % 2 ** 32, offset // 2 ** 32)]
    for turn in range(10):
        k = [(key % 2 ** 32 + turn * 0x9e3779b9) % 2 ** 32, (key // 2 ** 32 + turn * 0xbb67ae85) % 2 ** 32]
        (h0, l0), (h2, l2) = product(words[0], 0xd2511f53), product(words[2], 0xcd9e8d57)
        words = [h2 ^ words[1] ^ k[0], l2, h0 ^ words[3] ^ k[1], l0]
    halves = [v for w in words for v in (w % 65536, w // 65536)]
    bits = torch.stack(halves, 1).reshape(-1)[:n].reshape(s["x"].shape)
    dropped = math.floor(s["p"] * 65536 + 0.5)
    y = s["x"].double() * 65536 / (65536 - dropped) * (bits >= dropped)
    return y if s["r"] is None else y + s["r"].double()


def _exact_slope(gate, kind):
    with torch.enable_grad():
        g = gate.detach().requires_grad_()
        if kind == "silu":
            act = g * torch.sigmoid(g)
        elif kind == "gelu":
            act = g * torch.special.ndtr(g)
        else:
            act = g * torch.sigmoid(2 * math.sqrt(2 / math.pi) * g * (1 + 0.044715 * g * g))
        return act.detach(), torch.autograd.grad(act.sum(), g)[0]


def _exact_gated(s):
    x = s["x"].double()
    gate, up = x.matmul(s["wg"].double().T), x.matmul(s["wu"].double().T)
    if s["bias"]:
        gate, up = gate.add_(s["bg"].double()), up.add_(s["bu"].double())
    y = _exact_slope(gate, s["activation"])[0].mul_(up)
    return (y, gate, up) if s["sums"] else (y, None, None)


def _exact_gated_grad(s):
    act, slope = _exact_slope(s["gate"].double(), s["activation"])
    gy, x = s["grad_y"].double(), s["x"].double()
    both = torch.cat([slope.mul_(s["up"].double()).mul_(gy), act.mul_(gy)], 1)
    gx = both.matmul(torch.cat([s["wg"], s["wu"]]).double())
    gg, gu = both.T.matmul(x).chunk(2)
    biases = tuple(torch.ones(len(gy), dtype=torch.float64, device="cuda").matmul(both).chunk(2)) if s["bias"] else (None, None)
    return gx, gg, gu, *biases


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "norm_grad": _exact_norm_grad, "axes": _exact_axes, "dropout": _exact_dropout,
            "gated": _exact_gated, "gated_grad": _exact_gated_grad}[s["op"]](s)
