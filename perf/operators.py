"""The operators on token sequences, as workloads: what a transformer block on image tokens, and the language model that
reads those tokens, calls around its matrix products.

A case is a dict of plain values.  `op` names the entry point (helpers of ops_cv_amd.aclnn):

    norm        residual_norm              root-mean-square norm of x, or of x + residual, which comes back too
    norm_int8   residual_norm_int8         the same with the result in 8 bits, one scale per row
    norm_grad   residual_norm_backward     gradients of x (and of the residual, which is the same) and of the weight
    rotary      rotary                     queries and keys rotated by their positions; inverse: the gradient's rotation
    attend      window_attention           attention to a window around each token and to a few first tokens (sinks)
    attend_grad window_attention_backward  gradients of queries, keys and values

With `own` false run() computes the same in elementary torch operations in 32 bits, rounded once at the end.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
EPS = 1e-6
ROTARY_BASE = 10000.0

# no drawn case asks for more than the largest listed one: scores of the plain form, operations, elements of a cache
MOST_SCORES = 2.1e9
MOST_FLOPS = 1.5e11
MOST_CACHE = 5.3e8


def _norm(name, op, dtype, rows, width, residual=True, rstd=False):
    return {"name": name, "op": op, "dtype": dtype, "rows": rows, "width": width, "residual": residual, "rstd": rstd}


def _rotary(name, dtype, b, s, heads, kv_heads, d, rot, table, interleaved=False, inverse=False):
    return {"name": name, "op": "rotary", "dtype": dtype, "b": b, "s": s, "heads": heads, "kv_heads": kv_heads, "d": d,
            "rot": rot, "table": table, "interleaved": interleaved, "inverse": inverse}


def _attend(name, dtype, b, sq, skv, heads, kv_heads, d, left, right, sinks, ragged=False, lse=False, op="attend"):
    return {"name": name, "op": op, "dtype": dtype, "b": b, "sq": sq, "skv": skv, "heads": heads, "kv_heads": kv_heads,
            "d": d, "left": left, "right": right, "sinks": sinks, "ragged": ragged, "lse": lse}


def listed():
    return [
        # eight sequences that grow by one token: the call whose cost is the call itself
        _norm("norm_token", "norm", "bf16", 8, 4096),
        # a prompt's tokens on their way into attention
        _norm("norm_prompt", "norm", "bf16", 8192, 4096),
        # the input of a product in 8 bits, an odd number of tokens
        _norm("norm_int8", "norm_int8", "fp16", 4099, 5120),
        # a training step's way back through a norm
        _norm("norm_train", "norm_grad", "bf16", 16384, 2048),
        # one new token of each of 64 sequences, far into a long context
        _rotary("rotary_token", "bf16", 64, 1, 32, 8, 128, 128, 131072),
        # two prompts
        _rotary("rotary_prompt", "bf16", 2, 4096, 32, 8, 128, 128, 8192),
        # gradients of the tokens of 37 x 37 patches in single precision, half of each head rotated
        _rotary("rotary_train", "fp32", 4, 1369, 16, 16, 80, 40, 2048, interleaved=True, inverse=True),
        # one new token of each of 32 sequences against caches of up to 16384 tokens
        _attend("attend_token", "bf16", 32, 1, 16384, 32, 8, 128, 4095, 0, 4, ragged=True),
        # a long prompt
        _attend("attend_prompt", "bf16", 1, 8192, 8192, 32, 8, 128, 1023, 0, 4),
        # a vision encoder's layer: 37 x 37 patches that see both ways, the first token seen by all
        _attend("attend_image", "fp16", 8, 1369, 1369, 16, 16, 64, 256, 256, 1),
        # a training step's way back through attention
        _attend("attend_train", "bf16", 1, 4096, 4096, 32, 8, 128, 1023, 0, 4, op="attend_grad"),
        # the same in single precision on padded sequences, heads of 72
        _attend("attend_train_odd", "fp32", 2, 777, 777, 12, 4, 72, 100, 0, 3, ragged=True, op="attend_grad"),
    ]


def _spread(rng, low, high):
    """A whole number of the range by its logarithm, odd or a power of two."""
    n = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(low, min(high, 1 << round(math.log2(n)) if rng.random() < 0.5 else int(n) | 1))


def draw(rng):
    op = rng.choice(["norm", "norm_int8", "norm_grad", "rotary", "attend", "attend", "attend_grad", "attend_grad"])
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    if op.startswith("norm"):
        width = rng.choice([768, 1024, 1280, 2048, 4096, 5120, 8192, 2 * rng.randint(50, 700) + 1])
        rows = _spread(rng, 1, min(16384, (1 << 26) // width))
        if op == "norm_int8" and dtype == "fp32":
            dtype = "bf16"
        c = _norm("", op, dtype, rows, width, residual=rng.random() < 0.7, rstd=op == "norm" and rng.random() < 0.5)
    elif op == "rotary":
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 4])
        d = rng.choice([32, 64, 72, 80, 96, 128, 256])
        rot = rng.choice([d, d // 2, d // 4])
        s = _spread(rng, 1, 8192)
        b = _spread(rng, 1, max(1, min(64, (1 << 25) // (s * heads * d))))
        c = _rotary("", dtype, b, s, heads, kv_heads, d, rot, max(s, _spread(rng, 2048, 131072)), rng.random() < 0.5,
                    rng.random() < 0.3)
    else:
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
        d = rng.choice([32, 64, 72, 80, 96, 128, 128, 256])
        kind = rng.choice(["image", "prompt", "prompt"] if op == "attend_grad" else ["image", "prompt", "chunk", "token"])
        longest = 16384 if kind in ("chunk", "token") else 4096 if heads * d <= 4096 else 2048
        skv = _spread(rng, 64, longest)
        sq = {"image": skv, "prompt": skv, "chunk": min(skv, _spread(rng, 16, 512)), "token": rng.choice([1, 1, 2, 4])}[kind]
        left = min(_spread(rng, 32, 8192), 4095)
        right = left // rng.choice([1, 2]) if kind == "image" else 0
        grad = op == "attend_grad"
        scores = heads * sq * skv * (8 if dtype == "fp32" else 4 if grad else 1)
        flops = heads * sq * min(skv, left + right + 1) * d * (10 if grad else 4)
        b = _spread(rng, 1, max(1, min(32, int(MOST_SCORES / scores), int(MOST_FLOPS / flops),
                                       int(MOST_CACHE / (skv * kv_heads * d)))))
        c = _attend("", dtype, b, sq, skv, heads, kv_heads, d, left, right, rng.choice([0, 1, 4, 16, 64]),
                    rng.random() < 0.5, not grad and rng.random() < 0.5, op)
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------------- inputs

def _lengths(c, generator=None):
    """Lengths of the sequences: spread evenly from a quarter of the longest to all of it, in an order by the seed."""
    n = [c["skv"] if not c["ragged"] else max(c["sq"] if c["sq"] < c["skv"] else 1, c["skv"] * (c["b"] + 3 * i) // (4 * c["b"]))
         for i in range(1, c["b"] + 1)]
    if generator is not None and c["ragged"]:
        n = [n[i] for i in torch.randperm(c["b"], generator=generator).tolist()]
    return n


def _normal(g, *size, dtype, scale=1.0):
    return (torch.randn(*size, generator=g, device="cuda") * scale).to(dtype)


def prepare(case, seed):
    c = dict(case)
    dtype = DTYPES[c["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(seed)
    if c["op"] in ("norm", "norm_int8", "norm_grad"):
        rows, width = c["rows"], c["width"]
        c["weight"] = 1 + _normal(g, width, dtype=torch.float32, scale=0.1)
        c["weight"] = c["weight"].to(dtype)
        x = _normal(g, rows, width, dtype=dtype)
        r = _normal(g, rows, width, dtype=dtype, scale=2.0) if c["residual"] else None
        if c["op"] == "norm_grad":
            c["sum"] = x if r is None else x + r
            c["rstd_in"] = torch.rsqrt(c["sum"].float().square().mean(-1) + EPS)
            c["grad_y"] = _normal(g, rows, width, dtype=dtype, scale=0.01)
            c["grad_sum"] = _normal(g, rows, width, dtype=dtype, scale=0.01) if r is not None else None
        else:
            c["x"], c["r"] = x, r
    elif c["op"] == "rotary":
        c["q"] = _normal(g, c["b"], c["s"], c["heads"], c["d"], dtype=dtype)
        c["k"] = _normal(g, c["b"], c["s"], c["kv_heads"], c["d"], dtype=dtype)
        half = c["rot"] // 2
        turn = ROTARY_BASE ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        angle = torch.arange(c["table"], device="cuda", dtype=torch.float64)[:, None] * turn
        c["angles"] = torch.cat([angle.cos(), angle.sin()], -1).float()
        first = torch.randint(0, c["table"] - c["s"] + 1, (c["b"], 1), generator=g, device="cuda")
        c["positions"] = first + torch.arange(c["s"], device="cuda")
    else:
        c["q"] = _normal(g, c["b"], c["sq"], c["heads"], c["d"], dtype=dtype)
        c["k"] = _normal(g, c["b"], c["skv"], c["kv_heads"], c["d"], dtype=dtype)
        c["v"] = _normal(g, c["b"], c["skv"], c["kv_heads"], c["d"], dtype=dtype)
        c["scale"] = 1 / math.sqrt(c["d"])
        c["kv_lengths"] = c["q_lengths"] = None
        if c["ragged"]:
            n = _lengths(c, torch.Generator().manual_seed(seed))
            c["kv_lengths"] = torch.tensor(n, device="cuda", dtype=torch.int32)
            if c["sq"] == c["skv"]:
                c["q_lengths"] = c["kv_lengths"]
        if c["op"] == "attend_grad":
            c["out"], c["lse_in"] = _plain_attention(c)
            c["grad_out"] = _normal(g, *c["q"].shape, dtype=dtype, scale=0.1)
    return c


# ---------------------------------------------------------------------------------------------------- plain forms

def _values(q, scale, dtype):
    """What 8-bit numbers with a scale per row stand for."""
    return torch.mul(q, scale[:, None], out=torch.empty(q.shape, dtype=dtype, device=q.device))


def _plain_norm(s):
    h = s["x"].float() if s["r"] is None else s["x"].float() + s["r"].float()
    rstd = torch.rsqrt(h.square().mean(-1) + EPS)
    summed = None if s["r"] is None else h.to(s["x"].dtype)
    t = h * s["weight"].float()
    if s["op"] == "norm_int8":
        most = t.abs().amax(-1)
        step = torch.where(most > 0, 127 / most, 0)
        q = torch.round(t * step[:, None]).to(torch.int8)
        scale = most * rstd / 127
        return _values(q, scale, s["x"].dtype), scale, summed
    return (t * rstd[:, None]).to(s["x"].dtype), summed, rstd if s["rstd"] else None


def _plain_norm_grad(s):
    n = s["sum"].float() * s["rstd_in"][:, None]
    gy = s["grad_y"].float()
    gn = gy * s["weight"].float()
    gx = (gn - n * (gn * n).mean(-1, keepdim=True)) * s["rstd_in"][:, None]
    if s["grad_sum"] is not None:
        gx = gx + s["grad_sum"].float()
    return gx.to(s["sum"].dtype), (gy * n).sum(0).to(s["weight"].dtype)


def _plain_rotate(x, cos, sin, rot, interleaved):
    x = x.float()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    p, q = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([p, q], -1).flatten(-2) if interleaved else torch.cat([p, q], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _plain_rotary(s):
    cos, sin = s["angles"][s["positions"]][:, :, None].chunk(2, -1)
    sin = -sin if s["inverse"] else sin
    return tuple(_plain_rotate(x, cos, sin, s["rot"], s["interleaved"]).to(x.dtype) for x in (s["q"], s["k"]))


def _plain_mask(s):
    """(b, sq, skv): whether a query sees a key."""
    dev = s["q"].device
    kv_len = s["kv_lengths"] if s["kv_lengths"] is not None else torch.full((s["b"],), s["skv"], device=dev)
    q_len = s["q_lengths"] if s["q_lengths"] is not None else torch.full((s["b"],), s["sq"], device=dev)
    i = torch.arange(s["sq"], device=dev)
    p = ((kv_len - q_len)[:, None] + i)[..., None]
    j = torch.arange(s["skv"], device=dev)
    seen = (j < kv_len[:, None])[:, None] & (j <= p + s["right"]) & ((j >= p - s["left"]) | (j < s["sinks"]))
    return seen & (i < q_len[:, None])[..., None]


def _heads_first(x, kv_heads):
    """(b, s, heads, d) as (b, kv_heads, heads / kv_heads * s, d) in 32 bits."""
    b, n, heads, d = x.shape
    return x.float().view(b, n, kv_heads, heads // kv_heads, d).permute(0, 2, 3, 1, 4).reshape(b, kv_heads, -1, d)


def _tokens_first(x, like):
    b, n, heads, d = like.shape
    kv_heads = x.shape[1]
    return x.view(b, kv_heads, heads // kv_heads, n, d).permute(0, 3, 1, 2, 4).reshape(b, n, heads, d).to(like.dtype)


def _plain_scores(s):
    """(b, kv_heads, heads / kv_heads, sq, skv), minus infinity where nothing is seen."""
    q, k = _heads_first(s["q"], s["kv_heads"]), _heads_first(s["k"], s["kv_heads"])
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(s["scale"])
    scores = scores.view(s["b"], s["kv_heads"], -1, s["sq"], s["skv"])
    return scores.masked_fill_(~_plain_mask(s)[:, None, None], -math.inf)


def _plain_attention(s):
    scores = _plain_scores(s)
    most = scores.amax(-1, keepdim=True)
    most = torch.where(most == -math.inf, 0, most)
    p = scores.sub_(most).exp_()
    total = p.sum(-1, keepdim=True)
    v = _heads_first(s["v"], s["kv_heads"])
    out = torch.matmul(p.view(s["b"], s["kv_heads"], -1, s["skv"]), v) / torch.where(total > 0, total, 1).flatten(2, 3)
    lse = (most + total.log()).view(s["b"], s["heads"], s["sq"])
    return _tokens_first(out, s["q"]), lse


def _plain_attention_grad(s):
    lse = s["lse_in"].view(s["b"], s["kv_heads"], -1, s["sq"], 1)
    lse = torch.where(lse == -math.inf, 0, lse)
    p = _plain_scores(s).sub_(lse).exp_().view(s["b"], s["kv_heads"], -1, s["skv"])
    go, o = _heads_first(s["grad_out"], s["kv_heads"]), _heads_first(s["out"], s["kv_heads"])
    q, k, v = (_heads_first(s[n], s["kv_heads"]) for n in "qkv")
    gv = torch.matmul(p.transpose(2, 3).contiguous(), go)
    gs = torch.matmul(go, v.transpose(2, 3).contiguous()).sub_((go * o).sum(-1, keepdim=True)).mul_(p).mul_(s["scale"])
    gq = torch.matmul(gs, k)
    gk = torch.matmul(gs.transpose(2, 3).contiguous(), q)
    return _tokens_first(gq, s["q"]), _tokens_first(gk, s["k"]), _tokens_first(gv, s["v"])


# ---------------------------------------------------------------------------------------------------- one pass

def run(state):
    s = state
    if not own:
        if s["op"] in ("norm", "norm_int8"):
            return _plain_norm(s)
        if s["op"] == "norm_grad":
            return _plain_norm_grad(s)
        if s["op"] == "rotary":
            return _plain_rotary(s)
        if s["op"] == "attend_grad":
            return _plain_attention_grad(s)
        out, lse = _plain_attention(s)
        return out, lse if s["lse"] else None
    from ops_cv_amd import aclnn
    if s["op"] == "norm":
        return aclnn.residual_norm(s["x"], s["weight"], residual=s["r"], eps=EPS, need_rstd=s["rstd"])
    if s["op"] == "norm_int8":
        q, scale, summed, _ = aclnn.residual_norm_int8(s["x"], s["weight"], residual=s["r"], eps=EPS)
        return _values(q, scale, s["x"].dtype), scale, summed
    if s["op"] == "norm_grad":
        return aclnn.residual_norm_backward(s["grad_y"], s["sum"], s["weight"], s["rstd_in"], grad_sum=s["grad_sum"])
    if s["op"] == "rotary":
        return aclnn.rotary(s["q"], s["k"], s["angles"], positions=s["positions"], interleaved=s["interleaved"],
                            inverse=s["inverse"])
    masks = {n: s[n] for n in ("scale", "left", "right", "sinks", "q_lengths", "kv_lengths")}
    if s["op"] == "attend":
        return aclnn.window_attention(s["q"], s["k"], s["v"], need_lse=s["lse"], **masks)
    return aclnn.window_attention_backward(s["grad_out"], s["q"], s["k"], s["v"], s["out"], s["lse_in"], **masks)


# ---------------------------------------------------------------------------------------------------- work

def _seen_pairs(c):
    """Pairs of a query and a key that it sees, and keys seen by any query, over all sequences, for one head."""
    pairs = keys = 0
    for n in _lengths(c):
        rows = min(c["sq"], n) if c["sq"] == c["skv"] else c["sq"]
        lowest = n
        for p in range(n - rows, n):
            last = min(n - 1, p + c["right"])
            first = max(0, p - c["left"])
            lowest = min(lowest, first)
            pairs += last + 1 - first + min(c["sinks"], first)
        keys += n - lowest + min(c["sinks"], lowest)
    return pairs, keys


def work(case):
    c = case
    e = BYTES[c["dtype"]]
    if c["op"].startswith("norm"):
        n = c["rows"] * c["width"]
        if c["op"] == "norm_grad":  # grad_y, sum and, with a residual, grad_sum; the gradient; 32-bit rstd
            return {"bytes": n * e * (4 if c["residual"] else 3) + 2 * c["width"] * e + 4 * c["rows"], "flops": 10 * n}
        # values in 8 bits come back as the numbers that they stand for
        moved = n * e * (4 if c["residual"] else 2)
        return {"bytes": moved + c["width"] * e + 4 * c["rows"], "flops": 5 * n}
    if c["op"] == "rotary":
        n = c["b"] * c["s"] * (c["heads"] + c["kv_heads"]) * c["d"]
        return {"bytes": 2 * n * e + c["b"] * c["s"] * (4 * c["rot"] + 8), "flops": 3 * n * c["rot"] // c["d"]}
    pairs, keys = _seen_pairs(c)
    q = c["b"] * c["sq"] * c["heads"] * c["d"] * e
    kv = 2 * keys * c["kv_heads"] * c["d"] * e
    row = c["b"] * c["sq"] * c["heads"] * 4
    if c["op"] == "attend":  # two products
        return {"bytes": 2 * q + kv + (row if c["lse"] else 0), "flops": 4 * c["heads"] * c["d"] * pairs}
    # queries, outputs, their gradients and the queries' gradients; keys, values and theirs; five products
    return {"bytes": 4 * q + 2 * kv + row, "flops": 10 * c["heads"] * c["d"] * pairs}


# ---------------------------------------------------------------------------------------------------- 64 bits

def _exact_norm(s):
    h = s["x"].double()
    if s["r"] is not None:
        h = h + s["r"].double()
    root = (h.pow(2).sum(1, keepdim=True) / h.shape[1] + EPS).sqrt()
    y = h / root * s["weight"].double()
    summed = None if s["r"] is None else h
    if s["op"] == "norm_int8":
        scale = y.abs().max(1, keepdim=True).values / 127
        return None, scale[:, 0], summed
    return y, summed, 1 / root[:, 0] if s["rstd"] else None


def _exact_norm_grad(s):
    h, r = s["sum"].double(), s["rstd_in"].double()[:, None]
    gy, w = s["grad_y"].double(), s["weight"].double()
    along = (gy * w * h).sum(1, keepdim=True) / h.shape[1]
    gx = r * gy * w - r.pow(3) * h * along
    if s["grad_sum"] is not None:
        gx += s["grad_sum"].double()
    return gx, torch.einsum("ij,ij->j", gy, h * r)


def _exact_rotary(s):
    rot, out = s["rot"], []
    half = rot // 2
    first, second = (range(0, rot, 2), range(1, rot, 2)) if s["interleaved"] else (range(half), range(half, rot))
    first, second = (torch.tensor(list(r), device="cuda") for r in (first, second))
    at = s["angles"].double()[s["positions"]]
    turn = torch.complex(at[..., :half], at[..., half:])[:, :, None]
    turn = turn.conj() if s["inverse"] else turn
    for x in (s["q"], s["k"]):
        y = x.double().clone()
        z = torch.complex(y[..., first], y[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        out.append(y)
    return tuple(out)


def _exact_attention(s, grad):
    """One sequence and one query head at a time, its rows in blocks."""
    group = s["heads"] // s["kv_heads"]
    lens = s["kv_lengths"].tolist() if s["kv_lengths"] is not None else [s["skv"]] * s["b"]
    rows = s["q_lengths"].tolist() if s["q_lengths"] is not None else [s["sq"]] * s["b"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full((s["b"], s["heads"], s["sq"]), -math.inf, dtype=torch.float64, device="cuda")
    gq, gk, gv = (torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in "qkv") if grad else (None,) * 3
    for b in range(s["b"]):
        n, m = lens[b], rows[b]
        j = torch.arange(n, device="cuda")
        p = torch.arange(n - m, n, device="cuda")[:, None]
        hidden = (j > p + s["right"]) | ((j < p - s["left"]) & (j >= s["sinks"]))
        for h in range(s["heads"]):
            q, k, v = s["q"][b, :m, h].double(), s["k"][b, :n, h // group].double(), s["v"][b, :n, h // group].double()
            scores = (q @ k.T * s["scale"]).masked_fill(hidden, -math.inf)
            lse[b, h, :m] = torch.logsumexp(scores, 1)
            weights = torch.softmax(scores, 1).nan_to_num(0.0)
            out[b, :m, h] = weights @ v
            if grad:
                go = s["grad_out"][b, :m, h].double()
                gw = go @ v.T
                gs = weights * (gw - (weights * gw).sum(1, keepdim=True)) * s["scale"]
                gq[b, :m, h] = gs @ k
                gk[b, :n, h // group] += gs.T @ q
                gv[b, :n, h // group] += weights.T @ go
    return (gq, gk, gv) if grad else (out, lse if s["lse"] else None)


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] in ("norm", "norm_int8"):
        return _exact_norm(s)
    if s["op"] == "norm_grad":
        return _exact_norm_grad(s)
    if s["op"] == "rotary":
        return _exact_rotary(s)
    return _exact_attention(s, s["op"] == "attend_grad")
