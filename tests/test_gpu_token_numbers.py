"""The operators on token sequences at the ends of their types' ranges, against plain implementations in 64 bits."""
import math

import pytest
import torch

import token_oracle as O

pytestmark = pytest.mark.gpu

NONE = 2 ** 63 - 1


def gen(*key):
    return torch.Generator().manual_seed(sum((i + 1) * ord(c) for i, c in enumerate(str(key))))


def normal(g, *size, dtype="fp16", scale=1.0):
    return (torch.randn(*size, generator=g, dtype=torch.float64) * scale).to(O.DTYPES[dtype])


# -------------------------------------------------------------------------------- gradients of attention in FLOAT16

def gradient_bounds(r, q, k, v, go, scale, dtype):
    """How far the gradients may be, entry by entry.

    off_ij, the error of the scores' gradient gs_ij = w_ij (go_i . v_j - D_i) as an operand of the products that follow: it is
    rounded to the type (relative U); the weight and the two terms of the difference carry 32-bit errors (F32), D_i the
    rounding of `out` (U).  FLOAT16 has 2^-25 of absolute error on top, of whatever the largest operand is divided by: a row's
    own largest where rows are summed up (gq), a key's own largest where keys are (gk).  Weights as operands (gv): relative U,
    and nothing absolute that would show, since no weight exceeds 1 and the products have 32 bits."""
    u, tiny = O.U[dtype], O.TINY[dtype]
    group = q.shape[2] // k.shape[2]
    spread = lambda x: x.double().abs().repeat_interleave(group, 2).transpose(1, 2)  # noqa: E731
    gather = lambda x: x.transpose(1, 2).unflatten(2, (k.shape[2], group)).sum(3)  # noqa: E731
    w, gs = r["weights"], r["gs"].abs()
    vs, ks, qs = spread(v), spread(k), q.double().abs().transpose(1, 2)
    g = go.double().abs().transpose(1, 2)
    along = (g * r["out"].abs().transpose(1, 2)).sum(-1, keepdim=True)
    off = gs * (u + O.F32) + w * (g @ vs.transpose(2, 3) + along) * O.F32 + w * along * u
    low = 2.0 ** -25 if dtype == "fp16" else 0.0
    off_row = off + low * gs.amax(3, keepdim=True) * (w > 0)
    # a key's gradient is one sum over the rows of all the heads that share it
    most = gs.amax(2, keepdim=True).unflatten(1, (-1, group)).amax(2, keepdim=True).expand(-1, -1, group, -1, -1).flatten(1, 2)
    off_key = off + low * most * (w > 0)
    return ((off_row @ ks * scale).transpose(1, 2) + u * r["gq"].abs() + tiny,
            gather(off_key.transpose(2, 3) @ qs) * scale + u * r["gk"].abs() + tiny,
            gather((w * (u + O.F32)).transpose(2, 3) @ g) + u * r["gv"].abs() + tiny)


def check_gradients(device, aclnn, q, k, v, go, dtype, which=("gq", "gk", "gv"), **masks):
    r = O.attention(q, k, v, grad_out=go, **masks)
    bounds = gradient_bounds(r, q, k, v, go, masks["scale"], dtype)
    dev = [t.to(device) for t in (go, q, k, v, r["out"].to(q.dtype), r["lse"].float())]
    got = aclnn.window_attention_backward(*dev, **masks)
    for name, x, bound in zip(("gq", "gk", "gv"), got, bounds):
        assert r[name].abs().max() < 65000  # the results themselves are numbers of the type
        if name in which:
            O.within(x, r[name], bound, name)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("b,sq,d", [(1, 40, 64), (1, 40, 128), (1, 70, 256), (2, 300, 80), (130, 140, 32)])
def test_gradients_of_large_values(device, aclnn, dtype, b, sq, d):
    """Two keys a query, whose values differ by what makes the score's gradient, over the size of gradOut, pass 65504."""
    g = gen("large values", dtype, b, sq, d)
    q, k = normal(g, b, sq, 4, d, dtype=dtype, scale=0.1), normal(g, b, sq, 2, d, dtype=dtype)
    sign = torch.ones(sq).double()
    sign[::2] = -1
    size = 1.1 * 2 * 65504 / d
    v = (size * sign[None, :, None, None] * (1 + 0.01 * torch.randn(b, sq, 2, d, generator=g, dtype=torch.float64))).to(O.DTYPES[dtype])
    go = torch.full(q.shape, 2.0 ** -10, dtype=q.dtype)
    check_gradients(device, aclnn, q, k, v, go, dtype, scale=0.1, left=1, right=0, sinks=0)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("b,sq,heads,d,left", [(1, 300, 1, 64, 100), (2, 200, 4, 128, NONE), (70, 260, 4, 64, 100), (1, 150, 2, 256, 60)])
@pytest.mark.parametrize("which", [("gq", "gk"), ("gv",)], ids=["scores", "values"])
def test_gradients_beside_loud_rows(device, aclnn, dtype, b, sq, heads, d, left, which):
    """Every eighth query has a gradient 1e5 times as large as the others', and looks at its own key alone: what the other
    queries leave in the other keys keeps its bits."""
    g = gen("loud rows", dtype, b, sq, heads, d)
    q, k = normal(g, b, sq, heads, d, dtype=dtype, scale=0.1), normal(g, b, sq, 1, d, dtype=dtype)
    v = normal(g, b, sq, 1, d, dtype=dtype)
    go = normal(g, b, sq, heads, d, dtype=dtype, scale=0.3)
    loud = torch.arange(sq) % 8 == 3
    scale = 1 / math.sqrt(d)
    q[:, loud] = (k[:, loud] * (30 / math.sqrt(d))).expand(-1, -1, heads, -1)  # a score of 30 or so with its own key
    go[:, loud] = go[:, loud] * 2e4
    check_gradients(device, aclnn, q, k, v, go, dtype, which, scale=scale, left=left, right=0, sinks=0)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("b,sq,heads,d", [(1, 300, 1, 64), (2, 200, 4, 128), (70, 260, 4, 32), (1, 150, 2, 256), (70, 260, 4, 160)])
def test_gradients_that_grow_along_the_row(device, aclnn, dtype, b, sq, heads, d):
    """Every other query looks at its own key and the one before it, past many that have a millionth of their weight or less:
    the gradients of its first scores are a million times smaller than those of its last ones."""
    g = gen("growing", dtype, b, sq, heads, d)
    k, v = normal(g, b, sq, 1, d, dtype=dtype), normal(g, b, sq, 1, d, dtype=dtype)
    q = normal(g, b, sq, heads, d, dtype=dtype, scale=0.1)
    pair = (k.double() + k.double().roll(1, 1)) * (20 / math.sqrt(d))
    q[:, ::2] = pair[:, ::2].expand(-1, -1, heads, -1).to(q.dtype)
    go = normal(g, b, sq, heads, d, dtype=dtype)
    check_gradients(device, aclnn, q, k, v, go, dtype, ("gq", "gk"), scale=1 / math.sqrt(d), left=NONE, right=0, sinks=0)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("keys", [5000, 104531])
def test_value_gradients_of_small_weights(device, aclnn, dtype, keys):
    """Queries that weigh all keys alike: 1 / keys has its bits also below the normal numbers of FLOAT16."""
    g = gen("small weights", dtype, keys)
    q = torch.zeros(1, 2, 1, 64, dtype=O.DTYPES[dtype])
    k, v = normal(g, 1, keys, 1, 64, dtype=dtype), normal(g, 1, keys, 1, 64, dtype=dtype)
    go = normal(g, 1, 2, 1, 64, dtype=dtype, scale=3000)
    check_gradients(device, aclnn, q, k, v, go, dtype, scale=0.125, left=NONE, right=NONE, sinks=0)


# ------------------------------------------------------------------------------------------------- forward, weights

@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("sq", [1, 16384])
def test_many_small_weights_beside_a_large_one(device, aclnn, dtype, sq):
    """A first token that takes most of the weight, and a quarter of a million others that share the rest: each has a
    millionth of the largest weight, and they add up to a fifth of the whole.  All queries are the same one."""
    g = gen("small", dtype)
    n, d = 262144, 64
    q, k = torch.zeros(1, 1, 2, d, dtype=O.DTYPES[dtype]), torch.zeros(1, n, 1, d, dtype=O.DTYPES[dtype])
    q[..., 0], k[:, 0, :, 0] = 1, 14
    v = (3 + 0.1 * torch.randn(1, n, 1, d, generator=g, dtype=torch.float64)).to(O.DTYPES[dtype])
    v[:, 0] = 0
    # exp(-13.8352) is 16.45 steps of FLOAT16's smallest numbers
    masks = dict(scale=13.8352 / 14, left=NONE, right=NONE, sinks=0)
    out, lse = aclnn.window_attention(q.expand(1, sq, 2, d).to(device), k.to(device), v.to(device), need_lse=True, **masks)
    want = O.attention(q, k, v, **masks)
    # weights are rounded to the type (relative U); a running sum of the weights takes up to nine additions for 64 keys and
    # one of the weighted values one for 16, each of which rounds by 2^-24 of the sum
    sums = (n / 64 * 9 + n / 16) * 2.0 ** -24
    u = O.U[dtype]
    O.within(out, want["out"].expand(1, sq, 2, d), (2 * u + sums) * want["out"].abs(), "out")
    O.within(lse, want["lse"].expand(1, 2, sq), sums + 1e-5, "lse")


# ------------------------------------------------------------------------------------------------------ 8-bit norm

@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("width", [8, 100, 2048, 40000])
def test_8_bit_norm_of_tiny_rows(device, aclnn, dtype, width):
    """Rows whose largest product is too small for 127 / m to be a number of 32 bits: m below 3.7e-37."""
    x = torch.zeros(6, width, dtype=O.DTYPES[dtype])
    x[0, :4] = torch.tensor([1e-38, 0.0, 5.1e-39, -2.3e-39])
    x[1, :4] = torch.tensor([-3e-37, 1e-37, 0.0, 2e-38])
    x[2, 1], x[3, 0] = 1e-40, 3.8e-37
    x[4, :3] = torch.tensor([1.0, 1e-38, 0.0])
    w = torch.ones(width, dtype=O.DTYPES[dtype])
    q, scale, _, _ = aclnn.residual_norm_int8(x.to(device), w.to(device))
    t = x.double()
    most = t.abs().amax(1, keepdim=True)
    want = torch.where(most > 0, t * 127 / torch.where(most > 0, most, 1), 0)
    assert ((want - want.floor()) - 0.5).abs().min() > 1e-3  # no ties
    assert torch.equal(q.cpu().double(), want.round())
    rstd = 1 / torch.sqrt(t.square().mean(1) + 1e-6)
    O.within(scale, most[:, 0] * rstd / 127, O.F32 * most[:, 0] * rstd / 127 + 2.0 ** -149, "scale")


def test_8_bit_norm_of_zeros_without_eps(device, aclnn):
    for width in (16, 40000):
        x, w = torch.zeros(3, width), torch.ones(width)
        x[1] = 2
        q, scale, _, _ = aclnn.residual_norm_int8(x.to(device), w.to(device), eps=0.0)
        assert (q[0] == 0).all() and (q[1] == 127).all() and (q[2] == 0).all()
        assert scale[0] == 0 and scale[2] == 0 and abs(scale[1].item() - 1 / 127) < 1e-7
