"""Layer norm, rotary positions on several axes, dropout and gated projections against plain implementations in 64 bits
(block_oracle.py)."""
import math

import numpy as np
import pytest
import torch

import block_oracle as B

pytestmark = pytest.mark.gpu

DTYPES = list(B.DTYPES)


def rand(g, *size, dtype, scale=1.0, shift=0.0):
    return (torch.randn(*size, generator=g, dtype=torch.float64) * scale + shift).to(B.DTYPES[dtype])


def gen(*key):
    return torch.Generator().manual_seed(sum((i + 1) * ord(c) for i, c in enumerate(str(key))))


def close(got, want, off, dtype, what):
    B.within(got, want, off + B.U[dtype] * want.abs() + B.TINY[dtype], what)


def on(device, *tensors):
    return [None if t is None else t.to(device) for t in tensors]


# -------------------------------------------------------------------------------------------------------- layer norm

NORM_SIZES = [(1, 1), (3, 5), (4, 64), (7, 100), (2, 768), (130, 1024), (5, 1001), (4100, 1040), (4099, 1301), (3, 2056),
              (2, 4096), (3, 8192), (2, 9001), (2, 40000), (2, 33001)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width", NORM_SIZES)
def test_layer_norm(device, aclnn, dtype, rows, width):
    g = gen("layer norm", dtype, rows, width)
    x, r = rand(g, rows, width, dtype=dtype), rand(g, rows, width, dtype=dtype, scale=3, shift=2)
    w, b = rand(g, width, dtype=dtype), rand(g, width, dtype=dtype)
    for residual, weight, bias in ((None, w, b), (r, w, b), (r, None, None), (r, w, None), (None, None, b)):
        y, h, mean, rstd, off = B.layer_norm(x, residual, weight, bias, 1e-5)
        got, total, got_mean, got_rstd = aclnn.layer_norm(*on(device, x, weight, bias, residual), eps=1e-5, need_stats=True)
        close(got, y, off, dtype, "norm")
        size = h.abs().mean(-1)
        B.within(got_mean, mean, B.F32 * size, "mean")
        B.within(got_rstd, rstd, B.F32 * (1 + size * rstd) * rstd, "rstd")
        assert (total is None) == (residual is None)
        if residual is not None:
            assert torch.equal(total.cpu(), (x.float() + r.float()).to(x.dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width", NORM_SIZES + [(3000, 96), (700, 2048), (1100, 7)])
def test_layer_norm_gradients(device, aclnn, dtype, rows, width):
    g = gen("layer norm gradients", dtype, rows, width)
    h, gy, gs = rand(g, rows, width, dtype=dtype, shift=1), rand(g, rows, width, dtype=dtype), rand(g, rows, width, dtype=dtype)
    w = rand(g, width, dtype=dtype)
    mean = h.double().mean(-1)
    rstd = (1 / torch.sqrt(h.double().var(-1, correction=0) + 1e-5)).float()
    mean = mean.float()
    for grad_sum, weight in ((None, w), (gs, w), (gs, None)):
        want, off = B.layer_norm_grad(gy, grad_sum, h, weight, mean, rstd)
        dev = on(device, gy, h, weight, mean, rstd, grad_sum)
        got = aclnn.layer_norm_backward(*dev)
        close(got[0], want[0], off[0], dtype, "gradient of x")
        assert (got[1] is None) == (weight is None)
        if weight is not None:
            close(got[1], want[1], off[1], dtype, "gradient of the weight")
        close(got[2], want[2], off[2], dtype, "gradient of the bias")
        for need_weight, need_bias in ((False, False), (True, False), (False, True)):
            some = aclnn.layer_norm_backward(*dev, need_weight=need_weight, need_bias=need_bias)
            assert torch.equal(some[0], got[0])
            assert (some[1] is None) == (not need_weight or weight is None) and (some[2] is None) == (not need_bias)
            assert all(s is None or torch.equal(s, t) for s, t in zip(some, got))


def test_layer_norm_gradient_against_differences(device, aclnn):
    g = gen("layer norm differences")
    x, r, w, b = (rand(g, *s, dtype="fp32") for s in ((5, 300), (5, 300), (300,), (300,)))
    gy, gs = rand(g, 5, 300, dtype="fp32"), rand(g, 5, 300, dtype="fp32")
    y, total, mean, rstd = aclnn.layer_norm(*on(device, x, w, b, r), need_stats=True)
    gx, gw, gb = aclnn.layer_norm_backward(gy.to(device), total, w.to(device), mean, rstd, grad_sum=gs.to(device))

    def value(x, w, b):
        y, h = B.layer_norm(x, r, w, b, 1e-5)[:2]
        return (y * gy.double()).sum() + (h * gs.double()).sum()
    step = 1e-4
    for i, grad in enumerate((gx, gw, gb)):
        e = rand(g, *grad.shape, dtype="fp32").double()
        ahead, back = [[t.double() + (s * step * e if i == j else 0) for j, t in enumerate((x, w, b))] for s in (1, -1)]
        slope = (value(*ahead) - value(*back)) / (2 * step)
        terms = grad.cpu().double() * e
        # second-order differences leave step^2 of the third derivative, 32-bit results F32 of the terms
        assert abs(slope - terms.sum()) <= 1e-5 * terms.abs().sum()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_layer_norm_float_weight(device, aclnn, dtype):
    g = gen("layer norm weight", dtype)
    x, gy, w, b = rand(g, 6, 520, dtype=dtype), rand(g, 6, 520, dtype=dtype), rand(g, 520, dtype="fp32"), rand(g, 520, dtype="fp32")
    y, h, mean, rstd, off = B.layer_norm(x, None, w, b, 1e-5)
    got, _, m, r = aclnn.layer_norm(*on(device, x, w, b), need_stats=True)
    close(got, y, off, dtype, "norm")
    want, off = B.layer_norm_grad(gy, None, x, w, m.cpu(), r.cpu())
    gx, gw, gb = aclnn.layer_norm_backward(gy.to(device), x.to(device), w.to(device), m, r)
    assert gw.dtype == gb.dtype == torch.float32
    close(gx, want[0], off[0], dtype, "gradient of x")
    close(gw, want[1], off[1], "fp32", "gradient of the weight")
    close(gb, want[2], off[2], "fp32", "gradient of the bias")


def test_layer_norm_far_mean(device, aclnn):
    """A mean 4096 times the spread: the squares of what is left after its subtraction, which is exact here."""
    g = gen("far mean")
    x = (4096 + torch.randint(-3, 4, (4, 3000), generator=g)).float()
    got, _, mean, rstd = aclnn.layer_norm(x.to(device), need_stats=True)
    want = B.layer_norm(x, None, None, None, 1e-5)
    # the mean is a number of 32 bits near 4096: half a step of it, 2^-12, and the sum's roundings, which are a few of them
    B.within(mean, want[2], 2.0 ** -10, "mean")
    B.within(rstd, want[3], 1e-5 * want[3], "rstd")
    B.within(got, want[0], 2.0 ** -10 * want[3][:, None] + 1e-5 * want[0].abs(), "norm")


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_rows_that_are_not_finite(device, aclnn, dtype):
    """They stay where they are: every other row as without them.  A row of one value has no spread: its bias."""
    g = gen("not finite", dtype)
    x, w, b = rand(g, 9, 200, dtype=dtype), rand(g, 200, dtype=dtype), rand(g, 200, dtype=dtype)
    clean = aclnn.layer_norm(*on(device, x, w, b))[0]
    x[2, 7], x[5, 199], x[6] = math.nan, -math.inf, 0.25
    got = aclnn.layer_norm(*on(device, x, w, b))[0]
    for row in (0, 1, 3, 4, 7, 8):
        assert torch.equal(got[row], clean[row])
    assert got[2].isnan().all() and got[5].isnan().all()
    B.within(got[6], b.double(), 0.0, "a row of one value")


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_views_and_in_place(device, aclnn, dtype):
    g = gen("layer norm views", dtype)
    big = rand(g, 3, 9, 4, 160, dtype=dtype).to(device)
    w, b = rand(g, 160, dtype=dtype).to(device)[::2], rand(g, 80, dtype=dtype).to(device)
    for view in (big[:, ::2, :, 16:96], big[..., ::2], big[:, :, 1, 3:83], big.transpose(1, 2)[..., :80], big[:1, :, :, 80:],
                 big[0, 0, 0, :80], big[:, :1, :1, 1:81].expand(3, 5, 2, 80)):
        plain = view.contiguous()
        got, want = (aclnn.layer_norm(v, w, b, need_stats=True) for v in (view, plain))
        assert all(p is None or torch.equal(p, q) for p, q in zip(got, want))
        out = torch.full((*view.shape[:-1], 240), 7.0, dtype=view.dtype, device=device)
        aclnn.layer_norm(view, w, b, out=out[..., 3:83])
        assert torch.equal(out[..., 3:83], want[0]) and (out[..., :3] == 7).all() and (out[..., 83:] == 7).all()
        back = [aclnn.layer_norm_backward(v, v, w, want[2], want[3]) for v in (view, plain)]
        assert all(torch.equal(p, q) for p, q in zip(*back))
    x, r = rand(g, 50, 80, dtype=dtype).to(device), rand(g, 50, 80, dtype=dtype).to(device)
    want, total, mean, rstd = aclnn.layer_norm(x, w, b, r, need_stats=True)
    for into in (0, 1):
        both = [x.clone(), r.clone()]
        got, same, _, _ = aclnn.layer_norm(both[0], w, b, both[1], sum_out=both[into])
        assert torch.equal(got, want) and torch.equal(both[into], total) and same.data_ptr() == both[into].data_ptr()
    gx, gw, gb = aclnn.layer_norm_backward(x, total, w, mean, rstd, grad_sum=r)
    for into in (0, 1):
        both = [x.clone(), r.clone()]
        _, w2, b2 = aclnn.layer_norm_backward(both[0], total, w, mean, rstd, grad_sum=both[1], grad_x=both[into])
        assert torch.equal(both[into], gx) and torch.equal(w2, gw) and torch.equal(b2, gb)
    long = rand(g, 3, 70000, dtype=dtype).to(device)
    y, _, mean, rstd = aclnn.layer_norm(long, need_stats=True)
    want = aclnn.layer_norm_backward(y, long, None, mean, rstd)
    got = aclnn.layer_norm_backward(y, long, None, mean, rstd, grad_x=y)
    assert torch.equal(y, want[0]) and torch.equal(got[2], want[2])


def test_layer_norm_no_rows(device, aclnn):
    x = torch.empty(0, 64, device=device, dtype=torch.bfloat16)
    w = torch.ones(64, device=device, dtype=torch.bfloat16)
    y, _, mean, rstd = aclnn.layer_norm(x, w, need_stats=True)
    assert y.shape == x.shape and mean.shape == (0,)
    gx, gw, gb = aclnn.layer_norm_backward(y, x, w, mean, rstd)
    assert gx.shape == x.shape and (gw == 0).all() and (gb == 0).all()


# ------------------------------------------------------------------------------------------------------- rotary axes

AXES = [(2, 33, 4, 2, 64, [8, 12, 12], 0), (1, 100, 3, 3, 80, [20, 20], 1), (2, 17, 8, 1, 128, [24, 20, 20], 2),
        (1, 9, 2, 1, 72, [9, 5, 7], 0), (3, 5, 1, 1, 6, [1, 2], 2), (1, 64, 4, 4, 256, [40, 0, 64], 1),
        (2, 7, 2, 2, 96, [10, 11, 12, 13], 2), (1, 1, 1, 1, 2, [1], 0), (1, 3, 2, 0, 1024, [512], 0),
        (1, 2000, 16, 4, 128, [16, 24, 24], 0)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,s,heads,kv,d,sections,layout", AXES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_axes(device, aclnn, dtype, b, s, heads, kv, d, sections, layout, interleaved):
    g = gen("axes", dtype, b, s, heads, d, sections, layout, interleaved)
    q = rand(g, b, s, heads, d, dtype=dtype)
    k = rand(g, b, s, kv, d, dtype=dtype) if kv else None
    columns = max(sections) if layout == 1 else sum(sections)
    table = torch.randn(50, 2 * columns, generator=g)
    positions = torch.randint(0, 50, (len(sections), b, s), generator=g, dtype=torch.int32 if s % 2 else torch.int64)
    positions[-1, 0, 0] = 50 if sections[-1] else 0  # no row of the table
    if b > 1:
        positions[0, 1, s // 2] = -1
    for inverse in (False, True):
        got = aclnn.rotary_axes(*on(device, q, k, table, positions), sections, layout=layout, interleaved=interleaved,
                                inverse=inverse)
        for x, y in zip((q, k), got):
            assert (x is None) == (y is None)
            if x is not None:
                want, off = B.rotary_axes(x, table, positions, sections, layout, interleaved, inverse)
                close(y, want, off, dtype, "rotated")


@pytest.mark.parametrize("dtype", DTYPES)
def test_rotary_axes_of_equal_positions_are_one(device, aclnn, dtype):
    g = gen("one axis", dtype)
    q, k = rand(g, 2, 40, 4, 96, dtype=dtype).to(device), rand(g, 2, 40, 2, 96, dtype=dtype).to(device)
    table = aclnn.rotary_table(q, 64, 64)
    at = torch.randint(0, 64, (2, 40), generator=g).to(device)
    for interleaved in (False, True):
        want = aclnn.rotary(q, k, table, at, interleaved=interleaved)
        for sections in ([32], [8, 24], [5, 20, 7], [16, 0, 8, 8]):
            for layout in (aclnn.AXES_CONSECUTIVE, aclnn.AXES_DEALT):
                got = aclnn.rotary_axes(q, k, table, at.expand(len(sections), 2, 40), sections, layout=layout,
                                        interleaved=interleaved)
                assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_rotary_axes_views_in_place_and_back(device, aclnn):
    g = gen("axes views")
    q, k = rand(g, 2, 30, 4, 64, dtype="fp32").to(device), rand(g, 2, 30, 2, 64, dtype="fp32").to(device)
    table = aclnn.rotary_table(q, 40, 64)
    at = torch.randint(0, 40, (3, 2, 30), generator=g).to(device)
    sections = [8, 12, 12]
    want = aclnn.rotary_axes(q, k, table, at, sections)
    strided = torch.empty(30, 3, 2, 2, device=device, dtype=torch.int64)[..., 1].permute(1, 2, 0)
    strided.copy_(at)
    wide = torch.zeros(2, 30, 4, 100, device=device)
    wide[..., 5:69] = q
    backwards = table.flip(0).contiguous().flip(0)
    for q2, t2, at2 in ((q, table, strided), (wide[..., 5:69], table, at), (q.transpose(1, 2).contiguous().transpose(1, 2), table, at),
                        (q, torch.cat([table, table], 1)[:, :64], at), (q, backwards, at)):
        got = aclnn.rotary_axes(q2, k, t2, at2, sections)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    turned = [q.clone(), k.clone()]
    aclnn.rotary_axes(*turned, table, at, sections, query_out=turned[0], key_out=turned[1])
    assert all(torch.equal(x, y) for x, y in zip(turned, want))
    back = aclnn.rotary_axes(*want, table, at, sections, inverse=True)
    for x, y in zip(back, (q, k)):  # cosine^2 + sine^2 of rounded numbers, twice rounded products
        B.within(x, y.cpu().double(), 2e-6, "there and back")


# ----------------------------------------------------------------------------------------------------------- dropout

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [(1,), (7,), (8,), (3, 5), (5, 64), (9, 100), (1, 4097), (130, 1024), (2, 3, 7, 40)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.99999, 1.0])
def test_dropout(device, aclnn, dtype, size, p):
    g = gen("dropout", dtype, size, p)
    x, r = rand(g, *size, dtype=dtype), rand(g, *size, dtype=dtype)
    for state in ((0, 0), (-2 ** 63, 2 ** 63 - 1), (1234567890123, 42 << 32 | 7)):
        at = torch.tensor(state, dtype=torch.int64, device=device)
        for residual in (None, r):
            want, keep = B.dropout(x, residual, state, p)
            assert torch.equal(aclnn.dropout(x.to(device), at, p, None if residual is None else r.to(device)).cpu(), want)
        bad = x.clone()
        bad[~keep] = math.nan
        assert torch.equal(aclnn.dropout(bad.to(device), at, p).cpu(), B.dropout(x, None, state, p)[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_dropout_views_in_place_and_gradient(device, aclnn, dtype):
    g = gen("dropout views", dtype)
    big = rand(g, 6, 9, 160, dtype=dtype).to(device)
    state = torch.tensor([[5, 0], [9, 0]], device=device)[:, 0]  # strided
    for view in (big[:, ::2, 16:96], big[..., ::2], big[..., 3:83], big.transpose(0, 1), big[0, 0, :33], big[:, :, 1:34]):
        want = aclnn.dropout(view.contiguous(), state, 0.3)
        assert torch.equal(aclnn.dropout(view, state, 0.3), want)
        out = torch.full((*view.shape[:-1], 240), 7.0, dtype=view.dtype, device=device)
        aclnn.dropout(view, state, 0.3, out=out[..., 1:1 + view.shape[-1]])
        assert torch.equal(out[..., 1:1 + view.shape[-1]], want) and (out[..., 0] == 7).all()
        assert (out[..., 1 + view.shape[-1]:] == 7).all()
    x, r = big[0].contiguous(), big[1].contiguous()
    want = aclnn.dropout(x, state, 0.3, r)
    for into in (0, 1):
        both = [x.clone(), r.clone()]
        aclnn.dropout(both[0], state, 0.3, both[1], out=both[into])
        assert torch.equal(both[into], want)
    # the gradient keeps what the forward call kept
    ones = torch.ones_like(x)
    kept = aclnn.dropout(ones, state, 0.3) != 0
    assert torch.equal(aclnn.dropout(r, state, 0.3), torch.where(kept, aclnn.dropout(r, state, 0.0).float() * np.float32(
        65536 / (65536 - round(0.3 * 65536))), 0.0).to(x.dtype))
    assert 0.6 < kept.float().mean().item() < 0.8  # 1440 numbers: 0.7 with a deviation of 0.012


def test_dropout_offsets_are_masks(device, aclnn):
    """A tenth is dropped, evenly over the places in a group of eight, and independently of the next offset's mask."""
    ones, n = torch.ones(1 << 20, device=device), 1 << 20
    state = torch.tensor([11, 0], device=device)
    first = aclnn.dropout(ones, state, 0.1) == 0
    state[1] += 1
    second = aclnn.dropout(ones, state, 0.1) == 0
    sigma = math.sqrt(0.09 / n)
    for share, want, s in ((first, 0.1, sigma), (second, 0.1, sigma), (first & second, 0.01, math.sqrt(0.0099 / n))):
        assert abs(share.float().mean().item() - want) < 6 * s
    for i in range(8):
        assert abs(first[i::8].float().mean().item() - 0.1) < 6 * sigma * math.sqrt(8)


# ------------------------------------------------------------------------------------------------- gated projections

# rows, width, inner: one, a part of a tile, tiles and their edges, terms that end inside a stage, odd numbers
GATED = [(1, 1, 1), (1, 64, 64), (3, 8, 5), (7, 100, 33), (16, 512, 96), (17, 520, 130), (33, 64, 200), (64, 1000, 64),
         (128, 128, 64), (129, 136, 65), (200, 320, 300), (257, 72, 257), (1, 4096, 1024), (8, 1024, 2049), (300, 2048, 512)]


def gated_operands(g, rows, width, inner, dtype):
    x = rand(g, rows, width, dtype=dtype)
    wg, wu = (rand(g, inner, width, dtype=dtype, scale=width ** -0.5) for _ in range(2))
    return x, wg, wu, rand(g, inner, dtype=dtype), rand(g, inner, dtype=dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width,inner", GATED)
def test_gated(device, aclnn, dtype, rows, width, inner):
    g = gen("gated", dtype, rows, width, inner)
    x, wg, wu, bg, bu = gated_operands(g, rows, width, inner, dtype)
    kind = (rows + width + inner) % 3
    for biases in ((None, None), (bg, bu)):
        want, off = B.gated(x, wg, wu, *biases, kind)
        got = aclnn.gated_projection(*on(device, x, wg, wu, *biases), activation=kind, need_sums=True)
        for t, w, e, what in zip(got, want, off, ("y", "gate", "up")):
            close(t, w, e, dtype, what)
        alone = aclnn.gated_projection(*on(device, x, wg, wu, *biases), activation=kind)
        assert torch.equal(alone[0], got[0]) and alone[1] is None and alone[2] is None


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("rows,width,inner", [(700, 384, 512), (520, 200, 2100)])
def test_gated_large_tiles(device, aclnn, dtype, kind, rows, width, inner):
    """As many rows and features as give every CU a tile of 256 where a CU is one of a few."""
    g = gen("large", dtype, kind, rows)
    x, wg, wu, bg, bu = gated_operands(g, rows, width, inner, dtype)
    want, off = B.gated(x, wg, wu, bg, bu, kind)
    got = aclnn.gated_projection(*on(device, x, wg, wu, bg, bu), activation=kind, need_sums=True)
    for t, w, e, what in zip(got, want, off, ("y", "gate", "up")):
        close(t, w, e, dtype, what)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width,inner", GATED + [(5000, 64, 32), (40, 64, 2000), (1030, 40, 264)])
def test_gated_gradients(device, aclnn, dtype, rows, width, inner):
    g = gen("gated gradients", dtype, rows, width, inner)
    x, wg, wu, _, _ = gated_operands(g, rows, width, inner, dtype)
    gate, up, gy = (rand(g, rows, inner, dtype=dtype) for _ in range(3))
    kind = (rows + width + inner) % 3
    want, off = B.gated_grad(gy, x, wg, wu, gate, up, kind, dtype)
    dev = on(device, gy, x, wg, wu, gate, up)
    # which gradients are wanted decides how the sums are split: the bounds hold for any order of them
    for need_x, need_weights, need_bias in ((True, True, True), (True, False, False), (False, True, False), (False, False, True),
                                            (True, True, False)):
        got = aclnn.gated_projection_backward(*dev, activation=kind, need_x=need_x, need_weights=need_weights,
                                              need_bias=need_bias)
        assert [t is not None for t in got] == [need_x, need_weights, need_weights, need_bias, need_bias]
        for t, w, e, what in zip(got, want, off, ("x", "gate weight", "up weight", "gate bias", "up bias")):
            if t is not None:
                close(t, w, e, dtype, "gradient of the " + what)


@pytest.mark.parametrize("kind", [0, 1, 2])
def test_gated_gradients_against_differences(device, aclnn, kind):
    g = gen("gated differences", kind)
    parts = list(gated_operands(g, 21, 40, 50, "fp32"))
    gy = rand(g, 21, 50, dtype="fp32")
    _, gate, up = aclnn.gated_projection(*on(device, *parts), activation=kind, need_sums=True)
    grads = aclnn.gated_projection_backward(*on(device, gy, *parts[:3]), gate, up, activation=kind, need_bias=True)
    step = 1e-4
    for i, grad in enumerate(grads):
        e = rand(g, *grad.shape, dtype="fp32").double()
        ahead, back = [[t.double() + (s * step * e if i == j else 0) for j, t in enumerate(parts)] for s in (1, -1)]
        slope = sum(s * (B.gated(*v, kind)[0][0] * gy.double()).sum() for s, v in ((1, ahead), (-1, back))) / (2 * step)
        terms = grad.cpu().double() * e
        # second-order differences leave step^2 of the third derivative, 32-bit results F32 of the terms
        assert abs(slope - terms.sum()) <= 2e-5 * terms.abs().sum()


@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_views(device, aclnn, dtype):
    """Rows apart, rows that do not start on 16 bytes, columns, outputs inside larger tensors: as dense ones."""
    g = gen("gated views", dtype)
    x, wg, wu, bg, bu = on(device, *gated_operands(g, 60, 96, 72, dtype))
    want = aclnn.gated_projection(x, wg, wu, bg, bu, need_sums=True)
    gy = rand(g, 60, 72, dtype=dtype).to(device)
    grads = aclnn.gated_projection_backward(gy, x, wg, wu, *want[1:], need_bias=True)

    def apart(t, lead, width):
        big = torch.full((*t.shape[:-1], width), math.nan, dtype=t.dtype, device=device)
        big[..., lead:lead + t.shape[-1]] = t
        return big[..., lead:lead + t.shape[-1]]
    for how in (lambda t: apart(t, 0, t.shape[-1] + 16), lambda t: apart(t, 3, t.shape[-1] + 5), lambda t: apart(t, 8, 131),
                lambda t: t.t().contiguous().t() if t.dim() == 2 else t):
        v = [how(t) for t in (x, wg, wu)] + [apart(t[:, None].contiguous(), 1, 3)[:, 0] for t in (bg, bu)]
        outs = [how(torch.zeros_like(t)) for t in want]
        got = aclnn.gated_projection(*v, need_sums=True, out=outs[0], gate_out=outs[1], up_out=outs[2])
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        into = [how(torch.zeros_like(t)) for t in grads[:3]] + [apart(t[:, None].contiguous(), 1, 3)[:, 0] for t in grads[3:]]
        back = aclnn.gated_projection_backward(how(gy), *v[:3], how(want[1]), how(want[2]), need_bias=True, grad_x=into[0],
                                               grad_gate_weight=into[1], grad_up_weight=into[2], grad_gate_bias=into[3],
                                               grad_up_bias=into[4])
        assert all(torch.equal(p, q) for p, q in zip(back, grads))
    deep = aclnn.gated_projection(x.view(3, 5, 2, 2, 96), wg, wu, bg, bu)[0]
    assert torch.equal(deep.view(60, 72), want[0])
    one = aclnn.gated_projection(x[7], wg, wu, bg, bu)[0]
    close(one, B.gated(x[7:8].cpu(), wg.cpu(), wu.cpu(), bg.cpu(), bu.cpu(), 0)[0][0][0],
          B.gated(x[7:8].cpu(), wg.cpu(), wu.cpu(), bg.cpu(), bu.cpu(), 0)[1][0][0], dtype, "one row")
    # both weights in one tensor, one behind the other, and row by row in turn
    both = torch.cat([wg, wu])
    assert torch.equal(aclnn.gated_projection(x, both[:72], both[72:], bg, bu)[0], want[0])
    turns = torch.stack([wg, wu], 1)
    assert torch.equal(aclnn.gated_projection(x, turns[:, 0], turns[:, 1], bg, bu)[0], want[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_outside_stays(device, aclnn, dtype):
    """What lies around outputs and behind the last row stays, for sizes that end inside a tile."""
    g = gen("outside", dtype)
    for rows, width, inner in ((5, 40, 37), (130, 72, 70), (260, 64, 136)):
        x, wg, wu, _, _ = on(device, *gated_operands(g, rows, width, inner, dtype))
        outs = [torch.full((rows + 9, inner + 11), 7.0, dtype=x.dtype, device=device) for _ in range(3)]
        views = [t[4:4 + rows, 5:5 + inner] for t in outs]
        want = aclnn.gated_projection(x, wg, wu, need_sums=True)
        aclnn.gated_projection(x, wg, wu, need_sums=True, out=views[0], gate_out=views[1], up_out=views[2])
        for t, v, w in zip(outs, views, want):
            assert torch.equal(v, w)
            v.fill_(7)
            assert (t == 7).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_rows_that_are_not_finite(device, aclnn, dtype):
    """They stay in their rows, and what a weight's row holds in its feature."""
    g = gen("gated not finite", dtype)
    x, wg, wu, _, _ = gated_operands(g, 150, 88, 90, dtype)
    clean = aclnn.gated_projection(*on(device, x, wg, wu))[0]
    x[11, 87], x[149, 3], wu[40, 5] = math.nan, math.inf, math.nan
    got = aclnn.gated_projection(*on(device, x, wg, wu))[0]
    rows = torch.ones(150, dtype=torch.bool)
    rows[[11, 149]] = False
    columns = torch.ones(90, dtype=torch.bool)
    columns[40] = False
    assert torch.equal(got.cpu()[rows][:, columns], clean.cpu()[rows][:, columns])
    assert got[11].isnan().all() and got[:, 40].isnan().all() and not got[149].isfinite().any()


def test_gated_gradients_fp16_range(device, aclnn):
    """Gradients that FLOAT16 does not hold between the products, in rows of every size: the results have their bits."""
    g = gen("range")
    rows, width, inner = 96, 64, 80
    x, wg, wu, _, _ = gated_operands(g, rows, width, inner, "fp16")
    gate, up = rand(g, rows, inner, dtype="fp16"), rand(g, rows, inner, dtype="fp16")
    for low, high in ((2.0 ** -14, 2.0 ** -10), (2.0 ** -6, 2.0 ** 13)):
        size = torch.exp2(torch.linspace(math.log2(low), math.log2(high), rows, dtype=torch.float64))[:, None]
        gy = (torch.randn(rows, inner, generator=g, dtype=torch.float64) * size).half()
        u = (up.double() * (2.0 ** -6 if low < 1e-3 else 2.0 ** 6)).half()
        w = ((wg.double() * (2.0 ** 8 if low < 1e-3 else 2.0 ** -12)).half(), (wu.double() * (2.0 ** 8 if low < 1e-3 else 2.0 ** -12)).half())
        xs = (x.double() * (2.0 ** 8 if low < 1e-3 else 2.0 ** -12)).half()
        want, off = B.gated_grad(gy, xs, *w, gate, u, 0, "fp16")
        got = aclnn.gated_projection_backward(*on(device, gy, xs, *w, gate, u), need_bias=True)
        for i, what in ((0, "x"), (1, "gate weight"), (2, "up weight")):
            assert want[i].abs().max() < 65000
            close(got[i], want[i], off[i], "fp16", "gradient of the " + what)


@pytest.mark.parametrize("kind", [0, 1, 2])
def test_gated_far_gates(device, aclnn, kind):
    """Gates at the ends of the range: the activation is 0 or the gate, its slope 0 or 1, and nothing becomes NaN."""
    gates = torch.tensor([-3e38, -1e30, -1e5, -200.0, -20.0, 0.0, 20.0, 200.0, 1e5, 1e30, 3e38])
    n = len(gates)
    x = torch.eye(n)
    wg, wu = torch.diag(gates).t().contiguous(), torch.full((n, n), 0.5)
    y, gate, up = aclnn.gated_projection(*on(device, x, wg, wu), activation=kind, need_sums=True)
    diagonal = y.cpu().diagonal().double()
    # -20 times sigmoid(-20) or less
    B.within(diagonal, torch.where(gates > 0, 0.5 * gates, 0.0).double(), 2.1e-8 + B.F32 * gates.double().clamp(min=0), "far gates")
    sums = torch.diag(gates)
    grads = aclnn.gated_projection_backward(*on(device, torch.eye(n), x, torch.zeros(n, n), torch.zeros(n, n), sums, torch.ones(n, n)),
                                            activation=kind, need_x=False, need_weights=False, need_bias=True)
    slope = torch.where(gates > 0, 1.0, torch.where(gates == 0, 0.5, 0.0)).double()
    B.within(grads[3], slope, 1e-7, "slopes")
    B.within(grads[4], torch.where(gates > 0, gates, 0.0).double(), 4.2e-8 + B.F32 * gates.double().clamp(min=0), "values")


def test_gated_no_rows(device, aclnn):
    x = torch.empty(0, 64, device=device, dtype=torch.bfloat16)
    w = torch.ones(40, 64, device=device, dtype=torch.bfloat16)
    y, gate, up = aclnn.gated_projection(x, w, w, need_sums=True)
    assert y.shape == gate.shape == (0, 40)
    gx, gg, gu, bg, bu = aclnn.gated_projection_backward(y, x, w, w, gate, up, need_bias=True)
    assert gx.shape == x.shape and all((t == 0).all() for t in (gg, gu, bg, bu)) and gg.shape == (40, 64)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_the_same_from_call_to_call(device, aclnn, dtype):
    g = gen("again", dtype)
    x, wg, wu, _, _ = on(device, *gated_operands(g, 333, 520, 700, dtype))
    y, gate, up = aclnn.gated_projection(x, wg, wu, need_sums=True)
    first = aclnn.gated_projection_backward(y, x, wg, wu, gate, up, need_bias=True)
    for _ in range(5):
        assert torch.equal(aclnn.gated_projection(x, wg, wu)[0], y)
        assert all(torch.equal(p, q) for p, q in zip(aclnn.gated_projection_backward(y, x, wg, wu, gate, up, need_bias=True), first))
