"""The operators on token sequences against plain implementations in 64 bits (token_oracle.py)."""
import math

import numpy as np
import pytest
import torch

import token_oracle as O

pytestmark = pytest.mark.gpu


def rand(g, *size, dtype, scale=1.0):
    return (torch.randn(*size, generator=g, dtype=torch.float64) * scale).to(O.DTYPES[dtype])


def gen(*key):
    return torch.Generator().manual_seed(sum((i + 1) * ord(c) for i, c in enumerate(str(key))))


# ------------------------------------------------------------------------------------------------------------- norm

NORM_SIZES = [(1, 1), (3, 5), (4, 64), (7, 100), (2, 768), (130, 1024), (5, 1001), (3, 2056), (2, 4096), (3, 8192), (2, 9001),
              (2, 40000), (2, 33001)]


@pytest.mark.parametrize("dtype", O.DTYPES)
@pytest.mark.parametrize("rows,width", NORM_SIZES)
def test_norm(device, aclnn, dtype, rows, width):
    g = gen("norm", dtype, rows, width)
    x, r = rand(g, rows, width, dtype=dtype), rand(g, rows, width, dtype=dtype, scale=3)
    w = rand(g, width, dtype=dtype)
    u = O.U[dtype]
    for residual in (None, r):
        y, h, rstd = O.norm(x, residual, w, 1e-6)
        got, total, got_rstd = aclnn.residual_norm(x.to(device), w.to(device), None if residual is None else r.to(device),
                                                   eps=1e-6, need_rstd=True)
        O.within(got, y, (u + O.F32) * y.abs() + O.TINY[dtype], "norm")
        O.within(got_rstd, rstd, O.F32 * rstd, "rstd")
        assert (total is None) == (residual is None)
        if residual is not None:
            assert torch.equal(total.cpu(), (x.float() + r.float()).to(x.dtype))
        q, scale, _, _ = aclnn.residual_norm_int8(x.to(device), w.to(device), None if residual is None else r.to(device),
                                                  eps=1e-6)
        want, most = O.norm_int8(x, residual, w)
        assert np.array_equal(q.cpu().numpy(), want)
        O.within(scale, torch.from_numpy(most).double() * rstd / 127, O.F32 * torch.from_numpy(most).double() * rstd, "scale")


@pytest.mark.parametrize("dtype", O.DTYPES)
@pytest.mark.parametrize("rows,width", NORM_SIZES + [(3000, 96), (700, 2048), (1100, 7)])
def test_norm_gradients(device, aclnn, dtype, rows, width):
    g = gen("norm_grad", dtype, rows, width)
    h, gy, gs = (rand(g, rows, width, dtype=dtype) for _ in range(3))
    w = rand(g, width, dtype=dtype)
    rstd = (1 / torch.sqrt(h.double().square().mean(-1) + 1e-6)).float()
    u = O.U[dtype]
    for grad_sum in (None, gs):
        gx, gw = O.norm_grad(gy, grad_sum, h, w, rstd)
        dev = [t.to(device) for t in (gy, h, w, rstd)]
        got_x, got_w = aclnn.residual_norm_backward(*dev, grad_sum=None if grad_sum is None else gs.to(device))
        n = h.double().abs() * rstd.double()[:, None]
        gn = (gy.double() * w.double()).abs()
        slack = O.F32 * ((gn + n * (gn * n).mean(-1, keepdim=True)) * rstd.double()[:, None] + (0 if grad_sum is None else gs.double().abs()))
        O.within(got_x, gx, u * gx.abs() + slack + O.TINY[dtype], "gradient of x")
        O.within(got_w, gw, u * gw.abs() + O.F32 * (gy.double().abs() * n).sum(0) + O.TINY[dtype], "gradient of the weight")
        only_x, none = aclnn.residual_norm_backward(*dev, grad_sum=None if grad_sum is None else gs.to(device),
                                                    need_weight=False)
        assert none is None and torch.equal(only_x, got_x)


def test_norm_gradient_against_differences(device, aclnn):
    g = gen("norm differences")
    x, r, w = rand(g, 5, 300, dtype="fp32"), rand(g, 5, 300, dtype="fp32"), rand(g, 300, dtype="fp32")
    gy, gs = rand(g, 5, 300, dtype="fp32"), rand(g, 5, 300, dtype="fp32")
    y, total, rstd = aclnn.residual_norm(x.to(device), w.to(device), r.to(device), need_rstd=True)
    gx, gw = aclnn.residual_norm_backward(gy.to(device), total, w.to(device), rstd, grad_sum=gs.to(device))

    def value(x, w):
        y, h, _ = O.norm(x, r, w, 1e-6)
        return (y * gy.double()).sum() + (h * gs.double()).sum()
    step, e = 1e-4, rand(g, 5, 300, dtype="fp32").double()
    slope = (value(x.double() + step * e, w) - value(x.double() - step * e, w)) / (2 * step)
    along = (gx.cpu().double() * e).sum()
    # second-order differences leave step^2 of the third derivative, 32-bit results F32 of the terms
    assert abs(slope - along) <= 1e-5 * (gx.cpu().double() * e).abs().sum()
    f = rand(g, 300, dtype="fp32").double()
    slope = (value(x, w.double() + step * f) - value(x, w.double() - step * f)) / (2 * step)
    assert abs(slope - (gw.cpu().double() * f).sum()) <= 1e-5 * (gw.cpu().double() * f).abs().sum()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_norm_float_weight(device, aclnn, dtype):
    g = gen("weight", dtype)
    x, w = rand(g, 6, 520, dtype=dtype), rand(g, 520, dtype="fp32")
    y, h, rstd = O.norm(x, None, w, 1e-5)
    got, _, r = aclnn.residual_norm(x.to(device), w.to(device), eps=1e-5, need_rstd=True)
    O.within(got, y, (O.U[dtype] + O.F32) * y.abs() + O.TINY[dtype], "norm")
    gy = rand(g, 6, 520, dtype=dtype)
    gx, gw = aclnn.residual_norm_backward(gy.to(device), x.to(device), w.to(device), r)
    want_x, want_w = O.norm_grad(gy, None, x, w, rstd.float())
    assert gw.dtype == torch.float32
    O.within(gw, want_w, O.F32 * (gy.double() * x.double() * rstd[:, None]).abs().sum(0), "gradient of the weight")
    q, scale, _, _ = aclnn.residual_norm_int8(x.to(device), w.to(device), eps=1e-5)
    assert np.array_equal(q.cpu().numpy(), O.norm_int8(x, None, w)[0])


@pytest.mark.parametrize("dtype", O.DTYPES)
def test_norm_views_and_in_place(device, aclnn, dtype):
    g = gen("norm views", dtype)
    big = rand(g, 3, 9, 4, 160, dtype=dtype).to(device)
    w = rand(g, 80, dtype=dtype).to(device)
    for view in (big[:, ::2, :, 16:96], big[..., ::2], big[:, :, 1, 3:83], big.transpose(1, 2)[..., :80], big[:1, :, :, 80:],
                 big[0, 0, 0, :80], big[:, :1, :1, 1:81].expand(3, 5, 2, 80)):
        plain = view.contiguous()
        y, _, rstd = aclnn.residual_norm(view, w, need_rstd=True)
        py, _, prstd = aclnn.residual_norm(plain, w, need_rstd=True)
        assert torch.equal(y, py) and torch.equal(rstd, prstd)
        q, s, _, _ = aclnn.residual_norm_int8(view, w)
        pq, ps, _, _ = aclnn.residual_norm_int8(plain, w)
        assert torch.equal(q, pq) and torch.equal(s, ps)
    # outputs into windows of larger buffers leave the rest alone
    x, r = big[:, :, 0, :80], big[:, :, 1, :80]
    y, total, _ = aclnn.residual_norm(x, w, r)
    room = torch.full((3, 9, 100), 7.0, dtype=x.dtype, device=device)
    q_room = torch.full((3, 9, 200), 9, dtype=torch.int8, device=device)
    aclnn.residual_norm(x, w, r, out=room[..., 10:90])
    assert torch.equal(room[..., 10:90], y) and (room[..., :10] == 7).all() and (room[..., 90:] == 7).all()
    aclnn.residual_norm_int8(x, w, r, out=q_room[..., ::2][..., 3:83])
    assert torch.equal(q_room[..., ::2][..., 3:83], aclnn.residual_norm_int8(x, w, r)[0]) and (q_room[..., 1::2] == 9).all()
    # the sum over x, and over the residual
    for place in (0, 1):
        a, b = x.contiguous(), r.contiguous()
        y2, t2, _ = aclnn.residual_norm(a, w, b, sum_out=(a, b)[place])
        assert torch.equal(y2, y) and torch.equal(t2, total) and t2.data_ptr() == (a, b)[place].data_ptr()
    # gradients over gradients
    gy, gs = rand(g, 3, 9, 80, dtype=dtype).to(device), rand(g, 3, 9, 80, dtype=dtype).to(device)
    rstd = aclnn.residual_norm(x, w, r, need_rstd=True)[2]
    gx, gw = aclnn.residual_norm_backward(gy, total, w, rstd, grad_sum=gs)
    for place in (0, 1):
        a, b = gy.clone(), gs.clone()
        gx2, gw2 = aclnn.residual_norm_backward(a, total, w, rstd, grad_sum=b, grad_x=(a, b)[place])
        assert torch.equal(gx2, gx) and torch.equal(gw2, gw)


def test_norm_long_rows_in_place(device, aclnn):
    g = gen("long")
    x, r, w = (rand(g, 2, 40000, dtype="bf16").to(device), rand(g, 2, 40000, dtype="bf16").to(device),
               rand(g, 40000, dtype="bf16").to(device))
    y, total, rstd = aclnn.residual_norm(x, w, r, need_rstd=True)
    a = x.clone()
    y2, t2, _ = aclnn.residual_norm(a, w, r, sum_out=a)
    assert torch.equal(y2, y) and torch.equal(t2, total)
    gy = rand(g, 2, 40000, dtype="bf16").to(device)
    gx, gw = aclnn.residual_norm_backward(gy, total, w, rstd)
    b = gy.clone()
    gx2, gw2 = aclnn.residual_norm_backward(b, total, w, rstd, grad_x=b)
    assert torch.equal(gx2, gx) and torch.equal(gw2, gw)


def test_norm_special_rows(device, aclnn):
    x = torch.ones(5, 256)
    x[1], x[2, 3], x[3, 200], x[4] = 0, math.inf, math.nan, 1e-30
    w = torch.ones(256)
    q, scale, _, _ = aclnn.residual_norm_int8(x.to(device), w.to(device))
    q, scale = q.cpu(), scale.cpu()
    assert (q[0] == 127).all() and (q[1:4] == 0).all() and (q[4] == 127).all()
    assert scale[1] == 0 and scale[2].isnan() and scale[3].isnan() and scale[4] > 0
    y, _, _ = aclnn.residual_norm(x.to(device), w.to(device))
    assert y[0].isfinite().all() and (y[1] == 0).all() and y[3].isnan().all() and y[4].isfinite().all()
    empty, _, _ = aclnn.residual_norm(x.to(device)[:0], w.to(device))
    assert empty.shape == (0, 256)
    _, gw = aclnn.residual_norm_backward(x.to(device)[:0], x.to(device)[:0], w.to(device), torch.empty(0, device=device))
    assert (gw == 0).all()


# ----------------------------------------------------------------------------------------------------------- rotary

@pytest.mark.parametrize("rot,kw", [(2, {}), (64, {}), (128, dict(base=500000.0)), (64, dict(scaling=1, factor=4.0)),
                                    (64, dict(scaling=2, factor=8.0)), (1024, dict(magnitude=1.25)),
                                    (64, dict(scaling=3, factor=4.0, original_length=2048, magnitude=1.139))])
def test_rotary_table(device, aclnn, rot, kw):
    like = torch.empty(0, device=device)
    want = O.rotary_table(1000, rot, **kw)
    got = aclnn.rotary_table(like, 1000, rot, **kw)
    O.within(got, want, 2.0 ** -24 * want.abs() + 1e-12, "table")
    wide = torch.zeros(1000, rot + 6, device=device)
    aclnn.rotary_table(like, 1000, rot, out=wide[:, 3:3 + rot], **kw)
    assert torch.equal(wide[:, 3:3 + rot], got) and (wide[:, :3] == 0).all() and (wide[:, 3 + rot:] == 0).all()


def test_rotary_table_far_positions(device, aclnn):
    got = aclnn.rotary_table(torch.empty(0, device=device), 1 << 18, 16)
    want = O.rotary_table(1 << 18, 16)
    O.within(got, want, 2.0 ** -24 * want.abs() + 1e-9, "table")  # the last positions' angles have 2^-35 of 64-bit error


ROTARY = [(1, 1, 1, 1, 2, 2), (2, 3, 4, 2, 64, 64), (1, 7, 3, 1, 80, 40), (2, 5, 2, 2, 72, 36), (3, 2, 5, 0, 33, 10), (1, 4, 9, 3, 128, 128),
          (1, 600, 12, 4, 128, 64), (2, 1, 40, 8, 96, 24), (1, 3, 2, 1, 1000, 999 // 2 * 2), (1, 5, 1, 1, 7, 6)]


@pytest.mark.parametrize("dtype", O.DTYPES)
@pytest.mark.parametrize("b,s,heads,kv_heads,d,rot", ROTARY)
def test_rotary(device, aclnn, dtype, b, s, heads, kv_heads, d, rot):
    g = gen("rotary", dtype, b, s, heads, d, rot)
    q = rand(g, b, s, heads, d, dtype=dtype)
    k = rand(g, b, s, kv_heads, d, dtype=dtype) if kv_heads else None
    table = O.rotary_table(700, rot).float()
    positions = torch.randint(0, 700, (b, s), generator=g)
    dev = [None if t is None else t.to(device) for t in (q, k, table)]
    for interleaved in (False, True):
        for inverse in (False, True):
            for at in (None, positions, positions.int()):
                want_at = torch.arange(s).expand(b, s) if at is None else positions
                got = aclnn.rotary(*dev, positions=None if at is None else at.to(device), interleaved=interleaved,
                                   inverse=inverse)
                for x, y in zip((q, k), got):
                    if x is None:
                        assert y is None
                        continue
                    want = O.rotary(x, table, want_at, interleaved, inverse)
                    size = O.rotary_size(x, table, want_at, interleaved)
                    O.within(y, want, O.U[dtype] * want.abs() + 2.0 ** -22 * size + 2.0 ** -22 * want.abs() + O.TINY[dtype], "rotary")
                    assert torch.equal(y[..., rot:].cpu(), x[..., rot:])


def test_rotary_there_and_back(device, aclnn):
    g = gen("back")
    q = rand(g, 2, 50, 6, 64, dtype="fp32").to(device)
    table = aclnn.rotary_table(q, 50, 64)
    there, none = aclnn.rotary(q, None, table)
    back, _ = aclnn.rotary(there, None, table, inverse=True)
    assert none is None
    O.within(back, q.cpu(), 1e-5, "there and back")
    # the gradient's way: <R x, y> = <x, R' y>
    y = rand(g, 2, 50, 6, 64, dtype="fp32").to(device)
    home, _ = aclnn.rotary(y, None, table, inverse=True)
    a, b = (there.double() * y.double()).sum(), (q.double() * home.double()).sum()
    assert abs(a - b) <= 1e-5 * (there.double() * y.double()).abs().sum()


@pytest.mark.parametrize("dtype", O.DTYPES)
def test_rotary_views_places_and_bad_positions(device, aclnn, dtype):
    g = gen("rotary views", dtype)
    fused = rand(g, 2, 9, 10, 48, dtype=dtype).to(device)  # queries, keys and values of one product
    table = O.rotary_table(64, 32).float().to(device)
    q, k = fused[:, :, :6], fused[:, :, 6:8]
    for interleaved in (False, True):
        want = aclnn.rotary(q.contiguous(), k.contiguous(), table, interleaved=interleaved)
        for a, b in ((q, k), (q.transpose(1, 2).contiguous().transpose(1, 2), k), (fused[..., :6, :].flip(3).contiguous().flip(3), k)):
            got = aclnn.rotary(a, b, table, interleaved=interleaved)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        every = fused.clone()
        aclnn.rotary(every[:, :, :6], every[:, :, 6:8], table, interleaved=interleaved, query_out=every[:, :, :6],
                     key_out=every[:, :, 6:8])
        assert torch.equal(every[:, :, :6], want[0]) and torch.equal(every[:, :, 6:8], want[1])
        assert torch.equal(every[:, :, 8:], fused[:, :, 8:])
        odd = torch.zeros(2, 9, 6, 49, dtype=fused.dtype, device=device)  # rows that start on odd elements
        odd[..., 1:] = q
        cache = torch.full((2, 30, 2, 48), 5.0, dtype=fused.dtype, device=device)
        got = aclnn.rotary(odd[..., 1:], k, table, interleaved=interleaved, key_out=cache[:, 11:20])
        assert torch.equal(got[0], want[0]) and torch.equal(cache[:, 11:20], want[1])
        assert (cache[:, :11] == 5).all() and (cache[:, 20:] == 5).all()
        sparse = torch.zeros(2, 9, 6, 96, dtype=fused.dtype, device=device)
        sparse[..., ::2] = q  # a last dimension with gaps is packed
        assert torch.equal(aclnn.rotary(sparse[..., ::2], k, table, interleaved=interleaved)[0], want[0])
        positions = torch.zeros(2, 18, dtype=torch.int64, device=device)
        positions[0, 6], positions[1, 2], positions[1, 4] = 64, -1, 2 ** 40
        got = aclnn.rotary(q, k, table, positions=positions[:, ::2], interleaved=interleaved)
        bad = torch.zeros(2, 9, dtype=torch.bool, device=device)
        bad[0, 3] = bad[1, 1] = bad[1, 2] = True
        for y, x in zip(got, (q, k)):
            assert y[bad][..., :32].isnan().all() and torch.equal(y[..., 32:], x[..., 32:]) and y[~bad].isfinite().all()


# -------------------------------------------------------------------------------------------------------- attention

NONE = 2 ** 63 - 1
#        b  sq   skv  heads kv d    left  right sinks lengths
ATTENTION = [
    (1, 1, 1, 1, 1, 8, NONE, 0, 0, None),
    (2, 1, 77, 4, 2, 64, NONE, 0, 0, ([1, 1], [77, 1])),
    (2, 1, 500, 8, 1, 128, 100, 0, 4, ([1, 1], [500, 33])),
    (3, 1, 2100, 8, 2, 128, NONE, 0, 0, ([1, 1, 1], [2100, 0, 1024])),
    (2, 4, 700, 8, 1, 80, 63, 0, 70, ([4, 2], [700, 130])),
    (1, 5, 300, 6, 2, 72, 40, 0, 3, None),
    (1, 33, 33, 2, 2, 64, NONE, 0, 0, None),
    (2, 100, 100, 4, 2, 128, 31, 0, 4, ([100, 7], [100, 7])),
    (1, 130, 130, 3, 1, 96, 20, 15, 1, None),
    (2, 64, 200, 2, 1, 256, 50, 0, 16, ([64, 10], [200, 64])),
    (1, 37, 150, 2, 2, 40, NONE, NONE, 0, None),
    (1, 200, 90, 2, 1, 64, 30, 0, 5, None),           # more queries than keys: the first see nothing
    (2, 70, 70, 4, 4, 33, 16, 3, 2, ([70, 0], [70, 70])),  # odd head size, a sequence without queries
    (2, 20, 50, 2, 1, 1, 5, 0, 1, ([20, 20], [0, 50])),    # a sequence without keys
    (1, 260, 260, 1, 1, 160, 0, 0, 0, None),               # every token sees itself alone
    (1, 150, 150, 2, 1, 128, 10, 0, 140, None),            # sinks past the windows
    (1, 300, 300, 12, 4, 64, 64, 64, 8, None),
    (2, 90, 1000, 2, 1, 200, NONE, 0, 0, ([90, 50], [1000, 51])),
]


def attention_case(case, dtype, seed="attention"):
    b, sq, skv, heads, kv_heads, d, left, right, sinks, lengths = case
    g = gen(seed, dtype, case)
    q, k, v = rand(g, b, sq, heads, d, dtype=dtype), rand(g, b, skv, kv_heads, d, dtype=dtype), rand(g, b, skv, kv_heads, d, dtype=dtype)
    masks = dict(scale=1.3 / math.sqrt(d), left=left, right=right, sinks=sinks)
    lens = dict(q_lens=None, kv_lens=None) if lengths is None else dict(q_lens=lengths[0], kv_lens=lengths[1])
    return g, q, k, v, masks, lens


def on_device(device, lens, wide=False):
    return {n: None if lens[o] is None else torch.tensor(lens[o], dtype=torch.int64 if wide else torch.int32, device=device)
            for n, o in (("q_lengths", "q_lens"), ("kv_lengths", "kv_lens"))}


@pytest.mark.parametrize("dtype", O.DTYPES)
@pytest.mark.parametrize("case", ATTENTION, ids=[str(i) for i in range(len(ATTENTION))])
def test_attention(device, aclnn, dtype, case):
    g, q, k, v, masks, lens = attention_case(case, dtype)
    r = O.attention(q, k, v, **masks, **lens)
    bound = O.attention_bounds(r, q, k, v, masks["scale"], dtype)
    out, lse = aclnn.window_attention(q.to(device), k.to(device), v.to(device), need_lse=True, **masks, **on_device(device, lens))
    O.within(out, r["out"], bound["out"], "out")
    O.within(lse, r["lse"], O.F32 * (1 + r["lse"].abs()), "lse")
    again, none = aclnn.window_attention(q.to(device), k.to(device), v.to(device), **masks, **on_device(device, lens, True))
    assert none is None and torch.equal(again, out)


@pytest.mark.parametrize("dtype", O.DTYPES)
@pytest.mark.parametrize("case", ATTENTION, ids=[str(i) for i in range(len(ATTENTION))])
def test_attention_gradients(device, aclnn, dtype, case):
    g, q, k, v, masks, lens = attention_case(case, dtype)
    go = rand(g, *q.shape, dtype=dtype, scale=0.01)
    r = O.attention(q, k, v, grad_out=go, **masks, **lens)
    bound = O.attention_bounds(r, q, k, v, masks["scale"], dtype, go)
    dev = [t.to(device) for t in (go, q, k, v, r["out"].to(q.dtype), r["lse"].float())]
    got = aclnn.window_attention_backward(*dev, **masks, **on_device(device, lens))
    for name, x in zip(("gq", "gk", "gv"), got):
        O.within(x, r[name], bound[name], name)
    again = aclnn.window_attention_backward(*dev, **masks, **on_device(device, lens, True))
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("case", [ATTENTION[7], ATTENTION[8], ATTENTION[12]])
def test_attention_gradients_against_differences(device, aclnn, case):
    g, q, k, v, masks, lens = attention_case(case, "fp32", "differences")
    go = rand(g, *q.shape, dtype="fp32")
    dev = [t.to(device) for t in (q, k, v)]
    on = on_device(device, lens)
    out, lse = aclnn.window_attention(*dev, need_lse=True, **masks, **on)
    grads = aclnn.window_attention_backward(go.to(device), *dev, out, lse, **masks, **on)
    step = 1e-4
    for i, grad in enumerate(grads):
        e = rand(g, *grad.shape, dtype="fp32").double()
        ends = []
        for sign in (1, -1):
            x = [t.double() for t in (q, k, v)]
            x[i] = x[i] + sign * step * e
            ends.append((O.attention(*x, **masks, **lens)["out"] * go.double()).sum())
        terms = grad.cpu().double() * e
        assert abs((ends[0] - ends[1]) / (2 * step) - terms.sum()) <= 1e-5 * terms.abs().sum()


@pytest.mark.parametrize("dtype", O.DTYPES)
def test_attention_views(device, aclnn, dtype):
    """Strides of fused products, of heads outside tokens, of broadcast keys, of gaps and odd starts: the same bits."""
    case = (2, 70, 70, 4, 2, 64, 20, 0, 3, ([70, 40], [70, 40]))
    g, q, k, v, masks, lens = attention_case(case, dtype)
    on = on_device(device, lens)
    q, k, v = (t.to(device) for t in (q, k, v))
    go = rand(g, *q.shape, dtype=dtype).to(device)
    out, lse = aclnn.window_attention(q, k, v, need_lse=True, **masks, **on)
    grads = aclnn.window_attention_backward(go, q, k, v, out, lse, **masks, **on)
    fused = torch.cat([q, k, v], 2)
    views = [lambda t: t.transpose(1, 2).contiguous().transpose(1, 2),
             lambda t: torch.nn.functional.pad(t, (8, 8))[..., 8:-8],
             lambda t: torch.nn.functional.pad(t, (1, 2))[..., 1:-2],
             lambda t: t.repeat_interleave(2, 3)[..., ::2],
             lambda t: t.transpose(0, 3).contiguous().transpose(0, 3)]
    made = [(fused[:, :, :4], fused[:, :, 4:6], fused[:, :, 6:])] + [tuple(f(t) for t in (q, k, v)) for f in views]
    for n, (a, b, c) in enumerate(made):
        view = views[n - 1] if n else (lambda t: t)
        o, le = torch.full_like(view(out), 3.0), torch.full((2, 70, 4, 2), 3.0, device=device)[..., 1].transpose(1, 2)
        aclnn.window_attention(a, b, c, out=o, lse=le, **masks, **on)
        # elements that are not in 16-byte groups go by another kernel, of the same products in the same order
        assert torch.equal(o, out) and torch.equal(le, lse), n
        to = [torch.full_like(view(t), 3.0) for t in (q, k, v)]
        got = aclnn.window_attention_backward(view(go), a, b, c, o, le, grad_query=to[0], grad_key=to[1], grad_value=to[2],
                                              **masks, **on)
        assert all(torch.equal(x, y) for x, y in zip(got, grads)), n
    one = k[:, :, :1].expand(2, 70, 2, 64)  # a broadcast key head
    a, _ = aclnn.window_attention(q, one, v, **masks, **on)
    b, _ = aclnn.window_attention(q, one.contiguous(), v, **masks, **on)
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", O.DTYPES)
@pytest.mark.parametrize("sq", [1, 60])
def test_attention_ignores_what_is_not_seen(device, aclnn, dtype, sq):
    """Keys and values past a sequence's length, and between the sinks and the windows of its queries, hold NaN and
    infinities; queries past its length too."""
    b, skv, heads, kv_heads, d = 2, 400, 4, 2, 64
    kv_lens, left, sinks = [300, 131], 40, 3
    g, q, k, v, masks, lens = attention_case((b, sq, skv, heads, kv_heads, d, left, 0, sinks, ([sq, max(1, sq - 5)], kv_lens)), dtype)
    go = rand(g, *q.shape, dtype=dtype)
    on = on_device(device, lens)
    clean = [t.to(device) for t in (q, k, v)]
    out, lse = aclnn.window_attention(*clean, need_lse=True, **masks, **on)
    grads = aclnn.window_attention_backward(go.to(device), *clean, out, lse, **masks, **on)
    for n in range(b):
        first = kv_lens[n] - lens["q_lens"][n] - left
        for t, bad in ((k, math.nan), (v, math.inf)):
            t[n, sinks:first] = bad
            t[n, kv_lens[n]:] = -bad
        q[n, lens["q_lens"][n]:] = math.nan
        go[n, lens["q_lens"][n]:] = math.nan
    dirty = [t.to(device) for t in (q, k, v)]
    o, le = aclnn.window_attention(*dirty, need_lse=True, **masks, **on)
    assert torch.equal(o, out) and torch.equal(le, lse)
    got = aclnn.window_attention_backward(go.to(device), *dirty, o, le, **masks, **on)
    assert all(torch.equal(x, y) for x, y in zip(got, grads))


@pytest.mark.parametrize("dtype", O.DTYPES)
def test_attention_special_values_reach_only_who_sees_them(device, aclnn, dtype):
    case = (1, 200, 200, 2, 1, 64, 30, 0, 2, None)
    g, q, k, v, masks, lens = attention_case(case, dtype)
    clean, _ = aclnn.window_attention(q.to(device), k.to(device), v.to(device), **masks)
    for bad in (math.nan, math.inf, -math.inf):
        w = v.clone()
        w[0, 100, 0, 5] = bad
        got, _ = aclnn.window_attention(q.to(device), k.to(device), w.to(device), **masks)
        hit = torch.zeros(200, 64, dtype=torch.bool, device=device)
        hit[100:131, 5] = True
        assert torch.equal(got[0][~hit[:, None].expand(200, 2, 64)], clean[0][~hit[:, None].expand(200, 2, 64)])
        reached = got[0][hit[:, None].expand(200, 2, 64)]
        assert reached.isnan().all() if bad != bad else (reached == bad).all()
    x = k.clone()
    x[0, 100] = math.nan
    got, _ = aclnn.window_attention(q.to(device), x.to(device), v.to(device), **masks)
    assert got[0, 100:131].isnan().all()
    assert torch.equal(got[0, :100], clean[0, :100]) and torch.equal(got[0, 131:], clean[0, 131:])


def test_attention_large_scores(device, aclnn):
    """Scores far past the range of exp: the maximum is taken out before."""
    case = (1, 90, 90, 2, 2, 64, NONE, 0, 0, None)
    g, q, k, v, masks, lens = attention_case(case, "fp32")
    masks["scale"] = 40.0
    r = O.attention(q, k, v, **masks)
    out, lse = aclnn.window_attention(q.to(device), k.to(device), v.to(device), need_lse=True, **masks)
    # a score of size s carries 2^-22 s of absolute error (two roundings and its sum), which is the weights' relative one
    size = 40.0 * float((q.double().norm(dim=-1).max() * k.double().norm(dim=-1).max()))
    O.within(out, r["out"], 2.0 ** -21 * size * float(v.abs().max()), "out")
    O.within(lse, r["lse"], 2.0 ** -21 * size, "lse")


def test_small_gradients_of_fp16(device, aclnn):
    """Gradients near the smallest numbers of FLOAT16 divided over a thousand keys keep their size."""
    case = (1, 1000, 1000, 2, 1, 64, NONE, 0, 0, None)
    g, q, k, v, masks, lens = attention_case(case, "fp16")
    masks["scale"] = 0.01
    go = rand(g, *q.shape, dtype="fp16", scale=2e-3)
    r = O.attention(q, k, v, grad_out=go, **masks)
    dev = [t.to(device) for t in (go, q, k, v, r["out"].half(), r["lse"].float())]
    got = aclnn.window_attention_backward(*dev, grad_query=torch.empty(q.shape, dtype=torch.float16, device=device), **masks)
    for name, x in zip(("gq", "gk", "gv"), got):
        err = (x.double().cpu() - r[name]).norm() / r[name].norm()
        # results of 1e-6 are rounded to steps of 6e-8, a tenth of their size at most; gv is of 1e-3
        assert err <= (0.05 if name != "gv" else 2e-3), (name, err)


def test_operators_on_another_stream(device, aclnn):
    g = gen("stream")
    x, w = rand(g, 300, 512, dtype="bf16").to(device), rand(g, 512, dtype="bf16").to(device)
    q = rand(g, 1, 300, 4, 64, dtype="bf16").to(device)
    want = aclnn.residual_norm(x, w)[0], aclnn.window_attention(q, q, q, left=50)[0]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = aclnn.residual_norm(x, w, stream=side)[0], aclnn.window_attention(q, q, q, left=50, stream=side)[0]
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
