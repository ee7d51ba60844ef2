"""FLOAT16 gradients of the gated projections whose rows, or inner columns, are up to 2^40 apart: more than one scale for all of
them holds, so those of each row and each column have to be there."""
import pytest
import torch

import block_oracle as B

ROWS, WIDTH, INNER = 96, 64, 160


def operands(by_rows):
    """dGate = gradY up slope and dUp = gradY gate, about: each of the three is 2^(k / 2) in a row (a column) of size 2^k, k from
    -12 to 28; gates are positive and at least a quarter of that.  Sums over what differs in size are past FLOAT16's range: of
    rows apart x's gradient is looked at, of columns apart those of the weights."""
    g = torch.Generator().manual_seed(5 + by_rows)
    k = torch.linspace(-6, 14, ROWS if by_rows else INNER, dtype=torch.float64)
    size = torch.exp2(k)[:, None] if by_rows else torch.exp2(k)

    def rand(*n):
        return torch.randn(*n, generator=g, dtype=torch.float64)
    signed = [rand(ROWS, INNER).clamp(-3, 3) for _ in range(2)]
    gate = 0.25 + rand(ROWS, INNER).abs().clamp(max=3)
    grad_y, up, gate = ((t * size).half() for t in (*signed, gate))
    return grad_y, rand(ROWS, WIDTH).half(), rand(INNER, WIDTH).half(), rand(INNER, WIDTH).half(), gate, up


def expected(by_rows, rounded=None):
    """(gradient of x, of gate's and of up's weight; bounds).  `rounded`: what dGate and dUp become before the products, in
    64 bits, instead.

    What the functions lose: the sigmoid s of a positive gate g is off by 2^-22 of itself; g (s (1 - s)) by 2^-22 g where
    g < 17 and nothing beyond, where 1 - s is 0 and belongs under 2^-24: the slope, at least a half, by 2^-16 of itself.  Then
    the rounding to eleven bits, or to 2^-39 of the largest of the row for x's, of the column for the weights' gradients: that is
    2^14 or more in its scale, and the smallest step of FLOAT16 is 2^-24."""
    grad_y, x, wg, wu, gate, up = (t.double() for t in operands(by_rows))
    act, slope = B.activation(gate, 0)
    both = torch.cat([grad_y * up * slope, grad_y * act], 1)
    w = torch.cat([wg, wu])
    a, b = (both, both) if rounded is None else (rounded(both, 1), rounded(both, 0))
    rel = 2.0 ** -16 + B.U["fp16"]
    off = [(rel + B.gamma(n)) * both.abs() + 2.0 ** -39 * both.abs().amax(d, keepdim=True) for d, n in ((1, 2 * INNER), (0, ROWS))]
    gw, ew = b.t() @ x, off[1].t() @ x.abs()
    return (a @ w, gw[:INNER], gw[INNER:]), (off[0] @ w.abs(), ew[:INNER], ew[INNER:])


def check(got, want, bound, what):
    """Where FLOAT16 holds the result: within the bound and its rounding; past its range: infinite."""
    got, off = got.double().cpu(), bound + B.U["fp16"] * want.abs() + B.TINY["fp16"]
    held, past = want.abs() + off < 65504, want.abs() - off > 65520
    assert held.any(1).sum() > len(want) / 2
    B.within(got[held], want[held], off[held], what)
    assert (got[past] == torch.sign(want[past]) * torch.inf).all(), what


@pytest.mark.gpu
@pytest.mark.parametrize("by_rows", [True, False])
def test_rows_and_columns_of_every_size(device, aclnn, by_rows):
    want, off = expected(by_rows)
    dev = [t.to(device) for t in operands(by_rows)]
    for need_x, need_weights in ((True, True), (True, False), (False, True)):
        got = aclnn.gated_projection_backward(*dev, need_x=need_x, need_weights=need_weights)
        for i in (0,) if by_rows else (1, 2):
            if got[i] is not None:
                check(got[i], want[i], off[i], "gradient %d" % i)


def scaled(x, most):
    """Rounded to FLOAT16 in the scale that takes `most` to 2^14 and more."""
    s = torch.exp2(14 - torch.floor(torch.log2(most)))
    return (x * s).half().double() / s


@pytest.mark.parametrize("by_rows", [True, False])
def test_one_scale_would_not_do(by_rows):
    """The bounds hold for scales of rows and columns, and not for one scale of all."""
    want, off = expected(by_rows)
    own, _ = expected(by_rows, lambda t, d: scaled(t, t.abs().amax(d, keepdim=True)))
    one, _ = expected(by_rows, lambda t, d: scaled(t, t.abs().max()))
    for i in (0,) if by_rows else (1, 2):
        check(own[i].half(), want[i], off[i], "own scales")
        with pytest.raises(AssertionError):
            check(one[i].half(), want[i], off[i], "one scale")
