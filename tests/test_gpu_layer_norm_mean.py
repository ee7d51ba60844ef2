"""Layer norm of rows whose mean is large beside their spread: the mean costs its own rounding, whatever the width's sums lose."""
import pytest
import torch

import block_oracle as B

pytestmark = pytest.mark.gpu

# a wavefront a row, three vectors a lane, 256 threads, 1024, and rows that are read three times, odd ones of each
SIZES = [(3, 300), (3, 1000), (3, 1001), (4100, 1280), (4099, 1301), (3, 4096), (3, 4097), (3, 8192), (3, 30000), (3, 30001),
         (2, 1 << 19), (2, (1 << 20) + 24), (2, (1 << 20) + 9)]


@pytest.mark.parametrize("dtype", list(B.DTYPES))
@pytest.mark.parametrize("rows,width", SIZES)
def test_rows_of_one_value(device, aclnn, dtype, rows, width):
    """The mean is the value and the result the bias, exactly.

    The first sum is off by k roundings of 2^-24, k < 64 (8 elements of a vector, 16 to 32 vectors or a compensated sum, 6 steps
    between lanes, 16 wavefronts), and what it leaves of every element is exact; the mean of that is off by as much of itself,
    (64 * 2^-24)^2 of the value, or (1200 * 2^-24) * (64 * 2^-24) in rows of 2^20: less than the half step (2^-25) that
    rounds the mean to the value.  The variance is the difference of two squares of (64 * 2^-24 * 3000)^2 = 1.3e-4 at most,
    each off by 2 * 1200 * 2^-24 of itself in rows of 2^20 and 2 * 64 * 2^-24 in the others: 4e-8, 4e-3 of eps, or 2e-4."""
    g = torch.Generator(device=device).manual_seed(width)
    t = B.DTYPES[dtype]
    b = torch.randn(width, generator=g, device=device).to(t)
    for value, more in ((0.1, 0.0), (100.0, 0.1), (-3000.0, 0.3)):
        x = torch.full((rows, width), value, device=device).to(t)
        r = torch.full((rows, width), more, device=device).to(t)
        y, _, mean, rstd = aclnn.layer_norm(x, None, b, r, need_stats=True)
        assert (mean.double() == x[:, 0].double() + r[:, 0].double()).all() or dtype == "fp32" and (mean == x[:, 0] + r[:, 0]).all()
        assert torch.equal(y, b.expand_as(y))
        assert ((rstd.double() * 1e-5 ** 0.5 - 1).abs() <= (4e-3 if width >= 1 << 19 else 2e-4)).all()


@pytest.mark.parametrize("rows,width", SIZES)
def test_far_means(device, aclnn, rows, width):
    """A mean 3000 times the spread: half a step of it (2^-24 of its size at most) against the spread, and what the sums of
    the differences lose, gamma of the elements that a thread adds up one after the other and of the steps between threads."""
    g = torch.Generator(device=device).manual_seed(width + 1)
    x = 3000 + torch.randn(rows, width, generator=g, device=device)
    w, b = torch.randn(width, generator=g, device=device), torch.randn(width, generator=g, device=device)
    y, _, mean, rstd = aclnn.layer_norm(x, w, b, need_stats=True)
    h = x.double()
    want_mean = h.mean(-1, keepdim=True)
    d = h - want_mean
    want_rstd = 1 / torch.sqrt(d.square().mean(-1, keepdim=True) + 1e-5)
    sums = B.gamma(max(width / 1024, 32) + 64)
    off = 2.0 ** -24 * 3000 * 1.01 + sums * d.abs().mean(-1, keepdim=True)
    assert ((mean.double() - want_mean[:, 0]).abs() <= off[:, 0]).all()
    assert ((rstd.double() - want_rstd[:, 0]).abs() <= (sums + off[:, 0] ** 2) * want_rstd[:, 0]).all()
    n = d * want_rstd
    bound = (off * want_rstd + (sums + off ** 2 + 2.0 ** -22) * n.abs()) * w.double().abs() + 2.0 ** -23 * b.double().abs()
    assert ((y.double() - (n * w.double() + b.double())).abs() <= bound).all()
