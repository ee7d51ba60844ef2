"""Activations of the gated projections far below zero, where their values are small: bounds relative to the value, not the gate."""
import pytest
import torch

import block_oracle as B

pytestmark = pytest.mark.gpu

# A step is 2^-24 of the value.
# silu: the exponential's argument is off by a step and a half of itself (a constant's rounding and a product's), its value by that
#   times |g|; the exponential, the sum, the reciprocal and the product by 2, 1, 2 and 1.
# gelu: exp(-a^2 / 2), a = |g|: the square, the constant and their product are off by two steps and a half of the argument, the
#   value by that times a^2 / 2; the exponential, the reciprocal and the nine coefficients, which are up to twice the polynomial,
#   by 2, 3 and 19 steps with the fit's own half.
# gelu by tanh: sigmoid(u), |u| = 1.6 (a + 0.0447 a^3): two constants and five operations on numbers of one sign and the
#   exponential's one and a half, nine steps of u.
BOUNDS = {0: (80.0, lambda a: 6 + 1.5 * a), 1: (12.5, lambda a: 24 + 1.25 * a * a),
          2: (9.0, lambda a: 6 + 9 * 1.6 * (a + 0.0447 * a ** 3))}


@pytest.mark.parametrize("rows", [1, 200])
@pytest.mark.parametrize("kind", list(BOUNDS))
def test_tails(device, aclnn, kind, rows):
    most, steps = BOUNDS[kind]
    n = 1024
    gates = -torch.linspace(0.001, most, n)
    x = torch.zeros(rows, 4)
    x[:, 0] = 1
    wg, wu = torch.zeros(n, 4), torch.zeros(n, 4)
    wg[:, 0], wu[:, 0] = gates, 1
    y, gate, up = aclnn.gated_projection(x.to(device), wg.to(device), wu.to(device), activation=kind, need_sums=True)
    assert torch.equal(gate.cpu(), gates.expand(rows, n)) and (up == 1).all()
    g = gates.double()
    # in forms that keep the bits of a value next to 0 (torch.special.ndtr is 0 from -8.3 on)
    want = g * (torch.sigmoid(g), 0.5 * torch.erfc(g * -0.5 ** 0.5), torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (g + 0.044715 * g ** 3)))[kind]
    off = (y.cpu().double() / want - 1).abs() * 2.0 ** 24
    B.within(off, torch.zeros(rows, n), steps(g.abs()).expand(rows, n), "steps")
