"""Gradients of the gated projections of which only some are wanted: FLOAT16 finds scales for those that are multiplied."""
import pytest
import torch

import block_oracle as B
from test_blocks_boundary import phase1  # noqa: F401
from test_tokens_boundary import BF16, F16


def test_workspace(phase1):  # noqa: F811
    """Nothing beside the partial sums where only the biases' gradients are wanted, two words a scale in the others."""
    rows, width, inner = 768, 64, 128
    x, p, o, b = (rows, width), (inner, width), (rows, inner), (inner,)

    def ws(t, weights, biases, gx):
        v = [(s, t) for s in (o, x, p, p, o, o)]
        st, n, _ = phase1("opscvGatedProjectionBackward", *v, 0, (x, t) if gx else None, *([(p, t) if weights else None] * 2),
                          *([(b, t) if biases else None] * 2))
        assert st == 0
        return n
    assert ws(F16, False, True, False) == ws(BF16, False, True, False) > 0
    # multiples of 256 bytes each, so that slices have no gaps
    assert ws(F16, False, False, True) == ws(BF16, False, False, True) + 2 * rows * 4
    assert ws(F16, True, False, False) == ws(BF16, True, False, False) + 2 * 2 * inner * 4
    both = ws(F16, True, False, True) - ws(BF16, True, False, True)
    assert both == 2 * (rows + 2 * inner) * 4 + rows * 2 * inner * 2  # and the numbers in the columns' scales


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(B.DTYPES))
@pytest.mark.parametrize("rows,width,inner", [(1, 8, 8), (7, 100, 33), (70, 64, 300), (520, 136, 1031)])
def test_biases_alone(device, aclnn, dtype, rows, width, inner):
    """The same numbers as beside the others, and no other gradient's buffer is touched."""
    g = torch.Generator(device=device).manual_seed(rows)

    def rand(*size):
        return torch.randn(*size, generator=g, device=device).to(B.DTYPES[dtype])
    x, wg, wu, gate, up, gy = rand(rows, width), rand(inner, width), rand(inner, width), rand(rows, inner), rand(rows, inner), rand(rows, inner)
    whole = aclnn.gated_projection_backward(gy, x, wg, wu, gate, up, activation=1, need_bias=True)
    for need_x, need_weights in ((False, False), (True, False), (False, True)):
        some = aclnn.gated_projection_backward(gy, x, wg, wu, gate, up, activation=1, need_x=need_x, need_weights=need_weights,
                                               need_bias=True)
        assert torch.equal(some[3], whole[3]) and torch.equal(some[4], whole[4])
        want, off = B.gated_grad(*(t.cpu() for t in (gy, x, wg, wu, gate, up)), 1, dtype)
        for i, wanted in ((0, need_x), (1, need_weights), (2, need_weights)):
            assert (some[i] is not None) == wanted
            if wanted:
                B.within(some[i], want[i], off[i] + B.U[dtype] * want[i].abs() + B.TINY[dtype], "gradient %d" % i)
