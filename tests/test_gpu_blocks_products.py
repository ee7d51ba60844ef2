"""The gated projections at sizes that take each way of making their products: tiles of both sizes, terms in parts, few rows.
The plain implementation in 64 bits runs on the GPU as well."""
import pytest
import torch

import block_oracle as B
import host_plans as P

pytestmark = pytest.mark.gpu

TILE = {0: "128", 1: "256", 2: "few", 3: "slim", 4: "deep"}


def operands(device, dtype, rows, width, inner):
    g = torch.Generator(device=device).manual_seed(rows + width + inner)

    def rand(*size, scale=1.0):
        return (torch.randn(*size, generator=g, device=device, dtype=torch.float64) * scale).to(B.DTYPES[dtype])
    x, weights = rand(rows, width), [rand(inner, width, scale=width ** -0.5) for _ in range(2)]
    return x, weights, [rand(inner) for _ in range(2)], [rand(rows, inner) for _ in range(3)]


def close(got, want, off, dtype, what):
    bound = off + B.U[dtype] * want.abs() + B.TINY[dtype]
    B.within(got, want.cpu(), bound.cpu(), what)


def way(device, dtype, kind, size):
    p = P.gated_plan(dtype, kind, *size, units=torch.cuda.get_device_properties(device).multi_processor_count)
    return TILE[p[0]], p[1] > 1, p[2] > 1


# (type, size, tile, parts): the plan is asked, so that a change of its rules does not leave a way without a test
FORWARD = [("bf16", (65, 20, 30), "deep", False), ("bf16", (2049, 20, 1000), "128", False), ("fp16", (1030, 200, 2100), "128", False),
           *[(t, (129, width, 65), "deep", False) for t in ("bf16", "fp16") for width in (64, 128, 192, 250, 300, 640)],
           ("bf16", (512, 1032, 2000), "deep", False), ("fp16", (700, 383, 511), "deep", False),
           ("bf16", (65, 1032, 30), "128", True), ("bf16", (129, 2056, 257), "128", True),
           ("bf16", (2049, 1032, 2100), "256", False), ("bf16", (2049, 1031, 2101), "256", False), ("bf16", (4100, 8200, 520), "256", True),
           ("bf16", (20, 1032, 200), "few", False), ("bf16", (40, 520, 33), "few", False), ("bf16", (64, 2050, 4200), "few", False),
           ("fp16", (2049, 1032, 2100), "256", False), ("fp16", (4100, 8200, 520), "256", True), ("fp16", (300, 4100, 200), "128", True),
           ("fp32", (65, 520, 30), "slim", True), ("fp32", (300, 72, 520), "slim", False), ("fp32", (97, 63, 1031), "slim", False),
           ("fp32", (2049, 20, 520), "128", False), ("fp32", (1030, 2056, 30), "128", True), ("fp32", (389, 640, 1200), "slim", False),
           ("fp32", (2049, 2056, 2100), "256", True),
           ("fp32", (33, 1030, 70), "few", False), ("fp32", (60, 500, 2100), "few", False)]


@pytest.mark.parametrize("dtype,size,tile,parts", FORWARD)
def test_forward(device, aclnn, dtype, size, tile, parts):
    assert way(device, dtype, 0, size)[:2] == (tile, parts)
    x, weights, biases, _ = operands(device, dtype, *size)
    for kind, b in ((0, (None, None)), (1, biases), (2, biases)):
        want, off = B.gated(x, *weights, *b, kind)
        got = aclnn.gated_projection(x, *weights, *b, activation=kind, need_sums=True)
        for t, w, e, what in zip(got, want, off, ("y", "gate", "up")):
            close(t, w, e, dtype, what)
        assert torch.equal(aclnn.gated_projection(x, *weights, *b, activation=kind)[0], got[0])


# kind: 1 for x's gradient plus 2 for the weights'
BACKWARD = [("bf16", 1, (20, 20, 520), "128", (True, False)), ("bf16", 2, (1030, 20, 30), "128", (True, False)),
            ("bf16", 3, (1030, 20, 30), "128", (False, True)), ("bf16", 3, (2049, 20, 520), "128", (True, True)),
            ("bf16", 1, (2049, 4104, 520), "256", (False, False)), ("bf16", 1, (2049, 2056, 4200), "256", (True, False)),
            ("bf16", 2, (300, 8200, 520), "256", (False, False)), ("bf16", 3, (1030, 4104, 520), "256", (False, False)),
            ("bf16", 3, (1030, 4100, 520), "256", (False, False)), ("bf16", 3, (2049, 520, 4200), "256", (True, False)),
            ("fp16", 3, (2049, 520, 4200), "256", (True, False)), ("fp16", 2, (300, 8200, 520), "256", (False, False)),
            ("fp16", 3, (2049, 20, 520), "128", (True, True)),
            ("fp32", 1, (20, 20, 264), "slim", (True, False)), ("fp32", 1, (2049, 20, 520), "128", (True, False)), ("fp32", 1, (520, 4104, 30), "128", (False, False)),
            ("fp32", 3, (33, 300, 200), "slim", (True, False)), ("fp32", 3, (1, 1031, 30), "slim", (False, False)),
            ("fp32", 3, (160, 516, 1100), "slim", (True, False)), ("fp32", 3, (520, 20, 264), "128", (True, True)),
            ("fp32", 3, (300, 20, 2100), "slim", (True, True)), ("fp32", 3, (4100, 20, 264), "slim", (False, True)),
            ("fp32", 3, (65, 20, 30), "128", (False, False)),
            ("fp32", 1, (2049, 4104, 1100), "256", (True, False)), ("fp32", 2, (2049, 2056, 2100), "256", (True, False)),
            ("fp32", 3, (4100, 4104, 2100), "256", (False, True))]


@pytest.mark.parametrize("dtype,which,size,tile,parts", BACKWARD)
def test_backward(device, aclnn, dtype, which, size, tile, parts):
    assert way(device, dtype, which, size) == (tile, *parts)
    x, weights, _, (gate, up, gy) = operands(device, dtype, *size)
    kind = sum(size) % 3
    want, off = B.gated_grad(gy, x, *weights, gate, up, kind, dtype)
    got = aclnn.gated_projection_backward(gy, x, *weights, gate, up, activation=kind, need_x=bool(which & 1),
                                          need_weights=bool(which & 2))
    for t, w, e, what in zip(got, want, off, ("x", "gate weight", "up weight")):
        if t is not None:
            close(t, w, e, dtype, "gradient of the " + what)


@pytest.mark.parametrize("dtype", list(B.DTYPES))
@pytest.mark.parametrize("size", [(3, 1 << 19, 40), (70, (1 << 19) - 1, 9), (2, 24, 1 << 19), (200, 7, (1 << 19) - 3), (1 << 20, 8, 16),
                                  ((1 << 20) - 1, 3, 5)])
def test_ends_of_the_sizes(device, aclnn, dtype, size):
    x, weights, biases, (gate, up, gy) = operands(device, dtype, *size)
    want, off = B.gated(x, *weights, *biases, 0)
    got = aclnn.gated_projection(x, *weights, *biases, need_sums=True)
    for t, w, e, what in zip(got, want, off, ("y", "gate", "up")):
        close(t, w, e, dtype, what)
    want, off = B.gated_grad(gy, x, *weights, gate, up, 0, dtype)
    got = aclnn.gated_projection_backward(gy, x, *weights, gate, up, need_bias=True)
    for t, w, e, what in zip(got, want, off, ("x", "gate weight", "up weight", "gate bias", "up bias")):
        close(t, w, e, dtype, "gradient of the " + what)
