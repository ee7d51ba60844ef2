"""Gated projections of operands whose rows lie apart, each by a stride of its own, or of which only some are copied, in every way
of making the products: as dense operands, which the same plan serves."""
import math

import pytest
import torch

import block_oracle as B
import host_plans as P
from test_blocks_boundary import phase1  # noqa: F401
from test_gpu_blocks_products import TILE, operands
from test_tokens_boundary import BF16, F16, F32

TYPES = {"fp32": F32, "fp16": F16, "bf16": BF16}
# strides of x, gate's and up's weight: elements beside the width, in vectors of 16 bytes, and elements before the first one;
# a stride of an odd number of elements, or a start off 16 bytes, makes a copy
HOW = {"three strides": ((1, 0), (2, 1), (5, 2)), "up copied": ((0, 0), (3, 0), ("odd", 1)), "gate copied": ((1, 0), ("odd", 3), (2, 1)),
       "x copied": (("odd", 0), (1, 0), (4, 3)), "both weights copied": ((2, 2), ("odd", 0), ("odd", 5)),
       "far": (("far", 0), ("too far", 0), (2, 0))}


def stride(how, width, vec):
    return {"odd": width + 1 + width % 2 + 2 * vec, "far": 1 << 20, "too far": (1 << 20) + vec}.get(how) or width + how * vec


def apart(t, how, vec):
    """A copy of t whose rows lie so apart, with NaN between them."""
    (more, before), (rows, width) = how, t.shape
    pitch = stride(more, width, vec)
    first = before if more == "odd" else before * vec
    size = (rows - 1) * pitch + width + first
    big = torch.full((size,), math.nan, dtype=t.dtype, device=t.device) if size < 1 << 28 else torch.empty(size, dtype=t.dtype, device=t.device)
    view = torch.as_strided(big, t.shape, (pitch, 1), first)
    return view.copy_(t)


# widths of whole vectors; (type, size, tile, parts)
FORWARD = [("bf16", (129, 192, 65), "deep", False), ("fp16", (512, 1032, 520), "deep", False), ("bf16", (2049, 24, 1000), "128", False),
           ("fp16", (1030, 200, 2100), "128", False), ("bf16", (129, 2056, 257), "128", True), ("bf16", (2049, 1032, 2100), "256", False),
           ("fp16", (2049, 1032, 2100), "256", False), ("fp32", (300, 72, 520), "slim", False), ("fp32", (65, 520, 30), "slim", True),
           ("fp32", (2049, 20, 520), "128", False), ("fp32", (2049, 2056, 2100), "256", True),
           ("bf16", (20, 1032, 200), "few", False), ("fp32", (33, 1028, 70), "few", False)]


def units(device):
    return torch.cuda.get_device_properties(device).multi_processor_count


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,size,tile,parts", FORWARD)
def test_forward(device, aclnn, dtype, size, tile, parts):
    plan = P.gated_plan(dtype, 0, *size, units=units(device))
    assert (TILE[plan[0]], plan[1] > 1) == (tile, parts)
    x, weights, biases, outs = operands(device, dtype, *size)
    vec = 16 // x.element_size()
    want = aclnn.gated_projection(x, *weights, *biases, activation=1, need_sums=True)
    bound = B.gated(x, *weights, *biases, 1)
    for t, w, off in zip(want, *bound):
        B.within(t, w.cpu(), (off + B.U[dtype] * w.abs() + B.TINY[dtype]).cpu(), "dense")
    for name, how in HOW.items():
        v = [apart(t, h, vec) for t, h in zip((x, *weights), how)]
        into = [apart(torch.zeros_like(t), h, vec) for t, h in zip(outs, ((3, 0), ("odd", 1), (1, 2)))]
        got = aclnn.gated_projection(*v, *biases, activation=1, need_sums=True, out=into[0], gate_out=into[1], up_out=into[2])
        for p, q, what in zip(got, want, ("y", "gate", "up")):
            assert torch.equal(p, q), (name, what)
        del v, into


# of all gradients; (type, size, tile, parts of both)
BACKWARD = [("bf16", (1030, 24, 30), "128", (False, True)), ("bf16", (2049, 24, 520), "128", (True, True)),
            ("bf16", (1030, 4104, 520), "256", (False, False)), ("fp16", (2049, 520, 4200), "256", (True, False)),
            ("fp16", (2049, 24, 520), "128", (True, True)), ("fp32", (160, 516, 1100), "slim", (True, False)),
            ("fp32", (520, 20, 264), "128", (True, True)), ("fp32", (4100, 4104, 2100), "256", (False, True))]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,size,tile,parts", BACKWARD)
def test_backward(device, aclnn, dtype, size, tile, parts):
    plan = P.gated_plan(dtype, 3, *size, units=units(device))
    assert (TILE[plan[0]], plan[1] > 1, plan[2] > 1) == (tile, *parts)
    x, weights, _, sums = operands(device, dtype, *size)
    vec = 16 // x.element_size()
    want = aclnn.gated_projection_backward(sums[2], x, *weights, *sums[:2], activation=2, need_bias=True)
    wanted, off = B.gated_grad(sums[2], x, *weights, *sums[:2], 2, dtype)
    for t, w, o in zip(want, wanted, off):
        B.within(t, w.cpu(), (o + B.U[dtype] * w.abs() + B.TINY[dtype]).cpu(), "dense")
    del wanted, off
    for name, how in HOW.items():
        v = [apart(t, h, vec) for t, h in zip((x, *weights), how)]
        s = [apart(t, h, vec) for t, h in zip(sums, ((1, 2), ("odd", 1), (3, 0)))]
        into = [apart(torch.zeros_like(t), h, vec) for t, h in zip((x, *weights), ((2, 1), ("odd", 3), (1, 0)))]
        got = aclnn.gated_projection_backward(s[2], *v, *s[:2], activation=2, need_bias=True, grad_x=into[0],
                                              grad_gate_weight=into[1], grad_up_weight=into[2])
        for p, q, what in zip(got, want, ("x", "gate weight", "up weight", "gate bias", "up bias")):
            assert torch.equal(p, q), (name, what)
        del v, s, into


@pytest.mark.parametrize("dtype", list(TYPES))
def test_what_is_copied(phase1, dtype):  # noqa: F811
    """The workspaces that those operands ask for: those that are copied and no others."""
    rows, width, inner, t, e = 64, 128, 256, TYPES[dtype], 4 if dtype == "fp32" else 2
    vec, o = 16 // e, (64, 256)

    def asked(name, how):
        x, wg, wu = (((n, width), t, [stride(h[0], width, vec), 1]) for n, h in zip((rows, inner, inner), how))
        args = (x, wg, wu, None, None, 0, (o, t), None, None) if name == "opscvGatedProjection" else (
            (o, t), x, wg, wu, (o, t), (o, t), 0, ((rows, width), t), *([((inner, width), t)] * 2), None, None)
        st, ws, _ = phase1(name, *args)
        assert st == 0
        return ws
    for name in ("opscvGatedProjection", "opscvGatedProjectionBackward"):
        dense = asked(name, [(0, 0)] * 3)
        for how in HOW.values():
            copied = sum(n for n, h in zip((rows, inner, inner), how) if h[0] in ("odd", "too far"))
            assert asked(name, how) == dense + copied * width * e
