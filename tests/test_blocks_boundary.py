"""Layer norm, rotary positions on several axes, dropout and gated projections without a GPU: what their first phases accept,
refuse and ask for, and the generator's published answers."""
import ctypes

import numpy as np
import pytest

import block_oracle as B
from test_tokens_boundary import BF16, F16, F32, F64, I32, I64, INVALID, NULLPTR, Phase1, changed


class Phase1Ints(Phase1):
    """A list stands for an aclIntArray."""

    def __call__(self, name, *args):
        made = [ctypes.c_void_p(self.a.create_int_array(x)) if isinstance(x, list) else x for x in args]
        try:
            return super().__call__(name, *made)
        finally:
            for x, h in zip(args, made):
                if isinstance(x, list):
                    self.a.destroy_int_array(h)


@pytest.fixture
def phase1(aclnn):
    p = Phase1Ints(aclnn)
    yield p
    for h in p.handles:
        aclnn.destroy_tensor(h)


R, W, V = ((6, 64), BF16), ((64,), BF16), ((6,), F32)
NORM = dict(x=R, residual=R, weight=W, bias=W, eps=1e-5, y=R, sum=R, mean=V, rstd=V)


@pytest.mark.parametrize("kw,status", [
    ({}, 0), (dict(residual=None, sum=None, mean=None, rstd=None), 0), (dict(weight=None, bias=None), 0),
    (dict(weight=None), 0), (dict(bias=None), 0), (dict(weight=((64,), F32), bias=((64,), F32)), 0), (dict(mean=None), 0),
    (dict(eps=0.0), 0),
    (dict(x=((0, 64), BF16), residual=None, y=((0, 64), BF16), sum=None, mean=None, rstd=None), 0),
    (dict(x=None), NULLPTR), (dict(y=None), NULLPTR), (dict(bias=((64,), F32)), INVALID), (dict(weight=((64,), F32)), INVALID),
    (dict(weight=((63,), BF16)), INVALID), (dict(bias=((63,), BF16)), INVALID), (dict(bias=((1, 64), BF16)), INVALID),
    (dict(bias=((64,), F16), weight=None), INVALID), (dict(y=((6, 64), F16)), INVALID), (dict(y=((6, 63), BF16)), INVALID),
    (dict(residual=((5, 64), BF16)), INVALID), (dict(residual=((6, 64), F16)), INVALID), (dict(sum=((6, 64), F32)), INVALID),
    (dict(mean=((6,), BF16)), INVALID), (dict(mean=((6, 1), F32)), INVALID), (dict(rstd=((7,), F32)), INVALID),
    (dict(eps=-1.0), INVALID), (dict(eps=float("nan")), INVALID), (dict(eps=1e39), INVALID),
    (dict(x=((6, 64), F64), y=((6, 64), F64), residual=None, sum=None), INVALID),
    (dict(x=((2 ** 40, 2 ** 40, 64), BF16), y=((2 ** 40, 2 ** 40, 64), BF16), residual=None, sum=None, mean=None, rstd=None), INVALID),
    (dict(x=((6, 0), BF16), y=((6, 0), BF16), weight=None, bias=None, residual=None, sum=None), INVALID)])
def test_layer_norm(phase1, kw, status):
    st, ws, variant = phase1("opscvLayerNorm", *changed(NORM, **kw))
    assert st == status
    if not kw:
        assert (ws, variant) == (0, "layer_norm")


NORM_GRAD = dict(gy=R, gs=R, sum=R, weight=W, mean=V, rstd=V, gx=R, gw=W, gb=W)


@pytest.mark.parametrize("kw,status", [
    ({}, 0), (dict(gs=None), 0), (dict(gw=None), 0), (dict(gb=None), 0), (dict(gw=None, gb=None), 0),
    (dict(weight=None), 0), (dict(weight=((64,), F32), gw=((64,), F32), gb=((64,), F32)), 0),
    (dict(weight=None, gw=None, gb=((64,), F32)), 0),
    (dict(gy=None), NULLPTR), (dict(sum=None), NULLPTR), (dict(mean=None), NULLPTR), (dict(rstd=None), NULLPTR),
    (dict(gx=None), NULLPTR), (dict(gw=((64,), F32)), INVALID), (dict(gb=((64,), F32)), INVALID), (dict(gb=((65,), BF16)), INVALID),
    (dict(gy=((6, 64), F32)), INVALID), (dict(gx=((6, 65), BF16)), INVALID), (dict(gs=((64,), BF16)), INVALID),
    (dict(mean=((6,), BF16)), INVALID), (dict(rstd=((5,), F32)), INVALID)])
def test_layer_norm_gradients(phase1, kw, status):
    st, ws, variant = phase1("opscvLayerNormBackward", *changed(NORM_GRAD, **kw))
    assert st == status
    if status == 0:
        assert variant == "layer_norm_grad" and (ws > 0) == (kw.get("gw", 1) is not None or kw.get("gb", 1) is not None)


Q, K = ((2, 5, 4, 64), BF16), ((2, 5, 2, 64), BF16)
AXES = dict(q=Q, k=K, positions=((3, 2, 5), I64), table=((100, 64), F32), sections=[8, 12, 12], layout=0, interleaved=False,
            inverse=False, qo=Q, ko=K)


@pytest.mark.parametrize("kw,status", [
    ({}, 0), (dict(k=None, ko=None), 0), (dict(positions=((3, 2, 5), I32)), 0), (dict(interleaved=True, inverse=True), 0),
    (dict(layout=2), 0), (dict(layout=1, table=((100, 24), F32)), 0), (dict(sections=[0, 16, 16]), 0),
    (dict(sections=[1, 0, 0], table=((100, 2), F32)), 0), (dict(sections=[32], positions=((1, 2, 5), I64)), 0),
    (dict(sections=[8, 8, 8, 8], positions=((4, 2, 5), I64)), 0), (dict(table=((0, 64), F32)), 0),
    (dict(q=((2, 0, 4, 64), BF16), qo=((2, 0, 4, 64), BF16), k=None, ko=None, positions=((3, 2, 0), I64)), 0),
    (dict(q=None), NULLPTR), (dict(table=None), NULLPTR), (dict(qo=None), NULLPTR), (dict(k=None), NULLPTR), (dict(ko=None), NULLPTR),
    (dict(positions=None), NULLPTR), (dict(sections=None), NULLPTR), (dict(sections=[]), INVALID),
    (dict(sections=[8, 8, 8, 4, 4], positions=((5, 2, 5), I64)), INVALID), (dict(sections=[-1, 17, 16]), INVALID),
    (dict(sections=[2 ** 62, 2 ** 62, 2 ** 62]), INVALID), (dict(sections=[0, 0, 0], table=((100, 0), F32)), INVALID),
    (dict(sections=[8, 12, 13], table=((100, 66), F32)), INVALID), (dict(layout=3), INVALID), (dict(layout=-1), INVALID),
    (dict(layout=1), INVALID), (dict(table=((100, 62), F32)), INVALID), (dict(table=((100, 65), F32)), INVALID),
    (dict(table=((100, 64), F16)), INVALID), (dict(positions=((2, 2, 5), I64)), INVALID), (dict(positions=((2, 5), I64)), INVALID),
    (dict(positions=((3, 2, 4), I64)), INVALID), (dict(positions=((3, 2, 5), F32)), INVALID),
    (dict(q=((2, 5, 4, 1040), BF16), qo=((2, 5, 4, 1040), BF16), k=None, ko=None, sections=[520], positions=((1, 2, 5), I64),
          table=((100, 1040), F32)), INVALID),
    (dict(q=((2, 5, 4, 64), F64)), INVALID), (dict(qo=((2, 5, 4, 63), BF16)), INVALID), (dict(k=((2, 4, 2, 64), BF16)), INVALID)])
def test_rotary_axes(phase1, kw, status):
    st, ws, variant = phase1("opscvRotaryAxes", *changed(AXES, **kw))
    assert st == status
    if not kw:
        assert (ws, variant) == (0, "rotary_axes")


DROPOUT = dict(x=R, residual=R, state=((2,), I64), p=0.1, y=R)


@pytest.mark.parametrize("kw,status", [
    ({}, 0), (dict(residual=None), 0), (dict(p=0.0), 0), (dict(p=1.0), 0), (dict(x=((0, 64), BF16), residual=None, y=((0, 64), BF16)), 0),
    (dict(x=None), NULLPTR), (dict(state=None), NULLPTR), (dict(y=None), NULLPTR), (dict(p=-0.1), INVALID), (dict(p=1.1), INVALID),
    (dict(p=float("nan")), INVALID), (dict(state=((3,), I64)), INVALID), (dict(state=((2, 1), I64)), INVALID),
    (dict(state=((2,), I32)), INVALID), (dict(residual=((6, 63), BF16)), INVALID), (dict(residual=((6, 64), F32)), INVALID),
    (dict(y=((6, 64), F32)), INVALID), (dict(x=((6, 64), I32), y=((6, 64), I32), residual=None), INVALID)])
def test_dropout(phase1, kw, status):
    st, ws, variant = phase1("opscvDropout", *changed(DROPOUT, **kw))
    assert st == status
    if not kw:
        assert (ws, variant) == (0, "dropout")


X, P, O, BI = ((6, 64), BF16), ((40, 64), BF16), ((6, 40), BF16), ((40,), BF16)
GATED = dict(x=X, wg=P, wu=P, bg=BI, bu=BI, activation=0, y=O, gate=O, up=O)
SHARED = [
    (dict(x=None), NULLPTR), (dict(wg=None), NULLPTR), (dict(wu=None), NULLPTR), (dict(gate=None), NULLPTR), (dict(up=None), NULLPTR),
    (dict(wg=((40, 63), BF16)), INVALID), (dict(wu=((41, 64), BF16)), INVALID), (dict(wu=((40, 64), F16)), INVALID),
    (dict(wg=((40, 64, 1), BF16)), INVALID), (dict(gate=((6, 41), BF16)), INVALID), (dict(up=((6, 40), F32)), INVALID),
    (dict(gate=((5, 40), BF16)), INVALID), (dict(activation=3), INVALID), (dict(activation=-1), INVALID),
    (dict(x=((6, 64), F64)), INVALID), (dict(x=((6, 0), BF16)), INVALID)]


@pytest.mark.parametrize("kw,status", [
    ({}, 0), (dict(bg=None, bu=None), 0), (dict(gate=None, up=None), 0), (dict(activation=1), 0), (dict(activation=2), 0),
    (dict(x=((0, 64), BF16), y=((0, 40), BF16), gate=None, up=None), 0),
    (dict(x=((2, 3, 64), BF16), y=((2, 3, 40), BF16), gate=None, up=None), 0), (dict(x=((64,), BF16), y=((40,), BF16), gate=None, up=None), 0),
    (dict(bg=None), NULLPTR), (dict(bu=None), NULLPTR), (dict(y=None), NULLPTR), (dict(bg=((41,), BF16)), INVALID),
    (dict(bu=((40,), F32)), INVALID), (dict(y=((6, 64), BF16)), INVALID), (dict(y=((2, 3, 40), BF16)), INVALID),
    (dict(wg=((0, 64), BF16), wu=((0, 64), BF16), bg=None, bu=None, y=((6, 0), BF16), gate=None, up=None), INVALID),
    (dict(x=((6, 2 ** 19 + 1), BF16), wg=((40, 2 ** 19 + 1), BF16), wu=((40, 2 ** 19 + 1), BF16)), INVALID),
    (dict(x=((2 ** 30 + 1, 64), BF16), y=((2 ** 30 + 1, 40), BF16), gate=None, up=None), INVALID),
    # as many rows and features as are allowed, but not together
    (dict(x=((2 ** 30, 64), BF16), y=((2 ** 30, 40), BF16), gate=None, up=None), 0),
    (dict(x=((2 ** 30, 64), BF16), wg=((2 ** 19, 64), BF16), wu=((2 ** 19, 64), BF16), bg=None, bu=None,
          y=((2 ** 30, 2 ** 19), BF16), gate=None, up=None), INVALID)] + SHARED)
def test_gated(phase1, kw, status):
    st, ws, variant = phase1("opscvGatedProjection", *changed(GATED, **kw))
    assert st == status
    if not kw:
        assert (ws, variant) == (0, "gated_projection")


def test_gated_workspace(phase1):
    """Rows of whole vectors are read in place, others copied with zeros behind them."""
    def ws(width, dtype, strides=None):
        st, n, _ = phase1("opscvGatedProjection", ((6, width), dtype) + ((strides,) if strides else ()), ((40, width), dtype),
                          ((40, width), dtype), None, None, 0, ((6, 40), dtype), None, None)
        assert st == 0
        return n
    assert ws(64, BF16) == ws(68, F32) == ws(64, BF16, [72, 1]) == 0
    assert ws(63, BF16) >= (6 + 40 + 40) * 64 * 2 and ws(66, F32) >= (6 + 40 + 40) * 68 * 4
    assert 6 * 64 * 2 <= ws(64, BF16, [65, 1]) < 3 * 6 * 64 * 2  # odd rows
    assert ws(64, BF16, [1, 6]) == 6 * 64 * 2                   # columns are packed, and need no second copy
    assert ws(64, F16, [2 ** 20 + 8, 1]) >= 6 * 64 * 2          # rows too far apart for 32-bit offsets in a tile


GATED_GRAD = dict(gy=O, x=X, wg=P, wu=P, gate=O, up=O, activation=0, gx=X, gwg=P, gwu=P, gbg=BI, gbu=BI)


@pytest.mark.parametrize("kw,status", [
    ({}, 0), (dict(gx=None), 0), (dict(gwg=None, gwu=None), 0), (dict(gbg=None, gbu=None), 0),
    (dict(gx=None, gwg=None, gwu=None), 0), (dict(gwg=None, gwu=None, gbg=None, gbu=None), 0),
    (dict(gy=None), NULLPTR), (dict(gwg=None), NULLPTR), (dict(gwu=None), NULLPTR), (dict(gbg=None), NULLPTR), (dict(gbu=None), NULLPTR),
    (dict(gx=None, gwg=None, gwu=None, gbg=None, gbu=None), NULLPTR), (dict(gy=((6, 64), BF16)), INVALID), (dict(gx=O), INVALID),
    (dict(gwg=((64, 40), BF16)), INVALID), (dict(gwu=((40, 64), F32)), INVALID), (dict(gbg=((64,), BF16)), INVALID),
    (dict(gbu=((40,), F32)), INVALID),
    (dict(x=((2 ** 20 + 1, 64), BF16), gy=((2 ** 20 + 1, 40), BF16), gate=((2 ** 20 + 1, 40), BF16),
          up=((2 ** 20 + 1, 40), BF16), gx=((2 ** 20 + 1, 64), BF16)), INVALID)] + SHARED)
def test_gated_gradients(phase1, kw, status):
    st, ws, variant = phase1("opscvGatedProjectionBackward", *changed(GATED_GRAD, **kw))
    assert st == status
    if status == 0:
        assert variant == "gated_projection_grad" and ws > 0


def test_no_rows(phase1):
    """No rows: nothing to do, but the gradients of columns and weights, which are zeros."""
    none, vec = ((0, 64), BF16), ((0,), F32)
    assert phase1("opscvLayerNormBackward", none, None, none, W, vec, vec, none, None, None) == (0, 0, "")
    assert phase1("opscvLayerNormBackward", none, None, none, W, vec, vec, none, W, None)[2] == "layer_norm_grad"
    o = ((0, 40), BF16)
    assert phase1("opscvGatedProjectionBackward", o, none, P, P, o, o, 0, none, None, None, None, None) == (0, 0, "")
    assert phase1("opscvGatedProjectionBackward", o, none, P, P, o, o, 0, none, P, P, BI, BI)[2] == "gated_projection_grad"


def test_second_phases_refuse(aclnn, phase1):
    L = aclnn.load_library()
    names = ("LayerNorm", "LayerNormBackward", "RotaryAxes", "Dropout", "GatedProjection", "GatedProjectionBackward")
    for name in names:
        assert getattr(L, "opscv" + name)(None, 0, None, None) == NULLPTR

    def executor(name, args):
        ws, ex = ctypes.c_uint64(0), ctypes.c_void_p(None)
        made = [phase1.t(x) if isinstance(x, tuple) else x for x in args]
        assert getattr(L, "opscv" + name + "GetWorkspaceSize")(*made, ctypes.byref(ws), ctypes.byref(ex)) == 0
        return ws.value, ex
    for name, args in (("LayerNorm", NORM), ("Dropout", DROPOUT), ("GatedProjection", GATED)):
        _, ex = executor(name, args.values())
        assert getattr(L, "opscv" + name)(None, 0, ex, None) == NULLPTR  # no data
        _, ex = executor(name, args.values())
        assert L.opscvRotary(None, 0, ex, None) == INVALID  # another operator's
    for name, args in (("LayerNormBackward", NORM_GRAD), ("GatedProjectionBackward", GATED_GRAD)):
        ws, ex = executor(name, args.values())
        assert ws > 0 and getattr(L, "opscv" + name)(None, 0, ex, None) == NULLPTR
        ws, ex = executor(name, args.values())
        assert getattr(L, "opscv" + name)(ctypes.c_void_p(4096), ws - 1, ex, None) == INVALID
        ws, ex = executor(name, args.values())
        assert getattr(L, "opscv" + name)(ctypes.c_void_p(4104), ws, ex, None) == INVALID
    # an executor of plain rotary is not one of several axes
    from test_tokens_boundary import ROTARY
    _, ex = executor("Rotary", ROTARY.values())
    assert L.opscvRotaryAxes(None, 0, ex, None) == INVALID


def test_generator():
    """The published answers of Philox 4x32-10: counter and key of zeros, of ones, and of digits of pi."""
    def words(c, k):
        counter, offset = c[0] | c[1] << 32, c[2] | c[3] << 32
        return [int(w) for w in B.philox(np.array([counter], dtype=np.uint64), offset, k[0] | k[1] << 32)[0]]
    ones = 0xffffffff
    assert words([0] * 4, [0] * 2) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    assert words([ones] * 4, [ones] * 2) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
    assert words([0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344], [0xa4093822, 0x299f31d0]) == [
        0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1]
