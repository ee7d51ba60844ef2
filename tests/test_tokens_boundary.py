"""The operators on token sequences without a GPU: what their first phases accept, refuse and ask for.

Descriptors have NULL data pointers, as in the boundary tests of the other operators: a first phase is host-only."""
import ctypes

import pytest

NULLPTR, INVALID = 161001, 161002
F32, F16, BF16, I8, I32, I64, F64 = 0, 1, 27, 2, 3, 9, 11


class Phase1:
    """First phases on descriptors given as (dims, type) or (dims, type, strides); None: a NULL argument."""

    def __init__(self, aclnn):
        self.a, self.L, self.handles = aclnn, aclnn.load_library(), []

    def t(self, spec):
        if spec is None:
            return None
        h = self.a.create_tensor(spec[0], spec[1], strides=spec[2] if len(spec) > 2 else None,
                                 storage_dims=[1 << 40] if len(spec) > 2 else None)
        assert h, spec
        self.handles.append(h)
        return h

    def __call__(self, name, *args):
        ws, ex = ctypes.c_uint64(123), ctypes.c_void_p(None)
        made = [self.t(x) if isinstance(x, tuple) else x for x in args]
        st = getattr(self.L, name + "GetWorkspaceSize")(*made, ctypes.byref(ws), ctypes.byref(ex))
        variant = self.a.executor_variant(ex.value) if ex.value else None
        if ex.value:
            assert self.a.destroy_executor(ex.value) == 0
        else:
            assert self.L.aclGetRecentErrMsg()
        return st, ws.value, variant


@pytest.fixture
def phase1(aclnn):
    p = Phase1(aclnn)
    yield p
    for h in p.handles:
        aclnn.destroy_tensor(h)


def changed(good, **kw):
    args = list(good.values())
    for k, v in kw.items():
        args[list(good).index(k)] = v
    return args


NORM = dict(x=((6, 64), BF16), residual=((6, 64), BF16), weight=((64,), BF16), eps=1e-6, y=((6, 64), BF16), scale=None,
            sum=((6, 64), BF16), rstd=((6,), F32))


@pytest.mark.parametrize("kw,status", [
    ({}, 0), (dict(residual=None, sum=None, rstd=None), 0), (dict(weight=((64,), F32)), 0),
    (dict(y=((6, 64), I8), scale=((6,), F32)), 0),
    (dict(x=((0, 64), BF16), residual=None, y=((0, 64), BF16), sum=None, rstd=None), 0),
    (dict(x=None), NULLPTR), (dict(weight=None), NULLPTR), (dict(y=None), NULLPTR), (dict(y=((6, 64), I8)), NULLPTR),
    (dict(scale=((6,), F32)), INVALID), (dict(y=((6, 64), I8), scale=((6, 1), F32)), INVALID),
    (dict(y=((6, 64), I8), scale=((6,), BF16)), INVALID), (dict(y=((6, 64), F16)), INVALID), (dict(y=((6, 63), BF16)), INVALID),
    (dict(residual=((6, 64), F16)), INVALID), (dict(residual=((5, 64), BF16)), INVALID), (dict(sum=((6, 64), F32)), INVALID),
    (dict(weight=((63,), BF16)), INVALID), (dict(weight=((64,), F16)), INVALID), (dict(weight=((1, 64), BF16)), INVALID),
    (dict(rstd=((6,), BF16)), INVALID), (dict(rstd=((6, 64), F32)), INVALID), (dict(eps=-1.0), INVALID),
    (dict(eps=float("nan")), INVALID), (dict(x=((6, 64), F64), y=((6, 64), F64), residual=None, sum=None), INVALID),
    (dict(x=((6, 0), BF16), y=((6, 0), BF16), weight=((0,), BF16), residual=None, sum=None), INVALID),
    (dict(x=((1, 1, 1, 1, 1, 64), BF16)), INVALID)])
def test_norm(phase1, kw, status):
    assert phase1("opscvResidualNorm", *changed(NORM, **kw))[0] == status


def test_norm_workspace_and_names(phase1):
    assert phase1("opscvResidualNorm", *NORM.values()) == (0, 0, "residual_norm")
    rows = phase1("opscvResidualNorm", *changed(NORM, x=((6, 64), BF16, [100, 1])))
    assert rows == (0, 0, "residual_norm")  # rows apart are read in place
    st, ws, _ = phase1("opscvResidualNorm", *changed(NORM, x=((6, 64), BF16, [1, 6]), y=((6, 64), I8, [1, 6]), scale=((6,), F32)))
    assert st == 0 and ws >= 6 * 64 * 3  # columns are packed: two bytes in, one out
    assert phase1("opscvResidualNorm", *changed(NORM, x=((0, 64), BF16), y=((0, 64), BF16), residual=None, sum=None,
                                                rstd=None))[2] == ""


NORM_GRAD = dict(gy=((6, 64), F16), gs=((6, 64), F16), sum=((6, 64), F16), weight=((64,), F16), rstd=((6,), F32),
                 gx=((6, 64), F16), gw=((64,), F16))


@pytest.mark.parametrize("kw,status", [
    ({}, 0), (dict(gs=None, gw=None), 0), (dict(weight=((64,), F32), gw=((64,), F32)), 0),
    (dict(gy=None), NULLPTR), (dict(sum=None), NULLPTR), (dict(weight=None), NULLPTR), (dict(rstd=None), NULLPTR),
    (dict(gx=None), NULLPTR), (dict(gw=((64,), F32)), INVALID), (dict(gw=((63,), F16)), INVALID),
    (dict(gy=((6, 64), F32)), INVALID), (dict(gx=((6, 65), F16)), INVALID), (dict(gs=((64,), F16)), INVALID),
    (dict(rstd=((6,), F16)), INVALID), (dict(rstd=((7,), F32)), INVALID)])
def test_norm_gradients(phase1, kw, status):
    st, ws, variant = phase1("opscvResidualNormBackward", *changed(NORM_GRAD, **kw))
    assert st == status
    if status == 0:
        assert variant == "residual_norm_grad" and (ws > 0) == (kw.get("gw", 1) is not None)


TABLE = dict(base=10000.0, scaling=0, factor=1.0, original=0, magnitude=1.0, table=((100, 64), F32))


@pytest.mark.parametrize("kw,status", [
    ({}, 0), (dict(scaling=1, factor=4.0), 0), (dict(scaling=2, factor=4.0), 0), (dict(scaling=3, factor=4.0, original=2048), 0),
    (dict(table=((0, 64), F32)), 0), (dict(table=None), NULLPTR), (dict(table=((100, 63), F32)), INVALID),
    (dict(table=((100, 64), F16)), INVALID), (dict(table=((100, 1026), F32)), INVALID), (dict(table=((100,), F32)), INVALID),
    (dict(base=1.0), INVALID), (dict(base=float("inf")), INVALID), (dict(magnitude=float("nan")), INVALID),
    (dict(scaling=4), INVALID), (dict(scaling=-1), INVALID), (dict(scaling=1, factor=0.5), INVALID),
    (dict(scaling=2, factor=2.0, table=((100, 2), F32)), INVALID), (dict(scaling=3, factor=2.0), INVALID)])
def test_rotary_table(phase1, kw, status):
    assert phase1("opscvRotaryTable", *changed(TABLE, **kw))[0] == status


ROTARY = dict(q=((2, 5, 4, 64), BF16), k=((2, 5, 2, 64), BF16), positions=((2, 5), I64), table=((100, 32), F32),
              interleaved=False, inverse=False, qo=((2, 5, 4, 64), BF16), ko=((2, 5, 2, 64), BF16))


@pytest.mark.parametrize("kw,status", [
    ({}, 0), (dict(k=None, ko=None), 0), (dict(positions=None), 0), (dict(positions=((2, 5), I32)), 0),
    (dict(interleaved=True, inverse=True), 0), (dict(q=((2, 0, 4, 64), BF16), qo=((2, 0, 4, 64), BF16), k=None, ko=None, positions=None), 0),
    (dict(q=None), NULLPTR), (dict(table=None), NULLPTR), (dict(qo=None), NULLPTR), (dict(k=None), NULLPTR), (dict(ko=None), NULLPTR),
    (dict(q=((2, 5, 256), BF16)), INVALID), (dict(q=((2, 5, 4, 64), F64)), INVALID), (dict(qo=((2, 5, 4, 64), F16)), INVALID),
    (dict(qo=((2, 5, 4, 63), BF16)), INVALID), (dict(k=((2, 4, 2, 64), BF16)), INVALID), (dict(k=((2, 5, 2, 32), BF16)), INVALID),
    (dict(k=((2, 5, 2, 64), F16)), INVALID), (dict(positions=((2, 4), I64)), INVALID), (dict(positions=((10,), I64)), INVALID),
    (dict(positions=((2, 5), F32)), INVALID), (dict(table=((100, 66), F32)), INVALID), (dict(table=((100, 31), F32)), INVALID),
    (dict(table=((100, 32), F16)), INVALID)])
def test_rotary(phase1, kw, status):
    assert phase1("opscvRotary", *changed(ROTARY, **kw))[0] == status


ATTENTION = dict(q=((2, 9, 4, 64), F16), k=((2, 30, 2, 64), F16), v=((2, 30, 2, 64), F16), ql=((2,), I32), kl=((2,), I64),
                 scale=0.125, left=7, right=0, sinks=2, out=((2, 9, 4, 64), F16), lse=((2, 4, 9), F32))
REFUSED = [
    (dict(q=None), NULLPTR), (dict(k=None), NULLPTR), (dict(v=None), NULLPTR), (dict(out=None), NULLPTR),
    (dict(q=((2, 9, 256), F16)), INVALID), (dict(q=((2, 9, 4, 64), F64)), INVALID), (dict(k=((2, 30, 2, 64), BF16)), INVALID),
    (dict(v=((2, 29, 2, 64), F16)), INVALID), (dict(k=((3, 30, 2, 64), F16), v=((3, 30, 2, 64), F16)), INVALID),
    (dict(k=((2, 30, 3, 64), F16), v=((2, 30, 3, 64), F16)), INVALID), (dict(k=((2, 30, 0, 64), F16), v=((2, 30, 0, 64), F16)), INVALID),
    (dict(k=((2, 30, 2, 32), F16), v=((2, 30, 2, 32), F16)), INVALID), (dict(ql=((3,), I32)), INVALID), (dict(kl=((2, 1), I32)), INVALID),
    (dict(ql=((2,), F32)), INVALID), (dict(scale=0.0), INVALID), (dict(scale=-1.0), INVALID), (dict(scale=float("nan")), INVALID),
    (dict(scale=float("inf")), INVALID), (dict(left=-1), INVALID), (dict(right=-1), INVALID), (dict(sinks=-1), INVALID),
    (dict(out=((2, 9, 4, 63), F16)), INVALID), (dict(out=((2, 9, 4, 64), F32)), INVALID), (dict(lse=((2, 9, 4), F32)), INVALID),
    (dict(lse=((2, 4, 9), F16)), INVALID)]


@pytest.mark.parametrize("kw,status", [
    ({}, 0), (dict(ql=None, kl=None, lse=None), 0), (dict(left=2 ** 63 - 1, right=2 ** 63 - 1, sinks=2 ** 63 - 1), 0),
    (dict(k=((2, 0, 2, 64), F16), v=((2, 0, 2, 64), F16)), 0),
    (dict(q=((2, 9, 4, 257), F16), k=((2, 30, 2, 257), F16), v=((2, 30, 2, 257), F16), out=((2, 9, 4, 257), F16)), INVALID),
    (dict(q=((2, 9, 4, 0), F16), k=((2, 30, 2, 0), F16), v=((2, 30, 2, 0), F16), out=((2, 9, 4, 0), F16)), INVALID)] + REFUSED)
def test_attention(phase1, kw, status):
    assert phase1("opscvWindowAttention", *changed(ATTENTION, **kw))[0] == status


def backward(**kw):
    a = dict(ATTENTION, **kw)
    shape, keys = a["q"], a["k"]
    return [kw.get("go", shape), a["q"], a["k"], a["v"], a["out"], a["lse"], a["ql"], a["kl"], a["scale"], a["left"], a["right"],
            a["sinks"], kw.get("gq", shape), kw.get("gk", keys), kw.get("gv", a["v"])]


@pytest.mark.parametrize("kw,status", [({}, 0), (dict(ql=None, kl=None), 0), (dict(lse=None), NULLPTR), (dict(go=None), NULLPTR),
                                       (dict(gq=None), NULLPTR), (dict(gk=None), NULLPTR), (dict(gv=None), NULLPTR),
                                       (dict(go=((2, 9, 4, 64), F32)), INVALID), (dict(gq=((2, 9, 2, 64), F16)), INVALID),
                                       (dict(gk=((2, 30, 4, 64), F16)), INVALID), (dict(gv=((2, 30, 2, 64), BF16)), INVALID)] + REFUSED)
def test_attention_gradients(phase1, kw, status):
    st, ws, variant = phase1("opscvWindowAttentionBackward", *backward(**kw))
    assert st == status
    if status == 0:
        assert variant == "attention_grad" and ws >= 3 * 4 * 2 * 4 * 9  # statistics of every row


def test_attention_splits_and_workspace(phase1):
    """Few rows on many keys are cut into parts, whose results need workspace; many rows are not."""
    def variant(b, sq, skv, heads, kv_heads, d, dtype, left=2 ** 62):
        q, kv = ((b, sq, heads, d), dtype), ((b, skv, kv_heads, d), dtype)
        st, ws, name = phase1("opscvWindowAttention", q, kv, kv, None, None, 0.1, left, 0, 0, q, None)
        assert st == 0
        return name, ws
    assert variant(1, 1, 16384, 8, 1, 128, BF16)[0] == "attention_few_rows_split"
    name, ws = variant(1, 1, 16384, 8, 1, 128, BF16)
    assert ws > 0 and ws % (8 * (2 + 128) * 4) == 0  # per part: a row's largest score, its sum, and its values
    assert variant(1, 1, 16384, 8, 1, 128, BF16, left=100) == ("attention_few_rows", 0)
    assert variant(8, 4096, 4096, 16, 16, 64, F16) == ("attention_rows", 0)
    assert variant(8, 4096, 4096, 16, 16, 64, F32) == ("attention_few_rows", 0)
    q = ((2, 9, 4, 64), F16)
    apart = ((2, 30, 2, 64), F16, [30 * 500, 500, 100, 1])  # used in place
    gaps = ((2, 30, 2, 64), F16, [30 * 500, 500, 128, 2])   # packed
    over = ((2, 30, 2, 64), F16, [0, 0, 64, 1])             # tokens that lie on one another are packed
    for key, packed in ((apart, 0), (gaps, 1), (over, 1)):
        st, ws, _ = phase1("opscvWindowAttention", *changed(ATTENTION, k=key))
        assert st == 0 and (ws > 0) == bool(packed)


def test_null_outputs_of_the_first_phase(aclnn):
    L = aclnn.load_library()
    ex = ctypes.c_void_p(None)
    assert L.opscvRotaryTableGetWorkspaceSize(1e4, 0, 1.0, 0, 1.0, None, None, ctypes.byref(ex)) == NULLPTR


def test_second_phases_refuse(aclnn, phase1):
    """No executor, another operator's executor, no workspace, and NULL data: refused before anything is launched."""
    L = aclnn.load_library()
    for name in ("ResidualNorm", "ResidualNormBackward", "RotaryTable", "Rotary", "WindowAttention", "WindowAttentionBackward"):
        assert getattr(L, "opscv" + name)(None, 0, None, None) == NULLPTR

    def executor(name, *args):
        ws, ex = ctypes.c_uint64(0), ctypes.c_void_p(None)
        made = [phase1.t(x) if isinstance(x, tuple) else x for x in args]
        assert getattr(L, name + "GetWorkspaceSize")(*made, ctypes.byref(ws), ctypes.byref(ex)) == 0
        return ws.value, ex
    _, ex = executor("opscvResidualNorm", *NORM.values())
    assert L.opscvRotary(None, 0, ex, None) == INVALID
    _, ex = executor("opscvResidualNorm", *NORM.values())
    assert L.opscvResidualNorm(None, 0, ex, None) == NULLPTR
    ws, ex = executor("opscvWindowAttentionBackward", *backward())
    assert ws > 0 and L.opscvWindowAttentionBackward(None, 0, ex, None) == NULLPTR
    ws, ex = executor("opscvWindowAttentionBackward", *backward())
    assert L.opscvWindowAttentionBackward(ctypes.c_void_p(4096), ws - 1, ex, None) == INVALID
