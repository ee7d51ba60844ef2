"""Tensors without elements whose strides are not those of a dense tensor, such as torch.empty(0, 128)[:, :64]: there is nothing
to pack, and a null address stands for them.  The second phases get past their operands, as far as the launch."""
import ctypes

import numpy as np
import pytest
import torch

from test_tokens_boundary import BF16, F32, I64, NULLPTR

R, V = ((0, 64), BF16, [128, 1]), ((0,), F32, [2])  # rows apart, every second number
O, W, P, B = ((0, 40), BF16, [80, 1]), ((64,), BF16), ((40, 64), BF16), ((40,), BF16)
Q, K = ((2, 0, 4, 64), BF16, [-4096, 256, 64, 1]), ((2, 3, 4, 64), BF16)  # no query: sequences backwards
CALLS = {
    "opscvLayerNormBackward": [R, R, R, W, V, V, R, W, W],
    "opscvResidualNormBackward": [R, R, R, W, V, R, W],
    "opscvGatedProjectionBackward": [O, R, P, P, O, O, 0, R, P, P, B, B],
    "opscvWindowAttentionBackward": [Q, Q, K, K, Q, ((2, 4, 0), F32, [-64, 8, 1]), None, None, 0.125, 2 ** 40, 2 ** 40, 0, Q, K, K],
    # a table of no positions: every turned pair becomes NaN
    "opscvRotary": [K, None, ((2, 3), I64), ((0, 64), F32, [64, 2]), False, False, K, None],
}


@pytest.mark.skipif(torch.cuda.is_available(), reason="the launch that follows would read host memory")
@pytest.mark.parametrize("name", list(CALLS))
def test_second_phase(aclnn, name):
    L, handles, kept = aclnn.load_library(), [], []

    def made(spec):
        if not isinstance(spec, tuple):
            return spec
        data = 0
        if 0 not in spec[0]:
            kept.append(np.zeros(int(np.prod(spec[0])) * 8 + 16, dtype=np.uint8))
            data = kept[-1].ctypes.data // 16 * 16 + 16
        strides = spec[2] if len(spec) > 2 else None
        handles.append(aclnn.create_tensor(spec[0], spec[1], strides=strides, storage_dims=[1 << 40] if strides else None, data=data))
        return handles[-1]
    ws, ex = ctypes.c_uint64(0), ctypes.c_void_p(None)
    assert getattr(L, name + "GetWorkspaceSize")(*[made(x) for x in CALLS[name]], ctypes.byref(ws), ctypes.byref(ex)) == 0
    memory = np.zeros(ws.value + 4096, dtype=np.uint8)
    status = getattr(L, name)(ctypes.c_void_p(memory.ctypes.data // 256 * 256 + 256), ws.value, ex, None)
    for h in handles:
        aclnn.destroy_tensor(h)
    assert status != NULLPTR and b"launch failed" in L.aclGetRecentErrMsg(), L.aclGetRecentErrMsg()


@pytest.mark.gpu
def test_gradients_of_no_rows(device, aclnn):
    """Those of columns and weights are zeros."""
    def none(width, n=64, dtype=torch.bfloat16):
        return torch.empty(0, width, device=device, dtype=dtype)[:, :n]
    w = torch.ones(64, device=device, dtype=torch.bfloat16)
    values = torch.empty(0, 2, device=device)[:, 0]
    gx, gw, gb = aclnn.layer_norm_backward(none(128), none(96), w, values, values, grad_sum=none(72), grad_x=none(100))
    assert gx.shape == (0, 64) and (gw == 0).all() and (gb == 0).all()
    gx, gw = aclnn.residual_norm_backward(none(128), none(96), w, values)
    assert gx.shape == (0, 64) and (gw == 0).all()
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        p = torch.ones(40, 64, device=device, dtype=dtype)
        got = aclnn.gated_projection_backward(none(80, 40, dtype), none(128, 64, dtype), p, p, none(50, 40, dtype), none(41, 40, dtype),
                                              need_bias=True)
        assert got[0].shape == (0, 64) and all((t == 0).all() for t in got[1:])
