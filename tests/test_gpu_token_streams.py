"""The operators on token sequences run on the stream that they are given, and read views with long strides in place."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = 27, 0


def normal(device, seed, *size, dtype=torch.bfloat16):
    g = torch.Generator(device=device).manual_seed(seed)
    return torch.randn(*size, generator=g, device=device).to(dtype)


def operators(aclnn):
    """Every operator as (call, shapes of its inputs): call(inputs, stream) returns its outputs."""
    def attend(i, s):
        return aclnn.window_attention(i[0], i[1], i[2], left=50, sinks=2, need_lse=True, stream=s)

    def attend_grad(i, s):  # on any numbers in place of out and lse
        return aclnn.window_attention_backward(i[3], i[0], i[1], i[2], i[4], i[5], left=50, sinks=2, stream=s)
    qkv = [(1, 300, 4, 64), (1, 300, 2, 64), (1, 300, 2, 64)]
    return {
        "norm": (lambda i, s: aclnn.residual_norm(i[0], i[1], i[2], need_rstd=True, stream=s), [(300, 512), (512,), (300, 512)]),
        "norm int8": (lambda i, s: aclnn.residual_norm_int8(i[0], i[1], i[2], stream=s), [(300, 512), (512,), (300, 512)]),
        "norm gradient": (lambda i, s: aclnn.residual_norm_backward(i[0], i[1], i[2], i[3], stream=s),
                          [(300, 512), (300, 512), (512,), (300,)]),
        "rotary": (lambda i, s: aclnn.rotary(i[0], i[1], i[3], stream=s), qkv + [(300, 64)]),
        "attention": (attend, qkv),
        "attention of a token": (attend, [(2, 1, 8, 64), (2, 9000, 1, 64), (2, 9000, 1, 64)]),  # two kernels
        "attention gradient": (attend_grad, qkv + [qkv[0], qkv[0], (1, 4, 300)]),
    }


@pytest.mark.parametrize("name", ["norm", "norm int8", "norm gradient", "rotary", "attention", "attention of a token",
                                  "attention gradient"])
def test_the_stream_that_is_given(device, aclnn, name):
    """The inputs come late, behind long work on a side stream: a kernel on any other stream would read what they held before."""
    call, shapes = operators(aclnn)[name]
    floats = {"norm gradient": (3,), "rotary": (3,), "attention gradient": (5,)}.get(name, ())
    real = [normal(device, 10 + i, *s, dtype=torch.float32 if i in floats else torch.bfloat16) for i, s in enumerate(shapes)]
    want = call(real, None)
    late = [torch.zeros_like(t) for t in real]
    call(late, None)  # the kernels are loaded
    a = normal(device, 1, 8192, 8192)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(20):
            b = a @ a
        for x, y in zip(late, real):
            x.copy_(y)
    queued = torch.cuda.Event()
    queued.record(side)
    got = call(late, side)
    assert not queued.query()  # the inputs have not come yet
    torch.cuda.synchronize()
    assert b.shape == a.shape
    for x, y in zip(got, want):
        assert (x is None) == (y is None) and (x is None or torch.equal(x, y))


def workspace(aclnn, heads, table):
    """Bytes that the rotation of `heads` (dims, strides) into a dense tensor asks for."""
    L = aclnn.load_library()
    made = [aclnn.create_tensor(heads[0], BF16, strides=heads[1], storage_dims=[1 << 40]), aclnn.create_tensor(table, F32),
            aclnn.create_tensor(heads[0], BF16)]
    ws, ex = ctypes.c_uint64(0), ctypes.c_void_p(None)
    assert L.opscvRotaryGetWorkspaceSize(made[0], None, None, made[1], False, False, made[2], None, ctypes.byref(ws),
                                         ctypes.byref(ex)) == 0
    aclnn.destroy_executor(ex.value)
    for h in made:
        aclnn.destroy_tensor(h)
    return ws.value


@pytest.mark.parametrize("dims,strides", [((2, 3, 2, 64), (2_299_000_000, 128, 64, 1)), ((1, 3, 2, 64), (0, 64, 2_299_000_000, 1))])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_of_sequences_and_heads_far_apart(device, aclnn, dims, strides, interleaved):
    """Sequences, or heads, 4.6 GB apart, read and written where they are."""
    big = torch.zeros(2_300_000_000, dtype=torch.bfloat16, device=device)
    far = torch.as_strided(big, dims, strides, 0)
    x = normal(device, 3, *dims)
    far.copy_(x)
    table = aclnn.rotary_table(x, 64, 64)
    assert workspace(aclnn, (dims, strides), (64, 64)) == 0
    want = aclnn.rotary(x, None, table, interleaved=interleaved)[0]
    assert torch.equal(aclnn.rotary(far, None, table, interleaved=interleaved)[0], want)
    aclnn.rotary(far, None, table, interleaved=interleaved, query_out=far)
    assert torch.equal(far, want)
    far.zero_()
    assert not big.any()
