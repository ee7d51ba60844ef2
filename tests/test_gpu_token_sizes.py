"""The operators on token sequences at sizes that pass what one launch holds, against plain products in 32 bits on the GPU."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -23}


def normal(device, seed, *size, dtype):
    g = torch.Generator(device=device).manual_seed(seed)
    return torch.randn(*size, generator=g, device=device, dtype=dtype)


def check_tokens(aclnn, device, dtype, batch, heads, keys, d):
    """Single tokens of many sequences, every head with keys of its own, and their gradients, some sequences at a time."""
    q, go = normal(device, 1, batch, 1, heads, d, dtype=dtype), normal(device, 2, batch, 1, heads, d, dtype=dtype)
    k, v = normal(device, 3, batch, keys, heads, d, dtype=dtype), normal(device, 4, batch, keys, heads, d, dtype=dtype)
    lengths = torch.full((batch,), keys, dtype=torch.int32, device=device)
    lengths[1::3] = keys - 1
    masks = dict(scale=0.5, kv_lengths=lengths)
    out, lse = aclnn.window_attention(q, k, v, need_lse=True, **masks)
    grads = aclnn.window_attention_backward(go, q, k, v, out, lse, **masks)
    torch.cuda.synchronize()
    u = U[dtype]
    for b in torch.arange(batch, device=device).split(1 << 16):
        b = slice(int(b[0]), int(b[-1]) + 1)
        qf, kf, vf, gf = (t[b].float() for t in (q, k, v, go))
        s = (qf * kf).sum(-1) * 0.5
        s.masked_fill_((torch.arange(keys, device=device) >= lengths[b, None])[..., None], -torch.inf)
        w = torch.softmax(s, 1)
        o = (w[..., None] * vf).sum(1, keepdim=True)
        size = (w[..., None] * vf.abs()).sum(1, keepdim=True)
        assert ((out[b].float() - o).abs() <= 2 * u * size + 1e-5).all(), b
        assert ((lse[b][..., 0] - torch.logsumexp(s, 1)).abs() <= 1e-5).all(), b
        along = (gf * out[b].float()).sum(-1)
        slope = (gf * vf).sum(-1)
        gs = w * (slope - along) * 0.5
        off = w * ((gf * vf).abs().sum(-1) + (gf * o).abs().sum(-1)) * (2 * u)  # a rounding of gs and one of out
        for got, want, bound in ((grads[0], (gs[..., None] * kf).sum(1, keepdim=True), (off[..., None] * kf.abs()).sum(1, keepdim=True)),
                                 (grads[1], gs[..., None] * qf, off[..., None] * qf.abs()),
                                 (grads[2], w[..., None] * gf, 2 * u * w[..., None] * gf.abs())):
            assert ((got[b].float() - want).abs() <= bound + 2 * u * want.abs() + 1e-5).all(), b


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_tokens_of_hundreds_of_thousands_of_sequences(device, aclnn, dtype):
    """The pixels of a picture, each looking at the nine around it: 2.4 million workgroups."""
    check_tokens(aclnn, device, dtype, 300_000, 8, 9, 32)


def test_tokens_of_more_sequences_than_a_launch_holds(device, aclnn):
    """2^24 workgroups of 256 threads and a few: two launches."""
    check_tokens(aclnn, device, torch.bfloat16, (1 << 21) + 3, 8, 2, 8)
