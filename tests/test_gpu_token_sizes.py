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


@pytest.mark.parametrize("heads,kv_heads,d,rot,interleaved", [
    ((1 << 20) + 5, (1 << 20) + 3, 6, 6, False), ((1 << 20) + 5, 2, 8, 8, True), (3, (2 << 20) + 1, 4, 2, False),
    ((1 << 24) + (1 << 16), 0, 1023, 2, False)])
def test_rotary_of_very_many_heads(device, aclnn, heads, kv_heads, d, rot, interleaved):
    """More heads of a token than the threads of a launch have numbers for, or than one launch takes: as a few of them alone."""
    table = aclnn.rotary_table(torch.empty(0, device=device), 3, rot)
    positions = torch.tensor([[2]], device=device)
    made = []
    for n in (heads, kv_heads):
        x = torch.empty(1, 1, n, d, dtype=torch.bfloat16, device=device)
        for part in x[0, 0].split(1 << 22):
            part.normal_()
        made.append(x if n else None)
    # the first, the last, and those where spans of heads meet
    places = [[slice(a, a + 70) for a in (0, (1 << 20) - 20, (1 << 21) - 30, (1 << 24) - 40, max(0, n - 70)) if a < n] for n in (heads, kv_heads)]
    kept = [[x[:, :, p].clone() for p in ps] if x is not None else [] for x, ps in zip(made, places)]
    aclnn.rotary(made[0], made[1], table, positions=positions, interleaved=interleaved, query_out=made[0], key_out=made[1])
    for x, ps, before in zip(made, places, kept):
        for p, b in zip(ps, before):
            assert torch.equal(x[:, :, p], aclnn.rotary(b, None, table, positions=positions, interleaved=interleaved)[0]), p


@pytest.mark.parametrize("rows,width", [(3, (1 << 25) + 33), (1, (1 << 29) + 33)])
def test_norm_gradients_of_very_long_rows(device, aclnn, rows, width):
    """Rows whose columns are more than a launch of the weight's gradient holds side by side."""
    h, gy = (normal(device, s, rows, width, dtype=torch.bfloat16) for s in (1, 2))
    w = normal(device, 3, width, dtype=torch.bfloat16)
    rstd = torch.full((rows,), 0.75, device=device)
    gx, gw = aclnn.residual_norm_backward(gy, h, w, rstd)
    mean = torch.zeros(rows, dtype=torch.float64, device=device)
    parts = [slice(i, min(i + (1 << 24), width)) for i in range(0, width, 1 << 24)]
    for p in parts:
        mean += (gy[:, p].double() * w[p].double() * h[:, p].double() * 0.75).sum(1) / width
    for p in parts:
        n, g = h[:, p].double() * 0.75, gy[:, p].double()
        want = (g * w[p].double() - n * mean[:, None]) * 0.75
        assert ((gx[:, p].double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5 * ((g * w[p].double()).abs() + n.abs())).all()
        want = (g * n).sum(0)
        assert ((gw[p].double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5 * (g * n).abs().sum(0)).all()
