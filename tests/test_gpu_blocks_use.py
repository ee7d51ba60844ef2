"""Layer norm, rotary positions on several axes, dropout and gated projections as programs use them: on a given stream, under
graph capture, on memory past 32-bit offsets, on expanded and repeated tensors, and together in a block."""
import os
import subprocess
import sys

import pytest
import torch

import block_oracle as B

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32 = torch.float32


def normal(device, seed, *size, dtype=torch.bfloat16, scale=1.0):
    g = torch.Generator(device=device).manual_seed(seed)
    return (torch.randn(*size, generator=g, device=device) * scale).to(dtype)


def close(got, want, off, dtype, what):
    B.within(got, want.cpu(), (off + B.U[dtype] * want.abs() + B.TINY[dtype]).cpu(), what)


def places(device, tokens, batch=1):
    i = torch.arange(tokens, device=device)
    return torch.stack([i // 12, i // 4 % 3, i % 4])[:, None].expand(-1, batch, -1)


def operators(aclnn, device):
    """Every operator as (call, sizes of its inputs): call(inputs, stream) returns its outputs."""
    state, at = torch.tensor([5, 6], device=device), places(device, 300)
    table = aclnn.rotary_table(state, 100, 64)

    def gated(i, s):
        return aclnn.gated_projection(*i, need_sums=True, stream=s)

    def gated_grad(i, s):
        return aclnn.gated_projection_backward(*i, activation=1, need_bias=True, stream=s)
    return {
        "norm": (lambda i, s: aclnn.layer_norm(i[0], i[1], i[2], i[3], need_stats=True, stream=s),
                 [(300, 512), (512,), (512,), (300, 512)]),
        "norm gradient": (lambda i, s: aclnn.layer_norm_backward(i[0], i[1], i[2], i[3], i[4], stream=s),
                          [(300, 512), (300, 512), (512,), (300,), (300,)]),
        "rotary": (lambda i, s: aclnn.rotary_axes(i[0], i[1], table, at, (12, 10, 10), stream=s), [(1, 300, 4, 64), (1, 300, 2, 64)]),
        "dropout": (lambda i, s: (aclnn.dropout(i[0], state, 0.3, i[1], stream=s),), [(300, 512), (300, 512)]),
        "gated, few rows": (gated, [(5, 512), (700, 512), (700, 512)]),
        "gated, tiles": (gated, [(300, 136), (520, 136), (520, 136)]),
        "gated, copies and parts": (gated, [(130, 1030), (70, 1030), (70, 1030)]),  # three kernels
        "gated gradient": (gated_grad, [(300, 70), (300, 130), (70, 130), (70, 130), (300, 70), (300, 70)]),
    }


@pytest.fixture(scope="module")
def side(device):
    return torch.cuda.Stream()


NAMES = ["norm", "norm gradient", "rotary", "dropout", "gated, few rows", "gated, tiles", "gated, copies and parts", "gated gradient"]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("name", NAMES)
def test_the_stream_that_is_given(device, aclnn, side, name, dtype):
    """The inputs come late, behind long work on a side stream: a kernel on any other stream would read what they held before."""
    call, sizes = operators(aclnn, device)[name]
    statistics = (3, 4) if name == "norm gradient" else ()
    real = [normal(device, 10 + i, *s, dtype=F32 if i in statistics else dtype) for i, s in enumerate(sizes)]
    want = call(real, None)
    late = [torch.zeros_like(t) for t in real]
    call(late, None)  # the kernels are loaded
    a = torch.ones(1 << 28, device=device)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):  # some 400 us each
            a.mul_(1.0)
        for x, y in zip(late, real):
            x.copy_(y)
    queued = torch.cuda.Event()
    queued.record(side)
    got = call(late, side)
    assert not queued.query()  # the inputs have not come yet
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        assert (x is None) == (y is None) and (x is None or torch.equal(x, y))


def replays(device, make, call, outputs, bytes=64 << 20):
    """Records call(inputs, outputs, workspace) and replays it on other inputs, with eager work between the replays."""
    inputs, ws = make(0), torch.empty(bytes, dtype=torch.uint8, device=device)
    made = outputs()
    call(inputs, made, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(inputs, made, ws)
    for seed in (1, 2, 3, 4):
        fresh = make(seed)
        for a, b in zip(inputs, fresh):
            a.copy_(b)
        for t in made:
            t.fill_(7)
        ws.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        want = outputs()
        call(fresh, want, torch.empty_like(ws))
        torch.cuda.synchronize()
        for a, b in zip(made, want):
            assert torch.equal(a, b), seed


@pytest.mark.parametrize("rows,width", [(70, 512), (700, 1031), (3, 40000)])
def test_norm_in_a_graph(device, aclnn, rows, width):
    def new(*size, dtype=torch.bfloat16):
        return torch.empty(*size, dtype=dtype, device=device)
    replays(device, lambda s: [normal(device, s + 10 * i, *n) for i, n in enumerate([(rows, width)] * 3 + [(width,)] * 2)],
            lambda i, o, ws: (aclnn.layer_norm(i[0], i[3], i[4], i[1], out=o[0], sum_out=o[1], mean_out=o[2], rstd_out=o[3],
                                               need_stats=True, workspace=ws),
                              aclnn.layer_norm_backward(i[2], o[1], i[3], o[2], o[3], grad_sum=i[0], grad_x=o[4], grad_weight=o[5],
                                                        grad_bias=o[6], workspace=ws)),
            lambda: [new(rows, width), new(rows, width), new(rows, dtype=F32), new(rows, dtype=F32), new(rows, width), new(width),
                     new(width)])


def test_rotary_and_dropout_in_a_graph(device, aclnn):
    """The positions and the generator's state are read at every replay."""
    table = aclnn.rotary_table(torch.empty(0, device=device), 200, 64)
    replays(device, lambda s: [normal(device, s, 2, 48, 4, 64), normal(device, s + 9, 2, 48, 2, 64), places(device, 48, 2) + s,
                               torch.tensor([17, s], device=device)],
            lambda i, o, ws: (aclnn.rotary_axes(i[0], i[1], table, i[2], (12, 10, 10), query_out=o[0], key_out=o[1], workspace=ws),
                              aclnn.dropout(o[0], i[3], 0.25, i[0], out=o[2], workspace=ws)),
            lambda: [torch.empty(2, 48, h, 64, dtype=torch.bfloat16, device=device) for h in (4, 2, 4)])


def test_dropout_state_that_a_graph_advances(device, aclnn):
    """A recorded step that adds one to the offset: each replay draws the mask of an eager call with that offset."""
    x, state = normal(device, 1, 100, 520), torch.tensor([3, 2 ** 31 - 2], device=device)  # the offset's words: past the lower
    aclnn.dropout(x, state, 0.5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = aclnn.dropout(x, state, 0.5)
        state[1] += 1
    seen = []
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, aclnn.dropout(x, torch.tensor([3, 2 ** 31 - 2 + i], device=device), 0.5))
        seen.append(y == 0)
    assert all(not torch.equal(a, b) for a, b in zip(seen, seen[1:]))
    assert state.tolist() == [3, 2 ** 31 + 2]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,width,inner", [(5, 512, 700), (300, 136, 520), (130, 1030, 70), (513, 2056, 1100)])
def test_gated_in_a_graph(device, aclnn, dtype, rows, width, inner):
    def new(*size):
        return torch.empty(*size, dtype=dtype, device=device)
    sizes = [(rows, width), (inner, width), (inner, width), (inner,), (inner,), (rows, inner)]
    replays(device, lambda s: [normal(device, s + 10 * i, *n, dtype=dtype, scale=0.5) for i, n in enumerate(sizes)],
            lambda i, o, ws: (aclnn.gated_projection(*i[:5], out=o[0], gate_out=o[1], up_out=o[2], need_sums=True, workspace=ws),
                              aclnn.gated_projection_backward(i[5], *i[:3], o[1], o[2], grad_x=o[3], grad_gate_weight=o[4],
                                                              grad_up_weight=o[5], grad_gate_bias=o[6], grad_up_bias=o[7],
                                                              need_bias=True, workspace=ws)),
            lambda: [new(rows, inner), new(rows, inner), new(rows, inner), new(rows, width), new(inner, width), new(inner, width),
                     new(inner), new(inner)], bytes=256 << 20)


def test_two_graphs_of_one_workspace(device, aclnn):
    """Replayed one after the other in either order: nothing of one call is left in the workspace for the next."""
    ws = torch.empty(64 << 20, dtype=torch.uint8, device=device)
    sizes = [((130, 1030), (70, 1030)), ((200, 519), (130, 519))]
    inputs = [(normal(device, i, *x), normal(device, i + 2, *w, scale=0.1), normal(device, i + 4, *w, scale=0.1)) for i, (x, w) in enumerate(sizes)]
    want = [aclnn.gated_projection(*i)[0] for i in inputs]
    graphs, made = [], []
    torch.cuda.synchronize()
    for i in inputs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            made.append(aclnn.gated_projection(*i, workspace=ws)[0])
    for order in ((0, 1), (1, 0), (0, 0, 1), (1, 1, 0)):
        for k in order:
            graphs[k].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(made, want))


def test_rows_far_apart(device, aclnn):
    """Two rows 4.6 GB apart in every operand that may have them."""
    big = torch.zeros(2_300_000_000, dtype=torch.bfloat16, device=device)
    w, b = normal(device, 2, 1000), normal(device, 3, 1000)
    x, r = normal(device, 4, 2, 1000), normal(device, 5, 2, 1000)

    def far(i, t):
        v = torch.as_strided(big, tuple(t.shape), (2_299_000_000, 1), i * 10_000)
        v.copy_(t)
        return v
    out = far(2, torch.zeros_like(x))
    want = aclnn.layer_norm(x, w, b, r, need_stats=True)
    got = aclnn.layer_norm(far(0, x), w, b, far(1, r), need_stats=True, out=out, sum_out=far(3, x))
    assert all(torch.equal(s, t) for s, t in zip(got, want)) and torch.equal(out, want[0])
    grad = aclnn.layer_norm_backward(x, want[1], w, *want[2:], grad_sum=r)
    got = aclnn.layer_norm_backward(far(0, x), far(3, want[1]), w, *want[2:], grad_sum=far(1, r), grad_x=out)
    assert all(torch.equal(s, t) for s, t in zip(got, grad)) and torch.equal(out, grad[0])
    state = torch.tensor([1, 2], device=device)
    aclnn.dropout(far(0, x), state, 0.5, far(1, r), out=out)
    assert torch.equal(out, aclnn.dropout(x, state, 0.5, r))
    weights = [normal(device, 6 + i, 2, 1000, scale=0.03) for i in range(2)]
    sums = [far(i, torch.zeros(2, 2)) for i in (2, 3, 4)]
    want = aclnn.gated_projection(x, *weights, need_sums=True)
    got = aclnn.gated_projection(far(0, x), far(5, weights[0]), far(6, weights[1]), out=sums[0], gate_out=sums[1], up_out=sums[2],
                                 need_sums=True)
    assert all(torch.equal(s, t) and torch.equal(u, t) for s, t, u in zip(got, want, sums))
    gy = normal(device, 9, 2, 2)
    grad = aclnn.gated_projection_backward(gy, x, *weights, *want[1:])
    got = aclnn.gated_projection_backward(far(2, gy), far(0, x), far(5, weights[0]), far(6, weights[1]), sums[1], sums[2],
                                          grad_x=far(7, x), grad_gate_weight=far(8, x), grad_up_weight=far(9, x))
    assert all(torch.equal(s, t) for s, t in zip(got[:3], grad[:3]))


def test_heads_and_positions_far_apart(device, aclnn):
    big = torch.zeros(2_300_000_000, dtype=torch.bfloat16, device=device)
    x = normal(device, 1, 2, 30, 2, 64)
    table = aclnn.rotary_table(x, 64, 64)
    at = places(device, 30, 2)
    want = aclnn.rotary_axes(x, None, table, at, (12, 10, 10))[0]
    for strides in ((2_298_000_000, 128, 64, 1), (6400, 64, 2_298_000_000, 1)):
        far = torch.as_strided(big, (2, 30, 2, 64), strides, 0)
        far.copy_(x)
        assert torch.equal(aclnn.rotary_axes(far, None, table, at, (12, 10, 10), query_out=far)[0], want)
    del big
    wide = torch.zeros(3, 300_000_000, dtype=torch.int64, device=device)  # axes 2.4 GB apart
    rows = torch.as_strided(wide, (3, 2, 30), (300_000_000, 40, 1), 0)
    rows.copy_(at)
    assert torch.equal(aclnn.rotary_axes(x, None, table, rows, (12, 10, 10))[0], want)


def test_norm_and_dropout_past_32_bits(device, aclnn):
    """More than 2^32 elements: the last rows are those of a small call, the last masks those of the generator."""
    rows, width = 70_000, 65_536
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device=device)
    x[-3:] = normal(device, 1, 3, width)
    w, b = normal(device, 2, width), normal(device, 3, width)
    y, _, mean, rstd = aclnn.layer_norm(x, w, b, need_stats=True)
    few = aclnn.layer_norm(x[-3:].clone(), w, b, need_stats=True)
    assert torch.equal(y[-3:], few[0]) and torch.equal(mean[-3:], few[2]) and torch.equal(rstd[-3:], few[3])
    assert torch.equal(y[12345], b)
    gx = aclnn.layer_norm_backward(y, x, w, mean, rstd, need_weight=False, need_bias=False, grad_x=y)[0]
    assert torch.equal(gx[-3:], aclnn.layer_norm_backward(few[0], x[-3:].clone(), w, few[2], few[3], need_weight=False, need_bias=False)[0])
    state = torch.tensor([7, -1], device=device)
    x.fill_(1)
    aclnn.dropout(x, state, 0.5, out=y)
    first = rows * width - 4096
    words = torch.from_numpy(B.philox(range(first // 8, rows * width // 8), -1 % 2 ** 64, 7).astype("int64"))
    keep = torch.stack([words & 0xffff, words >> 16], -1).flatten() >= 32768
    assert torch.equal(y.flatten()[first:].cpu(), keep.to(torch.bfloat16) * 2)


def test_gated_past_32_bits(device, aclnn):
    """Outputs, and what the backward pass keeps, of more than 2^32 bytes; rows and features of them against 64 bits."""
    rows, width, inner = 140_000, 16, 16_384
    x, weights = normal(device, 1, rows, width), [normal(device, 2 + i, inner, width, scale=0.25) for i in range(2)]
    y, gate, up = aclnn.gated_projection(x, *weights, need_sums=True)
    some = torch.tensor([0, 255, 65_535, rows - 300, rows - 1], device=device)
    want, off = B.gated(x[some], *weights, None, None, 0)
    for t, w, e, what in zip((y, gate, up), want, off, ("y", "gate", "up")):
        close(t[some], w, e, "bf16", what)
    gy = y
    gx, *gw = aclnn.gated_projection_backward(gy, x, *weights, gate, up)[:3]
    want, off = B.gated_grad(gy[some], x[some], *weights, gate[some], up[some], 0, "bf16")
    close(gx[some], want[0], off[0], "bf16", "gradient of x")
    for f in (0, 8191, inner - 1):
        at = slice(f, f + 1)
        want, off = B.gated_grad(gy[:, at], x, weights[0][at], weights[1][at], gate[:, at], up[:, at], 0, "bf16")
        for i in range(2):
            close(gw[i][at], want[1 + i], off[1 + i], "bf16", "gradient of a weight")


def test_expanded_gradients(device, aclnn):
    """Gradients as a sum's backward pass hands them on: one number, or one row, with strides of zero."""
    x, w, b = normal(device, 1, 30, 520), normal(device, 2, 520), normal(device, 3, 520)
    _, _, mean, rstd = aclnn.layer_norm(x, w, b, need_stats=True)
    weights = [normal(device, 4 + i, 70, 520, scale=0.05) for i in range(2)]
    _, gate, up = aclnn.gated_projection(x, *weights, need_sums=True)
    state = torch.tensor([1, 0], device=device)
    for width, call in ((520, lambda g: aclnn.layer_norm_backward(g, x, w, mean, rstd, grad_sum=g)),
                        (70, lambda g: aclnn.gated_projection_backward(g, x, *weights, gate, up, need_bias=True)),
                        (520, lambda g: (aclnn.dropout(g, state, 0.5, g),))):
        for g in (normal(device, 6, 1, 1), normal(device, 7, 1, width), normal(device, 8, 30, 1)):
            for s, t in zip(call(g.expand(30, width)), call(g.expand(30, width).contiguous())):
                assert torch.equal(s, t)
    row = x[:1].expand(30, 520)  # the rows of x itself
    assert torch.equal(aclnn.layer_norm(row, w, b, row)[0], aclnn.layer_norm(row.contiguous(), w, b, row.contiguous())[0])
    assert torch.equal(aclnn.gated_projection(row, *weights)[0], aclnn.gated_projection(row.contiguous(), *weights)[0])


@pytest.mark.parametrize("dtype", list(B.DTYPES))
def test_one_tensor_twice(device, aclnn, dtype):
    x, w = (normal(device, i, *s, dtype=B.DTYPES[dtype], scale=0.3) for i, s in ((1, (70, 200)), (2, (200, 200))))
    v = x[0].contiguous()
    assert torch.equal(aclnn.layer_norm(x, v, v, x)[0], aclnn.layer_norm(x, v.clone(), v.clone(), x.clone())[0])
    got = aclnn.gated_projection(x, w, w, v, v, need_sums=True)
    assert torch.equal(got[1], got[2])
    assert all(torch.equal(s, t) for s, t in zip(got, aclnn.gated_projection(x, w, w.clone(), v, v.clone(), need_sums=True)))
    grads = aclnn.gated_projection_backward(x, x, w, w, x, x, need_bias=True)
    want = aclnn.gated_projection_backward(x, x.clone(), w, w.clone(), x.clone(), x.clone(), need_bias=True)
    assert all(torch.equal(s, t) for s, t in zip(grads, want))
    state = torch.tensor([1, 2], device=device)
    assert torch.equal(aclnn.dropout(x, state, 0.5, x), aclnn.dropout(x, state, 0.5, x.clone()))
    q = x.view(1, 70, 2, 100)
    table, at = aclnn.rotary_table(x, 100, 20), places(device, 70)
    got = aclnn.rotary_axes(q, q, table, at, (2, 4, 4))
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], aclnn.rotary_axes(q, None, table, at, (2, 4, 4))[0])


def example():
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import video_block
    finally:
        sys.path.pop(0)
    return video_block


def plain_block(p, x, table, places, masks, scale, heads, d, sections):
    """The example's block in 64 bits by torch's own functions; p: its parameters."""
    F = torch.nn.functional
    b, n, _ = x.shape

    def turn(t):
        pairs = B.pairs_of(sections, 0)
        half, parts = len(pairs), []
        for i, (axis, column) in enumerate(pairs):
            row = table[places[axis]]
            cos, sin = row[..., column][..., None], row[..., half + column][..., None]
            parts.append((t[..., i] * cos - t[..., half + i] * sin, t[..., half + i] * cos + t[..., i] * sin))
        return torch.cat([torch.stack([q[k] for q in parts], -1) for k in range(2)] + [t[..., 2 * half:]], -1)
    y = F.layer_norm(x, x.shape[-1:], p["norm1"], p["shift1"], 1e-5)
    q, k, v = (y @ p["into"].t()).view(b, n, 3, heads, d).unbind(2)
    q, k = turn(q), turn(k)
    weight = torch.softmax(q.transpose(1, 2) @ k.permute(0, 2, 3, 1) * d ** -0.5, -1)
    x = x + masks[0] * scale * ((weight @ v.transpose(1, 2)).transpose(1, 2).flatten(2) @ p["back"].t())
    y = F.layer_norm(x, x.shape[-1:], p["norm2"], p["shift2"], 1e-5)
    y = F.gelu(y @ p["gate"].t() + p["gate_bias"], approximate="tanh") * (y @ p["up"].t() + p["up_bias"])
    return x + masks[1] * scale * (y @ p["down"].t())


def test_a_block(device, aclnn):
    """The operators together, forward and backward: the example's block in 32 bits against the same mathematics in 64.

    About twenty operators stand between the input and the last gradient, each off by F32 of its result at most; none makes a
    relative error more than a few times larger (norms of rows of unit spread, slopes under 1.2, scores about 1): 20 * 5 * F32
    of a result's norm."""
    E = example()
    torch.manual_seed(0)
    b, n, width, heads, d, inner, sections, p = 2, 60, 96, 2, 48, 136, (4, 8, 8), 0.25
    block = E.Block(width, heads, d, inner, sections, aclnn.GATE_GELU_TANH, torch.float32, device)
    with torch.no_grad():
        for name in ("norm1", "shift1", "norm2", "shift2", "gate_bias", "up_bias"):
            getattr(block, name).add_(torch.randn_like(getattr(block, name)) * 0.2)
    x = torch.randn(b, n, width, device=device, requires_grad=True)
    grad = torch.randn(b, n, width, device=device)
    table, at = aclnn.rotary_table(x.detach(), 32, 2 * sum(sections)), places(device, n, b)
    states = torch.tensor([[9, 4], [9, 5]], device=device)
    y = block(x, table, at, states, p)
    y.backward(grad)
    masks = [torch.from_numpy(B.numbers(x.numel(), 9, k) >= 16384).view(b, n, width).double() for k in (4, 5)]
    plain = {k: v.detach().double().cpu().requires_grad_() for k, v in block.named_parameters()}
    x64 = x.detach().double().cpu().requires_grad_()
    want = plain_block(plain, x64, table.double().cpu(), at.cpu(), masks, 1 / (1 - p), heads, d, sections)
    want.backward(grad.double().cpu())
    pairs = [("y", y, want), ("x", x.grad, x64.grad)] + [(k, v.grad, plain[k].grad) for k, v in block.named_parameters()]
    for name, got, w in pairs:
        off = ((got.detach().double().cpu() - w).norm() / w.norm()).item()
        assert off < 20 * 5 * B.F32, (name, off)


def test_example(device):
    p = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "video_block.py"), "--steps", "3"], stdout=subprocess.PIPE,
                       stderr=subprocess.STDOUT, text=True, timeout=110, cwd=ROOT)
    assert p.returncode == 0, p.stdout
    assert "recorded answers" in p.stdout and "loss" in p.stdout


@pytest.mark.parametrize("heads,kv_heads,d,sections,layout", [((1 << 20) + 5, 3, 8, (1, 3), 0), (3, (2 << 20) + 1, 6, (1, 1), 2),
                                                              ((1 << 24) + (1 << 16), 0, 255, (0, 1), 1)])
def test_rotary_of_very_many_heads(device, aclnn, heads, kv_heads, d, sections, layout):
    """More heads of a token than one launch takes: as a few of them alone."""
    table = aclnn.rotary_table(torch.empty(0, device=device), 9, 2 * (max(sections) if layout == 1 else sum(sections)))
    at = torch.tensor([[[2, 5]], [[7, 3]]], device=device)
    made = [normal(device, 3, 1, 2, n, d) if n else None for n in (heads, kv_heads)]
    places_of = [[slice(a, a + 70) for a in (0, (1 << 20) - 20, (1 << 21) - 30, (1 << 24) - 40, max(0, n - 70)) if a < n]
                 for n in (heads, kv_heads)]
    kept = [[x[:, :, p].clone() for p in ps] if x is not None else [] for x, ps in zip(made, places_of)]
    aclnn.rotary_axes(made[0], made[1], table, at, sections, layout=layout, query_out=made[0], key_out=made[1])
    for x, ps, before in zip(made, places_of, kept):
        for p, b in zip(ps, before):
            assert torch.equal(x[:, :, p], aclnn.rotary_axes(b, None, table, at, sections, layout=layout)[0]), p


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_two_threads_call_at_once(device, aclnn, dtype):
    """First and second phases on two host threads, each on a stream of its own: the results of calls one after the other."""
    import threading

    def work(seed):
        x, w = normal(device, seed, 70, 264, dtype=dtype), [normal(device, seed + i, 130, 264, dtype=dtype, scale=0.1) for i in (1, 2)]
        state = torch.tensor([seed, 1], device=device)

        def calls():
            y = aclnn.layer_norm(x, None, None, x)[0]
            g = aclnn.gated_projection(y, *w, need_sums=True)
            return aclnn.gated_projection_backward(aclnn.dropout(g[0], state, 0.5), y, *w, *g[1:], need_bias=True)
        return calls
    jobs = [work(1), work(7)]
    want = [job() for job in jobs]
    torch.cuda.synchronize()
    got, failed = [None, None], []

    def run(i):
        try:
            for _ in range(30):
                got[i] = jobs[i]()
        except Exception as e:  # handed to the test's own thread
            failed.append(e)
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(s, t) for s, t in zip(a, b))


@pytest.mark.parametrize("dtype", list(B.DTYPES))
@pytest.mark.parametrize("rows,width", [(3, 1 << 19), (2, (1 << 20) + 24), (2, (1 << 20) + 9)])
def test_norms_of_very_long_rows(device, aclnn, dtype, rows, width):
    """Rows that no workgroup keeps in registers, forward and backward."""
    x, gy, w, b = (normal(device, i, *s, dtype=B.DTYPES[dtype]) for i, s in ((1, (rows, width)), (2, (rows, width)), (3, (width,)), (4, (width,))))
    want = B.layer_norm(*(t.cpu() for t in (x, x, w, b)), 1e-5)
    y, total, mean, rstd = aclnn.layer_norm(x, w, b, x, need_stats=True)
    close(y, want[0], want[4] + B.gamma(width / 1024) * want[1].abs() * want[3][:, None] * w.cpu().double().abs(), dtype, "norm")
    grads, off = B.layer_norm_grad(gy.cpu(), None, total.cpu(), w.cpu(), mean.cpu(), rstd.cpu())
    got = aclnn.layer_norm_backward(gy, total, w, mean, rstd)
    for t, g, o, what in zip(got, grads, off, ("x", "weight", "bias")):
        close(t, g, o, dtype, "gradient of " + what)


@pytest.mark.parametrize("rows,width", [(3, (1 << 25) + 33), (1, (1 << 29) + 33)])
def test_norm_gradients_of_very_many_columns(device, aclnn, rows, width):
    """Rows whose columns are more than a launch of the weight's gradient holds side by side."""
    h, gy, w = (normal(device, i, *s) for i, s in ((1, (rows, width)), (2, (rows, width)), (3, (width,))))
    mean, rstd = torch.full((rows,), 0.25, device=device), torch.full((rows,), 0.75, device=device)
    gx, gw, gb = aclnn.layer_norm_backward(gy, h, w, mean, rstd)
    parts = [slice(i, min(i + (1 << 24), width)) for i in range(0, width, 1 << 24)]
    along = torch.zeros(2, rows, 1, dtype=torch.float64, device=device)

    def values(p):
        return (h[:, p].double() - 0.25) * 0.75, gy[:, p].double(), w[p].double()
    for p in parts:
        n, g, v = values(p)
        along += torch.stack([(g * v).sum(1), (g * v * n).sum(1)])[..., None] / width
    for p in parts:
        n, g, v = values(p)
        want = (g * v - along[0] - n * along[1]) * 0.75
        assert ((gx[:, p].double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5 * ((g * v).abs() + 1 + n.abs())).all()
        for got, want, size in ((gw, (g * n).sum(0), (g * n).abs().sum(0)), (gb, g.sum(0), g.abs().sum(0))):
            assert ((got[p].double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5 * size).all()
