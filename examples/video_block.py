"""A small video model: the sampler cuts a moving window out of pictures, and blocks of the token operators say where it moved.

Frames are cut into patches, whose positions are (frame, row, column). Each block is layer norm -> rotary positions on three axes
-> attention -> dropout with the residual -> layer norm -> gated projection -> dropout with the residual. Training differentiates
through the operators' backward forms; the answers come from a recorded graph. The remaining projections are torch's matrix
products. Pictures and weights are random.

    python examples/video_block.py [--steps 400]
"""
import argparse
import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from ops_cv_amd import aclnn  # noqa: E402

FRAMES, SIZE, PATCH, WAYS = 4, 64, 8, 4
WIDTH, HEADS, D, INNER, BLOCKS = 256, 4, 64, 704, 2
SECTIONS = (8, 12, 12)  # pairs of features turned by the frame, the row and the column


class Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        y, _, mean, rstd = aclnn.layer_norm(x, weight, bias, need_stats=True)
        ctx.save_for_backward(x, weight, mean, rstd)
        return y

    @staticmethod
    def backward(ctx, grad):
        return aclnn.layer_norm_backward(grad, *ctx.saved_tensors)


class Rotary(torch.autograd.Function):
    """Query and key turned by their positions; the gradient is turned back."""

    @staticmethod
    def forward(ctx, query, key, table, positions, sections):
        ctx.save_for_backward(table, positions)
        ctx.sections = sections
        return aclnn.rotary_axes(query, key, table, positions, sections)

    @staticmethod
    def backward(ctx, grad_query, grad_key):
        return (*aclnn.rotary_axes(grad_query, grad_key, *ctx.saved_tensors, ctx.sections, inverse=True), None, None, None)


class Attend(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, value):
        out, lse = aclnn.window_attention(query, key, value, right=query.shape[1], need_lse=True)
        ctx.save_for_backward(query, key, value, out, lse)
        return out

    @staticmethod
    def backward(ctx, grad):
        return aclnn.window_attention_backward(grad, *ctx.saved_tensors, right=grad.shape[1])


class Gated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate_weight, up_weight, gate_bias, up_bias, activation):
        y, gate, up = aclnn.gated_projection(x, gate_weight, up_weight, gate_bias, up_bias, activation, need_sums=True)
        ctx.save_for_backward(x, gate_weight, up_weight, gate, up)
        ctx.activation = activation
        return y

    @staticmethod
    def backward(ctx, grad):
        return (*aclnn.gated_projection_backward(grad, *ctx.saved_tensors, ctx.activation, need_bias=True), None)


class Drop(torch.autograd.Function):
    """residual + dropout(x); the backward pass computes the mask again from the state."""

    @staticmethod
    def forward(ctx, x, residual, state, p):
        ctx.save_for_backward(state)
        ctx.p = p
        return aclnn.dropout(x, state, p, residual)

    @staticmethod
    def backward(ctx, grad):
        return aclnn.dropout(grad, ctx.saved_tensors[0], ctx.p), grad, None, None


class Block(torch.nn.Module):
    def __init__(self, width, heads, d, inner, sections, activation, dtype, device):
        super().__init__()
        self.heads, self.d, self.sections, self.activation = heads, d, sections, activation

        def weight(*size):
            return torch.nn.Parameter((torch.randn(*size, device=device) * size[-1] ** -0.5).to(dtype))

        def vector(n, value):
            return torch.nn.Parameter(torch.full((n,), value, dtype=dtype, device=device))
        self.norm1, self.shift1, self.norm2, self.shift2 = vector(width, 1.0), vector(width, 0.0), vector(width, 1.0), vector(width, 0.0)
        self.into, self.back = weight(3 * heads * d, width), weight(width, heads * d)
        self.gate, self.up, self.down = weight(inner, width), weight(inner, width), weight(width, inner)
        self.gate_bias, self.up_bias = vector(inner, 0.0), vector(inner, 0.0)

    def forward(self, x, table, positions, states, p):
        """`states`: the seeds and offsets of both dropouts, (2, 2); without p they are not read."""
        def add(y, state):
            return Drop.apply(y, x, state, p) if p > 0.0 else x + y
        b, n, _ = x.shape
        y = Norm.apply(x, self.norm1, self.shift1)
        q, k, v = (y @ self.into.t()).view(b, n, 3, self.heads, self.d).unbind(2)
        q, k = Rotary.apply(q, k, table, positions, self.sections)
        x = add(Attend.apply(q, k, v).flatten(2) @ self.back.t(), states[0])
        y = Norm.apply(x, self.norm2, self.shift2)
        y = Gated.apply(y, self.gate, self.up, self.gate_bias, self.up_bias, self.activation)
        return add(y @ self.down.t(), states[1])


class Model(torch.nn.Module):
    def __init__(self, device):
        super().__init__()
        def weight(*size):  # noqa: E306
            return torch.nn.Parameter((torch.randn(*size, device=device) * size[-1] ** -0.5).bfloat16())
        self.patches, self.ways = weight(WIDTH, 3 * PATCH * PATCH), weight(WAYS, WIDTH)
        self.blocks = torch.nn.ModuleList([Block(WIDTH, HEADS, D, INNER, SECTIONS, aclnn.GATE_GELU_TANH, torch.bfloat16, device)
                                           for _ in range(BLOCKS)])
        n = SIZE // PATCH
        self.table = aclnn.rotary_table(self.ways, max(FRAMES, n), 2 * sum(SECTIONS))
        grid = torch.meshgrid(torch.arange(FRAMES), torch.arange(n), torch.arange(n), indexing="ij")
        self.positions = torch.stack([g.flatten() for g in grid])[:, None].to(device)
        self.state = torch.tensor([1234, 0], device=device)  # seed, offset
        # the dropouts' offsets from it: made here, since what is copied from the host cannot be recorded
        self.offsets = torch.tensor([[0, i] for i in range(2 * BLOCKS)], device=device).view(BLOCKS, 2, 2)

    def forward(self, frames, p=0.0):
        """(videos, FRAMES, 3, SIZE, SIZE) -> scores of the ways."""
        b, n = len(frames), SIZE // PATCH
        cut = frames.view(b, FRAMES, 3, n, PATCH, n, PATCH).permute(0, 1, 3, 5, 2, 4, 6).reshape(b, FRAMES * n * n, -1)
        x = cut.bfloat16() @ self.patches.t()
        positions = self.positions.expand(-1, b, -1)
        # a mask for every dropout and call: the state is a device tensor, so a recorded pass draws new ones as well
        states = self.state + self.offsets if p > 0.0 else None
        for i, block in enumerate(self.blocks):
            x = block(x, self.table, positions, states[i] if p > 0.0 else (None, None), p)
        if p > 0.0:
            self.state[1] += 2 * BLOCKS
        return x.float().mean(1) @ self.ways.float().t()


def videos(pictures, way):
    """A window that moves over each picture, one of four ways."""
    dev, (b, _, h, w) = pictures.device, pictures.shape
    step = torch.tensor([[1.0, 0.0], [-1.0, 0.0], [0.0, 1.0], [0.0, -1.0]], device=dev)[way] * 0.12
    shift = (torch.arange(FRAMES, device=dev) - (FRAMES - 1) / 2)[None, :, None] * step[:, None]
    line = (torch.arange(SIZE, device=dev) + 0.5) / SIZE - 0.5
    grid = torch.stack(torch.meshgrid(line, line, indexing="xy"), -1)[None, None] + shift[:, :, None, None]
    frames = aclnn.grid_sampler2d(pictures.repeat_interleave(FRAMES, 0), grid.flatten(0, 1).contiguous())
    return frames.view(b, FRAMES, 3, SIZE, SIZE)


def main():
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--steps", type=int, default=400)
    a = p.parse_args()
    torch.manual_seed(0)
    dev = torch.device("cuda:0")
    model = Model(dev)
    optimizer = torch.optim.AdamW(model.parameters(), lr=3e-4)

    def batch():
        way = torch.randint(WAYS, (16,), device=dev)
        return videos(torch.rand(16, 3, 24, 24, device=dev), way), way
    for step in range(a.steps):
        frames, way = batch()
        loss = F.cross_entropy(model(frames, p=0.1), way)
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        if step in (0, a.steps - 1):
            print(f"step {step}: loss {loss.item():.3f}", flush=True)
    with torch.no_grad():
        frames, _ = batch()
        model(frames)  # once outside the recording, so that libraries are set up
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            scores = model(frames)
        right = same = 0
        for _ in range(4):
            fresh, way = batch()
            frames.copy_(fresh)
            graph.replay()
            right += (scores.argmax(-1) == way).sum().item()
            same += torch.equal(scores, model(fresh))
    print(f"recorded answers: {right} of 64 right, {same} of 4 batches as without the recording", flush=True)
    if same != 4:
        raise SystemExit("the recording and the model disagree")


if __name__ == "__main__":
    main()
