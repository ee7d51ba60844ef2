"""A small picture-and-text model: the sampler feeds the token operators, in training and in answering.

Pictures are resampled to one size through `grid_sampler2d` (a rotated crop each), cut into patches and put before the text's
tokens. Each block is residual RMS norm -> rotary positions -> attention with a sliding window and sinks -> residual RMS norm
-> gated product. Training differentiates through the operators' backward forms; answering writes rotated keys straight
into a cache and takes one token at a time, the cache's lengths being device tensors, so that a step is one recorded graph.
The projections are torch's matrix products. Weights and data are random.

    python examples/token_block.py [--steps 20] [--tokens 16]
"""
import argparse
import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from ops_cv_amd import aclnn  # noqa: E402

VOCAB, WIDTH, HEADS, KV_HEADS, D, BLOCKS = 256, 512, 8, 2, 64, 2
SIZE, PATCH, TEXT, WINDOW, SINKS = 160, 16, 60, 128, 4


class Norm(torch.autograd.Function):
    """(norm of x + residual, x + residual)."""

    @staticmethod
    def forward(ctx, x, residual, weight):
        y, total, rstd = aclnn.residual_norm(x, weight, residual, need_rstd=True)
        ctx.save_for_backward(total, weight, rstd)
        return y, total

    @staticmethod
    def backward(ctx, grad_y, grad_total):
        total, weight, rstd = ctx.saved_tensors
        grad, grad_weight = aclnn.residual_norm_backward(grad_y, total, weight, rstd, grad_sum=grad_total)
        return grad, grad, grad_weight


class Rotary(torch.autograd.Function):
    """Query and key turned by their positions; the gradient is turned back."""

    @staticmethod
    def forward(ctx, query, key, table):
        ctx.save_for_backward(table)
        return aclnn.rotary(query, key, table)

    @staticmethod
    def backward(ctx, grad_query, grad_key):
        return (*aclnn.rotary(grad_query, grad_key, ctx.saved_tensors[0], inverse=True), None)


class Attend(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, value):
        out, lse = aclnn.window_attention(query, key, value, left=WINDOW, sinks=SINKS, need_lse=True)
        ctx.save_for_backward(query, key, value, out, lse)
        return out

    @staticmethod
    def backward(ctx, grad):
        return aclnn.window_attention_backward(grad, *ctx.saved_tensors, left=WINDOW, sinks=SINKS)


class Model(torch.nn.Module):
    def __init__(self, device):
        super().__init__()
        def weight(*size):  # noqa: E306
            return torch.nn.Parameter((torch.randn(*size, device=device) * size[0] ** -0.5).bfloat16())
        self.patches, self.words = weight(3 * PATCH * PATCH, WIDTH), weight(VOCAB, WIDTH)
        self.norms = torch.nn.ParameterList([torch.nn.Parameter(torch.ones(WIDTH, device=device).bfloat16())
                                             for _ in range(2 * BLOCKS + 1)])
        self.into = torch.nn.ParameterList([weight(WIDTH, (HEADS + 2 * KV_HEADS) * D) for _ in range(BLOCKS)])
        self.back = torch.nn.ParameterList([weight(HEADS * D, WIDTH) for _ in range(BLOCKS)])
        self.up = torch.nn.ParameterList([weight(WIDTH, 4 * WIDTH) for _ in range(BLOCKS)])
        self.down = torch.nn.ParameterList([weight(2 * WIDTH, WIDTH) for _ in range(BLOCKS)])
        self.table = aclnn.rotary_table(self.words, 1024, D)

    def embed(self, pictures, angle):
        """Pictures of any size -> a rotated crop of SIZE x SIZE -> patches -> tokens."""
        c, s = angle.cos() * 0.7, angle.sin() * 0.7
        zero = torch.zeros_like(c)
        turn = torch.stack([c, -s, zero, s, c, zero], 1).view(-1, 2, 3)
        grid = F.affine_grid(turn, (len(angle), 3, SIZE, SIZE), align_corners=False)
        crops = aclnn.grid_sampler2d(pictures, grid)
        n = SIZE // PATCH
        cut = crops.view(-1, 3, n, PATCH, n, PATCH).permute(0, 2, 4, 1, 3, 5).reshape(len(angle), n * n, -1)
        return cut.bfloat16() @ self.patches

    def project(self, i, y):
        b, n, _ = y.shape
        q, k, v = (y @ self.into[i]).split([HEADS * D, KV_HEADS * D, KV_HEADS * D], -1)
        return q.view(b, n, HEADS, D), k.view(b, n, KV_HEADS, D), v.view(b, n, KV_HEADS, D)

    def gated(self, i, y):
        a, g = (y @ self.up[i]).chunk(2, -1)
        return (a * F.silu(g)) @ self.down[i]

    def forward(self, x):
        """Every token's features: the way of training."""
        add = torch.zeros_like(x)
        for i in range(BLOCKS):
            y, x = Norm.apply(add, x, self.norms[2 * i])
            q, k, v = self.project(i, y)
            q, k = Rotary.apply(q, k, self.table)
            y, x = Norm.apply(Attend.apply(q, k, v).flatten(2) @ self.back[i], x, self.norms[2 * i + 1])
            add = self.gated(i, y)
        return Norm.apply(add, x, self.norms[-1])[0]

    @torch.no_grad()
    def extend(self, x, cache, positions, lengths, slots):
        """Features of the new tokens, whose keys and values go into the cache at `slots` (a slice, or an index tensor for
        single tokens); `lengths` counts them in."""
        add = torch.zeros_like(x)
        for i, (keys, values) in enumerate(cache):
            y, x, _ = aclnn.residual_norm(add, self.norms[2 * i], x)
            q, k, v = self.project(i, y)
            if isinstance(slots, slice):
                q, _ = aclnn.rotary(q, k, self.table, positions, key_out=keys[:, slots])
                values[:, slots] = v
            else:
                q, k = aclnn.rotary(q, k, self.table, positions)
                keys.index_copy_(1, slots, k)
                values.index_copy_(1, slots, v)
            out, _ = aclnn.window_attention(q, keys, values, left=WINDOW, sinks=SINKS, kv_lengths=lengths)
            y, x, _ = aclnn.residual_norm(out.flatten(2) @ self.back[i], self.norms[2 * i + 1], x)
            add = self.gated(i, y)
        return aclnn.residual_norm(add, self.norms[-1], x)[0]


def answer(model, start, tokens):
    """Greedy tokens after `start` (b, n, WIDTH): the prompt in one call, then one recorded step replayed."""
    b, n, _ = start.shape
    dev = start.device
    cache = [tuple(torch.zeros(b, n + tokens, KV_HEADS, D, dtype=start.dtype, device=dev) for _ in range(2)) for _ in range(BLOCKS)]
    first = torch.arange(n, device=dev).expand(b, n)
    lengths = torch.full((b,), n, device=dev)
    y = model.extend(start, cache, first, lengths, slice(0, n))
    token = (y[:, -1] @ model.words.t()).argmax(-1)
    position, slot = torch.full((b, 1), n, device=dev), torch.full((1,), n, device=dev)

    def step():
        lengths.copy_(position[:, 0] + 1)
        y = model.extend(model.words[token][:, None], cache, position, lengths, slot)
        token.copy_((y[:, 0] @ model.words.t()).argmax(-1))
        position.add_(1)
        slot.add_(1)
        return y

    held = [t.clone() for t in (token, position, slot)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # once outside the recording, so that libraries are set up
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        features = step()
    for t, was in zip((token, position, slot), held):
        t.copy_(was)
    said, seen = [token.clone()], []
    for _ in range(tokens - 1):
        graph.replay()
        said.append(token.clone())
        seen.append(features.clone())
    return torch.stack(said, 1), torch.cat([y[:, -1:]] + seen, 1)


def main():
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--steps", type=int, default=20)
    p.add_argument("--tokens", type=int, default=16)
    a = p.parse_args()
    torch.manual_seed(0)
    dev = torch.device("cuda:0")
    model = Model(dev)
    pictures, text = torch.rand(4, 3, 200, 240, device=dev), torch.randint(VOCAB, (4, TEXT), device=dev)
    angle = torch.tensor([0.0, 0.3, -0.2, 1.0], device=dev)
    optimizer = torch.optim.AdamW(model.parameters(), lr=1e-3)
    for step in range(a.steps):
        x = torch.cat([model.embed(pictures, angle), model.words[text]], 1)
        y = model(x)[:, -TEXT - 1:-1]
        loss = F.cross_entropy((y @ model.words.t()).float().flatten(0, 1), text.flatten())
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        if step in (0, a.steps - 1):
            print(f"step {step}: loss {loss.item():.3f}", flush=True)
    with torch.no_grad():
        start = torch.cat([model.embed(pictures, angle), model.words[text[:, :8]]], 1)
        said, seen = answer(model, start, a.tokens)
        whole = model(torch.cat([start, model.words[said[:, :-1]]], 1))[:, start.shape[1] - 1:]
    off = ((seen.float() - whole.float()).norm() / whole.float().norm()).item()
    print(f"decoded {tuple(said.shape)} tokens, features within {off:.1e} of the whole sequence at once", flush=True)
    if not off < 2e-2:  # bfloat16 of 2^-8 through a few roundings of two blocks
        raise SystemExit("the cache and the whole sequence disagree")


if __name__ == "__main__":
    main()
