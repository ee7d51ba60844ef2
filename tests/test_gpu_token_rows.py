"""Window attention where its kernels have many rows a workgroup (prompts, pictures and their gradients in 16-bit types: 128
rows, from as many tiles on as the card has CUs), against a plain implementation in 64 bits."""
import ctypes
import math

import pytest
import torch

import token_oracle as O

pytestmark = pytest.mark.gpu

NONE = 2 ** 63 - 1
ACL = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 27}

#   b   sq   skv  heads kv left right sinks lengths of the queries and keys
KINDS = {
    # a window, sinks apart from it, sequences of many lengths, more keys than queries
    "window": (8, 193, 400, 16, 8, 150, 0, 5, ([193, 193, 60, 1, 0, 193, 192, 33], [400, 399, 131, 1, 77, 193, 250, 64])),
    # both ways, the first token seen by all
    "picture": (6, 513, 513, 9, 9, 70, 60, 1, None),
    # all that went before, three heads to a key head, some queries without keys
    "prompt": (5, 330, 300, 21, 7, NONE, 0, 0, ([330, 200, 330, 7, 330], [300, 300, 10, 300, 0])),
}


def variant(aclnn, q, k, masks):
    """Name of the kernels that the forward call of these operands runs."""
    L, made = aclnn.load_library(), []

    def t(x):
        made.append(aclnn.create_tensor(tuple(x.shape), ACL[x.dtype]))
        return made[-1]
    ws, ex = ctypes.c_uint64(0), ctypes.c_void_p(None)
    st = L.opscvWindowAttentionGetWorkspaceSize(t(q), t(k), t(k), None, None, masks["scale"], masks["left"], masks["right"],
                                                masks["sinks"], t(q), None, ctypes.byref(ws), ctypes.byref(ex))
    assert st == 0
    name = aclnn.executor_variant(ex.value)
    aclnn.destroy_executor(ex.value)
    for h in made:
        aclnn.destroy_tensor(h)
    return name


def odd_start(t):
    """The same numbers in rows that begin on odd elements: read one by one instead of in vectors."""
    return torch.nn.functional.pad(t, (1, 2))[..., 1:-2]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("kind,d", [("window", 24), ("window", 64), ("window", 96), ("window", 128), ("window", 200),
                                    ("picture", 32), ("picture", 64), ("picture", 80), ("picture", 128),
                                    ("prompt", 33), ("prompt", 72), ("prompt", 128), ("prompt", 256)])
def test_attention_of_many_rows(device, aclnn, dtype, kind, d):
    b, sq, skv, heads, kv_heads, left, right, sinks, lengths = KINDS[kind]
    g = torch.Generator().manual_seed(sum(map(ord, kind + dtype)) + d)
    made = lambda *size, scale=1.0: (torch.randn(*size, generator=g) * scale).to(O.DTYPES[dtype])  # noqa: E731
    q, go = made(b, sq, heads, d), made(b, sq, heads, d, scale=0.01)
    k, v = made(b, skv, kv_heads, d), made(b, skv, kv_heads, d)
    masks = dict(scale=1.3 / math.sqrt(d), left=left, right=right, sinks=sinks)
    lens = dict(zip(("q_lens", "kv_lens"), lengths)) if lengths else {}
    on = {n: torch.tensor(lens[o], dtype=torch.int32, device=device)
          for n, o in (("q_lengths", "q_lens"), ("kv_lengths", "kv_lens")) if lens}
    assert variant(aclnn, q, k, masks).startswith("attention_rows")
    r = O.attention(q, k, v, grad_out=go, **masks, **lens)
    bound = O.attention_bounds(r, q, k, v, masks["scale"], dtype, go)
    dev = [t.to(device) for t in (q, k, v)]
    out, lse = aclnn.window_attention(*dev, need_lse=True, **masks, **on)
    O.within(out, r["out"], bound["out"], "out")
    O.within(lse, r["lse"], O.F32 * (1 + r["lse"].abs()), "lse")
    back = [go.to(device), *dev, r["out"].to(q.dtype).to(device), r["lse"].float().to(device)]
    grads = aclnn.window_attention_backward(*back, **masks, **on)
    for name, x in zip(("gq", "gk", "gv"), grads):
        O.within(x, r[name], bound[name], name)
    # element by element: the same products in the same order
    odd = [odd_start(t) for t in dev]
    a, b = aclnn.window_attention(*odd, need_lse=True, out=odd_start(torch.empty_like(out)), **masks, **on)
    assert torch.equal(a, out) and torch.equal(b, lse)
    again = aclnn.window_attention_backward(odd_start(back[0]), *odd, *back[4:], **masks, **on)
    assert all(torch.equal(x, y) for x, y in zip(again, grads))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 160])
def test_values_that_are_not_finite_among_many_rows(device, aclnn, dtype, d):
    """A key or value that is not finite reaches exactly the queries that see it, wherever it lies in their tiles."""
    b, sq, skv, heads, kv_heads, left, right, sinks, _ = KINDS["window"]
    g = torch.Generator().manual_seed(d)
    made = lambda *size: torch.randn(*size, generator=g).to(O.DTYPES[dtype]).to(device)  # noqa: E731
    q, k, v = made(b, sq, heads, d), made(b, skv, kv_heads, d), made(b, skv, kv_heads, d)
    masks = dict(left=left, right=right, sinks=sinks)
    assert variant(aclnn, q, k, dict(masks, scale=1.0)).startswith("attention_rows")
    clean, _ = aclnn.window_attention(q, k, v, **masks)
    position = torch.arange(sq, device=device) + skv - sq
    group = heads // kv_heads
    for key in (2, 30, 100, 207, 300, skv - 1):  # a sink, one that nobody sees, some, many, the last
        sees = (position >= key) & ((position - left <= key) | (key < sinks))
        for bad in (math.nan, math.inf, -math.inf):
            w = v.clone()
            w[3, key, 2, d // 3] = bad
            got, _ = aclnn.window_attention(q, k, w, **masks)
            hit = torch.zeros_like(clean, dtype=torch.bool)
            hit[3, sees, 2 * group:3 * group, d // 3] = True
            assert torch.equal(got[~hit], clean[~hit])
            assert got[hit].isnan().all() if bad != bad else (got[hit] == bad).all()
        x = k.clone()
        x[3, key, 2] = math.nan
        got, _ = aclnn.window_attention(q, x, v, **masks)
        hit = torch.zeros_like(clean, dtype=torch.bool)
        hit[3, sees, 2 * group:3 * group] = True
        assert torch.equal(got[~hit], clean[~hit]) and got[hit].isnan().all()
