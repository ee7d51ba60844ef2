"""The operators on token sequences as programs use them: under graph capture, on memory past 32-bit offsets, with lengths
out of range, one after the other in a block, and through the example."""
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import token_oracle as O

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def normal(device, seed, *size, dtype=torch.bfloat16):
    g = torch.Generator(device=device).manual_seed(seed)
    return torch.randn(*size, generator=g, device=device).to(dtype)


def replays(device, make, call, outputs):
    """Records call(inputs, outputs, workspace) and replays it on other inputs, with eager work between the replays."""
    inputs, ws = make(0), torch.empty(64 << 20, dtype=torch.uint8, device=device)
    made = outputs()
    call(inputs, made, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(inputs, made, ws)
    for seed in (1, 2, 3):
        fresh = make(seed)
        for a, b in zip(inputs, fresh):
            a.copy_(b)
        for t in made:
            t.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        want = outputs()
        call(fresh, want, torch.empty_like(ws))
        torch.cuda.synchronize()
        for a, b in zip(made, want):
            assert torch.equal(a, b), seed


def test_norm_and_rotary_in_a_graph(device, aclnn):
    def new(*size, dtype=torch.bfloat16):
        return torch.empty(*size, dtype=dtype, device=device)
    replays(device, lambda s: [normal(device, s, 70, 512), normal(device, s + 9, 70, 512), normal(device, s + 5, 512)],
            lambda i, o, ws: (aclnn.residual_norm(i[0], i[2], i[1], out=o[0], sum_out=o[1], rstd_out=o[2]),
                              aclnn.residual_norm_int8(i[0], i[2], i[1], out=o[3], scale_out=o[4], sum_out=o[1]),
                              aclnn.residual_norm_backward(i[0], o[1], i[2], o[2], grad_sum=i[1], grad_x=o[5],
                                                           grad_weight=o[6], workspace=ws)),
            lambda: [new(70, 512), new(70, 512), new(70, dtype=torch.float32), new(70, 512, dtype=torch.int8),
                     new(70, dtype=torch.float32), new(70, 512), new(512)])
    table = aclnn.rotary_table(torch.empty(0, device=device), 64, 64)
    replays(device, lambda s: [normal(device, s, 2, 40, 6, 64), normal(device, s + 9, 2, 40, 2, 64)],
            lambda i, o, ws: aclnn.rotary(i[0], i[1], table, query_out=o[0], key_out=o[1]),
            lambda: [new(2, 40, 6, 64), new(2, 40, 2, 64)])


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_attention_in_a_graph(device, aclnn, dtype):
    def make(s):
        return [normal(device, s, 2, 300, 4, 64, dtype=dtype), normal(device, s + 5, 2, 300, 2, 64, dtype=dtype),
                normal(device, s + 6, 2, 300, 2, 64, dtype=dtype), normal(device, s + 7, 2, 300, 4, 64, dtype=dtype),
                torch.tensor([300 - s, 200 + s], dtype=torch.int32, device=device)]

    def call(i, o, ws):
        masks = dict(left=50, sinks=3, q_lengths=i[4], kv_lengths=i[4])
        aclnn.window_attention(i[0], i[1], i[2], out=o[0], lse=o[1], workspace=ws, **masks)
        aclnn.window_attention_backward(i[3], i[0], i[1], i[2], o[0], o[1], grad_query=o[2], grad_key=o[3], grad_value=o[4],
                                        workspace=ws, **masks)
    new = lambda *size, t=dtype: torch.empty(*size, dtype=t, device=device)  # noqa: E731
    replays(device, make, call, lambda: [new(2, 300, 4, 64), new(2, 4, 300, t=torch.float32), new(2, 300, 4, 64), new(2, 300, 2, 64),
                                         new(2, 300, 2, 64)])


def test_single_tokens_in_a_graph(device, aclnn):
    """A cache whose lengths grow between the replays; the keys are split, so partial results go through the workspace."""
    k, v = normal(device, 1, 3, 5000, 1, 128), normal(device, 2, 3, 5000, 1, 128)
    replays(device, lambda s: [normal(device, s, 3, 1, 8, 128),
                               torch.tensor([17 + s, 5000 - s, 2500 * (s % 2)], dtype=torch.int64, device=device)],
            lambda i, o, ws: aclnn.window_attention(i[0], k, v, kv_lengths=i[1], out=o[0], lse=o[1], workspace=ws),
            lambda: [torch.empty(3, 1, 8, 128, dtype=k.dtype, device=device), torch.empty(3, 8, 1, device=device)])


def test_lengths_out_of_range_are_clamped(device, aclnn):
    q, k = normal(device, 1, 5, 20, 2, 64), normal(device, 2, 5, 50, 2, 64)
    wild = torch.tensor([-5, 2 ** 40, 50, 0, 2 ** 31], device=device)
    tame = torch.tensor([0, 50, 50, 0, 50], dtype=torch.int32, device=device)
    some = torch.tensor([2 ** 33, -1, 7, 20, 2 ** 62], device=device)
    few = torch.tensor([20, 0, 7, 20, 20], dtype=torch.int32, device=device)
    a = aclnn.window_attention(q, k, k, left=9, kv_lengths=wild, q_lengths=some, need_lse=True)
    b = aclnn.window_attention(q, k, k, left=9, kv_lengths=tame, q_lengths=few, need_lse=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert (a[0][0] == 0).all() and (a[0][1] == 0).all() and (a[0][3] == 0).all() and a[1][0].eq(-math.inf).all()
    for x, y in zip(aclnn.window_attention_backward(q, q, k, k, *a, left=9, kv_lengths=wild, q_lengths=some),
                    aclnn.window_attention_backward(q, q, k, k, *b, left=9, kv_lengths=tame, q_lengths=few)):
        assert torch.equal(x, y) and x.isfinite().all()
    strided = torch.stack([wild, some], 1)[:, 0]  # lengths apart are read in place
    assert torch.equal(aclnn.window_attention(q, k, k, left=9, kv_lengths=strided, q_lengths=few)[0], b[0])


def test_cache_past_32_bit_offsets(device, aclnn):
    """One sequence's cache of 5 GB: 40 million tokens, a window at its end and the sinks at its start."""
    n, d = 40_000_000, 64
    k, v = (torch.zeros(1, n, 1, d, dtype=torch.float16, device=device) for _ in range(2))
    q = normal(device, 1, 1, 3, 2, d, dtype=torch.float16)
    near = n - 700
    k[:, near:], v[:, near:] = normal(device, 2, 1, 700, 1, d, dtype=torch.float16), normal(device, 3, 1, 700, 1, d, dtype=torch.float16)
    k[:, :4], v[:, :4] = normal(device, 4, 1, 4, 1, d, dtype=torch.float16), normal(device, 5, 1, 4, 1, d, dtype=torch.float16)
    lens = torch.tensor([n - 10], device=device)
    out, lse = aclnn.window_attention(q, k, v, left=500, sinks=4, kv_lengths=lens, need_lse=True)
    # the same keys in a short cache: sinks, a gap that nobody sees, and the end
    short_k, short_v = (torch.cat([t[:, :4], t[:, near:]], 1) for t in (k, v))
    want, want_lse = aclnn.window_attention(q, short_k, short_v, left=500, sinks=4, need_lse=True,
                                            kv_lengths=torch.tensor([704 - 10], device=device))
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    go = normal(device, 6, 1, 3, 2, d, dtype=torch.float16)
    gq, gk, gv = aclnn.window_attention_backward(go, q, k, v, out, lse, left=500, sinks=4, kv_lengths=lens)
    wq, wk, wv = aclnn.window_attention_backward(go, q, short_k, short_v, want, want_lse, left=500, sinks=4,
                                                 kv_lengths=torch.tensor([704 - 10], device=device))
    assert torch.equal(gq, wq)
    bound = 2.0 ** -10  # other tiles, other order of the sums: a rounding of the result or two
    for g, w in ((gk, wk), (gv, wv)):
        got = torch.cat([g[:, :4], g[:, near:]], 1)
        assert ((got.float() - w.float()).abs() <= bound * w.float().abs() + 1e-6).all()
        assert not g[:, 4:near].any()


def test_views_far_into_memory(device, aclnn):
    """Rows and heads that begin more than 2^32 bytes into their storage."""
    big = torch.zeros(2_300_000_000, dtype=torch.bfloat16, device=device)
    x = big[-64 * 4096:].view(64, 4096)
    x.copy_(normal(device, 1, 64, 4096))
    w = normal(device, 2, 4096)
    assert torch.equal(aclnn.residual_norm(x, w)[0], aclnn.residual_norm(x.clone(), w)[0])
    rows = torch.as_strided(big, (2, 4096), (2_299_000_000, 1), 0)  # two rows 4.6 GB apart
    rows[1].copy_(x[0])
    assert torch.equal(aclnn.residual_norm(rows, w)[0][1], aclnn.residual_norm(x[:1].clone(), w)[0][0])
    table = aclnn.rotary_table(w, 64, 64)
    heads = torch.as_strided(big, (1, 2, 1, 64), (0, 2_299_000_000, 64, 1), 0)
    want = aclnn.rotary(heads.contiguous(), None, table)[0]
    assert torch.equal(aclnn.rotary(heads, None, table)[0], want)


def test_results_do_not_depend_on_the_batch(device, aclnn):
    """A sequence alone and among others has the same results, bit for bit, where the keys are not split."""
    q, k, v = (normal(device, s, 6, 180, h, 128) for s, h in ((1, 8), (2, 2), (3, 2)))
    whole = aclnn.window_attention(q, k, v, left=64, sinks=2, need_lse=True)
    for i in (0, 5):
        one = aclnn.window_attention(q[i:i + 1], k[i:i + 1], v[i:i + 1], left=64, sinks=2, need_lse=True)
        assert torch.equal(one[0], whole[0][i:i + 1]) and torch.equal(one[1], whole[1][i:i + 1])


def test_example_block(device):
    p = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "token_block.py"), "--steps", "3"], stdout=subprocess.PIPE,
                       stderr=subprocess.STDOUT, text=True, timeout=110, cwd=ROOT)
    assert p.returncode == 0, p.stdout
    assert "decoded" in p.stdout and "loss" in p.stdout


@pytest.mark.parametrize("dtype,sq,heads,d", [(torch.bfloat16, 300, 8, 128), (torch.float16, 7, 2, 64), (torch.float32, 150, 2, 72),
                                              (torch.float16, 160, 4, 256), (torch.bfloat16, 1500, 64, 32)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_gradients_of_queries_beside_keys_that_are_not_finite(device, aclnn, dtype, sq, heads, d, bad):
    """A key that is not finite reaches the gradients of the queries that see it, and no other query's, by a single bit."""
    skv, left, sinks = sq + 90, 40, 3
    q, go = normal(device, 1, 1, sq, heads, d, dtype=dtype), normal(device, 2, 1, sq, heads, d, dtype=dtype)
    k, v = normal(device, 3, 1, skv, 2, d, dtype=dtype), normal(device, 4, 1, skv, 2, d, dtype=dtype)
    masks = dict(left=left, sinks=sinks)

    def grads(k, v):
        out, lse = aclnn.window_attention(q, k, v, need_lse=True, **masks)
        return aclnn.window_attention_backward(go, q, k, v, out, lse, **masks)
    clean = grads(k, v)
    position = torch.arange(sq, device=device) + skv - sq
    for key in (20, skv - sq // 2 - 1):  # seen by nobody, and by some
        for which in (0, 1):
            pair = [k.clone(), v.clone()]
            pair[which][0, key, 0, d // 3] = bad
            got = grads(*pair)
            sees = (position >= key) & (position - left <= key)
            half = heads // 2  # heads of the first key head
            assert torch.equal(got[0][:, ~sees], clean[0][:, ~sees]) and torch.equal(got[0][:, :, half:], clean[0][:, :, half:])
            reached = got[0][:, sees][:, :, :half]  # a score of minus infinity leaves 0 times infinity, at the key's own feature
            assert not (reached if which else reached[..., d // 3]).isfinite().any()
            if not sees.any():
                assert torch.equal(got[1], clean[1]) and torch.equal(got[2], clean[2])
