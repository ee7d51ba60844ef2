"""The operators on token sequences at the sizes that a launch holds: what does not fit is refused by the first phases, which
need no GPU, and not by the launch."""
import pytest

from test_tokens_boundary import BF16, F32, INVALID, phase1  # noqa: F401

NONE = 2 ** 62


def attention(phase1, b, sq, skv, heads, kv_heads, d, dtype, grad):  # noqa: F811
    q, kv, lse = ((b, sq, heads, d), dtype), ((b, skv, kv_heads, d), dtype), ((b, heads, sq), F32)
    if grad:
        return phase1("opscvWindowAttentionBackward", q, q, kv, kv, q, lse, None, None, 0.1, NONE, 0, 0, q, kv, kv)
    return phase1("opscvWindowAttention", q, kv, kv, None, None, 0.1, NONE, 0, 0, q, lse)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_of_many_sequences(phase1, dtype, grad):  # noqa: F811
    for b, sq, skv, heads, d in ((300_000, 1, 9, 8, 32), ((1 << 21) + 3, 1, 2, 8, 8), ((1 << 27), 1, 1, 8, 1), (1 << 20, 130, 5, 2, 8)):
        st, ws, name = attention(phase1, b, sq, skv, heads, heads, d, dtype, grad)
        assert st == 0 and name == ("attention_grad" if grad else name) and (ws > 0) == grad
        if grad:  # scratch for the sequences of one launch, of which there are several
            assert ws <= b * heads * ((sq + 7) // 8 * 8) * 8 + 65536


@pytest.mark.parametrize("grad", [False, True])
def test_attention_of_rows_that_no_launch_holds(phase1, grad):  # noqa: F811
    # 32 rows a workgroup of 256 threads: 2^29 rows and no more
    assert attention(phase1, 2, 1 << 28, 9, 1, 1, 8, F32, grad)[0] == 0
    assert attention(phase1, 1, 1 << 28, 9, 2, 1, 8, F32, grad)[0] == INVALID
    assert attention(phase1, 1, 1 << 28, 9, 4, 1, 8, BF16, grad)[0] == 0  # 128 rows a workgroup
    # keys of a sequence: workgroups of the gradients only
    assert attention(phase1, 1, 4, 1 << 28, 64, 64, 8, BF16, grad)[0] == (INVALID if grad else 0)
    # more tokens, or rows, than the kernels' numbers hold
    assert attention(phase1, 1, (1 << 28) + 1, 9, 1, 1, 8, BF16, grad)[0] == INVALID
    assert attention(phase1, 1, 1 << 28, 9, 8, 1, 8, BF16, grad)[0] == INVALID
