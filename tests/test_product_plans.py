"""Plans of the gated projections' products: what fits a launch, parts that cover their terms, and the time to plan."""
import heapq
import random

import pytest

import host_plans as P

THREADS = {0: 256, 1: 512, 3: 256, 4: 512}
VEC = {"fp32": 4, "fp16": 8, "bf16": 8}
STAGE = {"fp32": 32, "fp16": 64, "bf16": 64}


def up(a, b):
    return -(-a // b)


def products(dtype, kind, rows, width, inner):
    """(tokens, features, stages) of the products that a plan is about."""
    s, v = STAGE[dtype], VEC[dtype]
    if kind == 0:
        return [(rows, 2 * inner, up(width, s))]
    padded = up(inner, s) * s
    both = [(rows, up(width, v) * v, 2 * padded // s), (2 * padded, up(width, v) * v, up(rows, s))]
    return [p for i, p in enumerate(both) if kind >> i & 1]


def test_last_end():
    """Against workgroups that are given out one by one."""
    rng = random.Random(1)
    for _ in range(3000):
        counts, lengths = [rng.randint(0, 60) for _ in range(2)], [rng.randint(1, 30) for _ in range(2)]
        slots = rng.randint(1, 20)
        free = [0] * slots
        for count, length in zip(counts, lengths):
            for _ in range(count):
                heapq.heapreplace(free, free[0] + length)
        assert P.product_last_end(counts, lengths, slots) == max(free), (counts, lengths, slots)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("kind", [0, 1, 2, 3])
def test_plans_fit(dtype, kind):
    rng = random.Random(kind)
    for _ in range(1000):
        rows = int(2 ** rng.uniform(0, 30 if kind == 0 else 20))
        width, inner = (int(2 ** rng.uniform(0, 19)) for _ in range(2))
        p = P.gated_plan(dtype, kind, rows, width, inner)
        sizes = products(dtype, kind, rows, width, inner)
        least = sum(up(t, 256) * up(f, 256) for t, f, _ in sizes) * 512
        assert (p is None) == (least >= 2 ** 32), (rows, width, inner)
        if p is None:
            continue
        if p[0] == 2:
            assert kind == 0 and rows <= 64
            continue
        side, groups = 256 if p[0] == 1 else 128, 0
        assert p[0] != 4 or (kind == 0 and dtype != "fp32" and p[1] == 1)
        assert p[0] != 3 or (kind != 2 and dtype == "fp32")
        for i, (tokens, features, stages) in enumerate(sizes):
            parts, length = p[1 + i], p[3 + i]
            assert (parts - 1) * length < stages <= parts * length  # none is empty
            assert parts == 1 or (parts <= 16 and length >= 4)
            high, wide = (32, 256) if p[0] == 3 and i == 0 else (side, side)
            groups += parts * up(tokens, high) * up(features, wide)
        assert groups * THREADS[p[0]] < 2 ** 32 and (p[0] != 4 or groups <= 256)


def test_largest_results():
    """A result of a terabyte fits a launch: what does not is refused before the card's memory ends."""
    assert P.gated_plan("bf16", 0, 2 ** 30, 1, 65) is not None
    assert P.gated_plan("bf16", 0, 2 ** 20, 1, 2 ** 17) is not None
    assert P.gated_plan("fp32", 0, 2 ** 30, 1, 2 ** 19) is None


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_host_time(dtype):
    """Some 20 us is the most that random sizes take."""
    for kind, size in ((0, (8, 4096, 14336)), (3, (777, 1001, 2731)), (3, (3000, 3000, 3000)), (3, (64, 8192, 8192))):
        assert P.gated_plan_nanoseconds(dtype, kind, *size) < 500_000
