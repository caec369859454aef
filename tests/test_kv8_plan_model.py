"""The shares of sdv_kv8_plan.h, modelled: every unit of every tile lies in one range, the closed
form counts what it should, parts lie in slots of their own, and no 32-bit sum overflows."""
from __future__ import annotations

import random

import pytest

STEP = 64
M32 = (1 << 32) - 1


def floor_sum(n, m, a, b):
    ans = 0
    while n > 0:
        if a >= m:
            ans += n * (n - 1) // 2 * (a // m)
            a %= m
        if b >= m:
            ans += n * (b // m)
            b %= m
        y = a * n + b
        assert y <= M32
        if y < m:
            break
        n, b = y // m, y % m
        m, a = a, m
    assert ans <= M32
    return ans


def tiles(n, G, TR):
    return (n * G + TR - 1) // TR


def before(n, T, G, TR, i, tree, unit=1):
    if tree:
        return i * -(-max(T, 1) // (STEP * unit))
    m = STEP * unit * G
    return floor_sum(i, m, TR, max(T - n, 0) * G + TR + m - 1)


def units_of(n, T, G, TR, i, tree, unit=1):
    """Units of `unit` steps of tile i."""
    if tree:
        return -(-max(T, 1) // (STEP * unit))
    ctx = max(T - n, 0)
    if i == tiles(n, G, TR) - 1:
        return -(-(ctx + n) // (STEP * unit))
    m = STEP * unit * G
    return (ctx * G + TR * (i + 1) + m - 1) // m


def keys(n, T, G, TR, i):
    """Keys that the tile's last row sees, in a context of max(T - n, 0)."""
    last = min(n * G, TR * (i + 1)) - 1
    return max(T - n, 0) + last // G + 1


@pytest.mark.parametrize("unit", [1, 4])
@pytest.mark.parametrize("G", [1, 2, 3, 6, 7, 20])
@pytest.mark.parametrize("TR", [16, 32, 128, 256])
def test_units_cover_the_keys(G, TR, unit):
    rng = random.Random(G * TR)
    for _ in range(60):
        n = rng.choice([1, 2, 5, rng.randint(1, 70), rng.randint(1, 3000)])
        T = rng.choice([0, n - 1, n, n + rng.randint(0, 40), n + rng.randint(0, 40000)])
        total = 0
        for i in range(tiles(n, G, TR)):
            s = units_of(n, T, G, TR, i, False, unit)
            assert total == before(n, T, G, TR, i, False, unit)
            need, step = keys(n, T, G, TR, i), STEP * unit
            assert s * step >= need and (s - 1) * step < need + (0 if i == tiles(n, G, TR) - 1 else 1)
            # the tile's steps, of which the last unit may hold fewer
            steps = units_of(n, T, G, TR, i, False)
            assert (s - 1) * unit < steps <= s * unit
            total += s


@pytest.mark.parametrize("seed", range(24))
def test_ranges(seed):
    rng = random.Random(seed)
    G, TR, KV = rng.choice([1, 3, 6, 7]), rng.choice([16, 32, 256]), rng.choice([1, 2, 4])
    tree = seed % 4 == 3
    seqs = []
    for _ in range(rng.choice([1, 2, 9, 40])):
        n = rng.choice([0, 1, 1, 5, rng.randint(1, 64 if tree else 600)])
        seqs.append((n, n + rng.randint(0, 5000)))
    grid, unit = rng.choice([1, 8, 256, 512]), rng.choice([1, 4])
    head = 0 if unit > 1 else rng.choice([0, 5])  # units that stand for a tile's start
    order = [(h, b, i, head + units_of(n, T, G, TR, i, tree, unit)) for h in range(KV) for b, (n, T) in enumerate(seqs)
             for i in range(tiles(n, G, TR))]
    units = sum(x[3] for x in order)
    if units == 0:
        return
    ranges = min(grid, units)
    share, rest = units // ranges, units % ranges
    start = lambda w: w * share + min(w, rest)  # noqa: E731
    split = rest * (share + 1)
    owner = lambda x: x // (share + 1) if x < split else rest + (x - split) // share  # noqa: E731
    assert start(0) == 0 and start(ranges) == units
    for w in range(ranges):
        assert start(w) < start(w + 1)
        assert owner(start(w)) == w and owner(start(w + 1) - 1) == w
    # walk the ranges as the kernels do
    tile0, at = [], 0
    for x in order:
        tile0.append(at)
        at += x[3]
    parts, whole, used = {}, set(), set()
    t = 0
    for w in range(ranges):
        u, end, first = start(w), start(w + 1), True
        while tile0[t] + order[t][3] <= u:
            t += 1
        k = t
        while u < end:
            lo, hi = max(u - tile0[k] - head, 0), min(order[k][3], end - tile0[k]) - head
            if lo >= hi:
                break  # the range ends in the tile's start
            if lo == 0 and hi == order[k][3] - head:
                whole.add(k)
            else:
                slot = 2 * w + (0 if first else 1)
                assert slot not in used and slot < 2 * grid
                used.add(slot)
                parts.setdefault(k, []).append((w, slot, lo, hi))
            first = False
            u = min(tile0[k] + order[k][3], end)
            k += 1
    # every tile is whole in one range, or its parts cover it in order and lie where the merge looks
    assert whole.isdisjoint(parts) and len(whole) + len(parts) == len(order)
    for k, own in parts.items():
        w0 = owner(tile0[k] + head)
        count = owner(tile0[k] + order[k][3] - 1) - w0 + 1
        second = 1 if start(w0) < tile0[k] else 0
        assert [p[0] for p in own] == list(range(w0, w0 + count))
        assert [p[1] for p in own] == [2 * w0 + second] + [2 * (w0 + j) for j in range(1, count)]
        assert [p[2] for p in own] == [0] + [p[3] for p in own][:-1] and own[-1][3] == order[k][3] - head
