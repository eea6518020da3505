"""The closed-form numbering that the recurrence's pieces and the grouped products' row tiles share: piece j of entry u, whose
range is [off[u], off[u+1]), has the number off[u] / L + u + j.  Numbers are unique, ascend with (u, j), stay below
total / L + n, and the entry of a number is the last u with off[u] / L + u <= number -- the search that the kernels make."""
import random

import pytest


def entry_of(off, L, number):
    lo, hi = 0, len(off) - 1
    while hi - lo > 1:
        mid = (lo + hi) // 2
        if off[mid] // L + mid <= number:
            lo = mid
        else:
            hi = mid
    return lo


def entry_of_64(off, L, number):
    """The same, 64 candidates at a time, as a wave searches."""
    lo, n = 0, len(off) - 1
    while n > 1:
        step = (n + 63) // 64
        c = sum(1 for lane in range(64) if lane * step < n and off[lo + lane * step] // L + lo + lane * step <= number)
        if c == 0:
            break
        first = (c - 1) * step
        n = min(n - first, step)
        lo += first
    return lo


@pytest.mark.parametrize("seed", range(60))
def test_numbers(seed):
    r = random.Random(seed)
    L = r.choice([32, 64, 128, 256])
    n = r.choice([1, 2, 5, 63, 64, 65, 200, 5000])
    off = [r.choice([0, 0, 7, 300])]
    for _ in range(n):
        off.append(off[-1] + r.choice([0, 0, 1, L - 1, L, L + 1, r.randrange(0, 5 * L)]))
    total = off[-1] + r.choice([0, 0, 500])
    last = -1
    for u in range(n):
        pieces = -(-(off[u + 1] - off[u]) // L)
        first = off[u] // L + u
        assert first > last                      # (an entry without a range has a number of its own too)
        for j in range(max(pieces, 1)):
            last = first + j
            assert last < total // L + n
            if n < 300 or r.random() < 0.02:
                assert entry_of(off, L, last) == u and entry_of_64(off, L, last) == u
