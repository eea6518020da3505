"""Offset tables that descend, overlap or point outside: whatever they hold, the recurrence's pieces and the grouped products' tiles and
shares stay inside the buffers.  The kernels' arithmetic, restated; the GPU runs of the same tables stand at the end."""
import random

import pytest

SB = 16


def clamp(v, lo, hi):
    return min(max(v, lo), hi)


def tables(r, n, total):
    kind = r.randrange(4)
    if kind == 0:
        return [r.randrange(-50, total + 50) for _ in range(n + 1)]
    if kind == 1:
        return sorted((r.randrange(0, total + 1) for _ in range(n + 1)), reverse=True)
    if kind == 2:
        return [r.choice([0, total, -(1 << 62), (1 << 62), total // 2]) for _ in range(n + 1)]
    return [r.choice([0, total]) for _ in range(n + 1)]


def ranges(off, u, total):
    lo = clamp(off[u], 0, total)
    return lo, clamp(off[u + 1], lo, total)


def entry_of(off, L, number, total):
    lo, hi = 0, len(off) - 1
    while hi - lo > 1:
        mid = (lo + hi) // 2
        if clamp(off[mid], 0, total) // L + mid <= number:
            lo = mid
        else:
            hi = mid
    return lo


@pytest.mark.parametrize("seed", range(150))
def test_pieces_and_row_tiles(seed):
    r = random.Random(seed)
    n, total, L = r.choice([1, 2, 3, 9, 70]), r.choice([1, 100, 1000, 5000]), r.choice([64, 128, 256])
    off = tables(r, n, total)
    pieces = total // L + n
    for s in range(pieces):
        u = entry_of(off, L, s, total)
        base, stop = ranges(off, u, total)
        j = s - (base // L + u)
        first = stop + 1 if j < 0 else base + j * L
        if first >= stop:
            continue
        end = min(first + L, stop)
        assert 0 <= first < end <= total
        assert base // SB + u + (end - 1 - base) // SB < total // SB + n          # states
    for u in range(n):                                                            # the carries of an utterance's pieces
        lo, hi = ranges(off, u, total)
        m = -(-(hi - lo) // L)
        assert 0 <= lo // L + u and lo // L + u + max(m, 1) - 1 < pieces


@pytest.mark.parametrize("seed", range(150))
def test_shares_of_slabs(seed):
    r = random.Random(seed)
    E, total, KS, tiles, G = r.choice([1, 2, 5, 70]), r.choice([1, 100, 3000]), r.choice([32, 64]), r.choice([1, 2, 6]), r.choice([2, 7, 512])
    off = tables(r, E, total)
    slabs = []
    for e in range(E):
        a, b = ranges(off, e, total)
        slabs.append(max(-(-(b - a) // KS), 1))
    whole = sum(slabs) * tiles
    share = -(-whole // G)
    for me in range(G):
        at, end = me * share, min(me * share + share, whole)
        if at >= end:
            continue
        e, before = 0, 0
        while before + slabs[e] <= at // tiles:
            before += slabs[e]
            e += 1
        while at < end:
            while at >= (before + slabs[e]) * tiles:
                before += slabs[e]
                e += 1
            n = slabs[e]
            inside = at - before * tiles
            s0 = inside % n
            s1 = min(n, s0 + end - at)
            assert e < E and 0 <= inside // n < tiles and s0 < s1
            if s0 == 0 and s1 < n:                                                # left to others: they exist
                assert end == me * share + share and me + -(-(n - s1) // share) < G
            at += s1 - s0


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(12))
def test_nothing_is_written_outside(ctx, seed):
    """Results of such tables mean nothing; what lies around the outputs stays."""
    import torch

    from speechrecognition_amd import host
    r = random.Random(seed)
    n, total, D, N = r.choice([1, 3, 9, 70]), r.choice([100, 1000, 5000]), 40, 72
    off = torch.tensor(tables(r, n, total), device="cuda")
    guard, held = 512, []

    def out(rows, cols):
        buf = torch.full((rows * cols + 2 * guard,), 7.0, device="cuda")
        held.append(buf)
        return buf[guard:guard + rows * cols].view(rows, cols)

    def room(size):
        return out(max(size // 4, 4), 1).view(-1).view(torch.uint8)

    x, g, dy = torch.randn(total, D, device="cuda"), torch.rand(total, D, device="cuda"), torch.randn(total, N, device="cuda")
    w = torch.randn(n, N, D, device="cuda")
    h, dg, dx, last, y, gx, dw, db = out(total, D), out(total, D), out(total, D), out(n, D), out(total, N), out(total, D), out(n * N, D), out(n, N)
    states = room(host.gated_scan_states_bytes(ctx, n, total, D))
    for longest in (0, 10):
        scratch = room(host.gated_scan_scratch_bytes(ctx, n, total, longest, D))
        torch.cuda.synchronize()
        host.gated_scan(ctx, host.SCAN_VALUE, g, x, off, longest, h, h_last=last, states=states, scratch=scratch)
        host.gated_scan_backward(ctx, host.SCAN_VALUE, g, x, off, longest, states, x, dg, dx, scratch=scratch)
    scratch = room(host.group_matmul_dw_scratch_bytes(ctx, n, total, D, N))
    torch.cuda.synchronize()
    host.group_matmul(ctx, x, w, off, y)
    host.group_matmul_dx(ctx, dy, w, off, gx)
    host.group_matmul_dw(ctx, dy, x, off, dw.view(n, N, D), dbias=db, scratch=scratch)
    ctx.sync()
    for buf in held:
        assert (buf[:guard] == 7).all() and (buf[-guard:] == 7).all()
