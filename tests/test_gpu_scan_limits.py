"""The recurrence's results do not depend on whether utterances are cut into pieces: infinities and vanishing products of gates.  No
counterpart in the reference."""
import numpy as np
import pytest

from speechrecognition_amd import host
from tests.test_gpu_scan import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("max_frames", [0, 1])             # cut into pieces, and whole
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("lens", [[5000], [3, 1200, 0, 900]])
def test_infinities_pass_pieces_as_they_pass_frames(ctx, dtype, sigmoid, lens, max_frames):
    """Gates whose product over a few hundred frames underflows: an infinite value, initial state or gradient stays infinite, with its
    sign, up to a gate of exactly zero or an infinity of the other sign, which make it NaN."""
    import torch
    big = int(np.argmax(lens))
    c = Case(ctx, lens, 8, dtype, sigmoid, max_frames=max_frames)
    assert (host.gated_scan_scratch_bytes(ctx, c.n, c.T, max_frames, c.D) > 0) == (max_frames == 0)
    lo, hi = int(c.off[big]), int(c.off[big + 1])
    c.g.fill_(-1.0 if sigmoid else 0.25)
    if not sigmoid:
        c.g[:, 1] = -0.25
        c.g[lo + 600, 5] = 0.0
    c.x[lo + 100, 0] = float("-inf")
    c.x[lo + 101, 1] = float("inf")
    c.h0[big, 2] = float("inf")
    c.dl[big, 3] = float("-inf")
    c.dh[hi - 200, 4] = float("inf")
    c.x[lo + 100, 5] = float("inf")
    c.x[lo + 100, 6] = float("inf")
    c.x[lo + 500, 6] = float("-inf")
    torch.cuda.synchronize()
    c.run()
    ctx.sync()

    # frame by frame, on the CPU, in 64 bits
    g, x, dh, h, dx, h0, hl, dl, d0 = (v.double().cpu().numpy() for v in (c.g, c.x, c.dh, c.h, c.dx, c.h0, c.hl, c.dl, c.d0))
    a = 1 / (1 + np.exp(-g)) if sigmoid else g
    b = (1 - a) * x if sigmoid else x
    with np.errstate(invalid="ignore"):
        for u in range(c.n):
            s = h0[u]
            for t in range(c.off[u], c.off[u + 1]):
                s = a[t] * s + b[t]
                same(h[t], s, ("h", u, t))
            same(hl[u], s, ("h_last", u))
            s = dl[u]
            for t in range(c.off[u + 1] - 1, c.off[u] - 1, -1):
                s = s + dh[t]
                same(dx[t], s * (1 - a[t]) if sigmoid else s, ("dx", u, t))
                s = s * a[t]
            same(d0[u], s, ("dh0", u))


def same(got, want, where):
    """Infinities and NaN alike; finite values are compared elsewhere."""
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isposinf(got), np.isposinf(want)) and np.array_equal(np.isneginf(got), np.isneginf(want)), (where, got, want)


@pytest.mark.parametrize("sigmoid", [False, True])
def test_products_that_vanish_leave_finite_states_alone(ctx, sigmoid):
    """States of 1e30 in front of pieces whose gates multiply to less than the smallest number, and values of zero behind: zero."""
    import torch
    c = Case(ctx, [3000], 4, "f32", sigmoid, max_frames=0)
    c.g.fill_(-2.0 if sigmoid else 0.125)
    c.g[:, 1] *= 1 if sigmoid else -1
    for v in (c.x, c.dh):
        v.zero_()
    c.h0.fill_(1e30)
    c.dl.fill_(-1e30)
    torch.cuda.synchronize()
    assert host.gated_scan_scratch_bytes(ctx, c.n, c.T, 0, c.D) > 0
    c.run()
    ctx.sync()
    for v in (c.h[500:], c.hl, c.dx[:2500], c.d0):
        assert not v.any()
    assert (c.h[:20] != 0).all() and (c.dx[-20:] != 0).all()
