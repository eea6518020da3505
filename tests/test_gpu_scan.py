"""srx_gated_scan_dev and its backward pass against the recurrence written out in 64 bits (tests/learned_ref.py), every
element within a bound summed from the kernel's roundings.  No counterpart in the reference."""
import numpy as np
import pytest

from speechrecognition_amd import _capi, host
from tests import learned_ref as R

pytestmark = pytest.mark.gpu
EVERY = _capi.SRX_SCAN_STATE_EVERY


def _t(dtype):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]


def _offsets(lens, front=0):
    return np.concatenate([[front], front + np.cumsum(lens)]).astype(np.int64)


def _strided(torch, a, dtype, pad, shift=0):
    """A [rows][cols] tensor whose rows lie cols + pad elements apart, `shift` elements into its allocation."""
    rows, cols = a.shape
    buf = torch.full((rows * (cols + pad) + shift + 8,), -7.0, dtype=_t(dtype), device="cuda")
    v = buf[shift:shift + rows * (cols + pad)].view(rows, cols + pad)[:, :cols] if rows else buf[:0].view(0, cols)
    v.copy_(torch.from_numpy(np.ascontiguousarray(a)))
    return v


class Case:
    def __init__(self, ctx, lens, D, dtype, sigmoid, front=0, behind=0, pad=0, shift=0, with_state=True, max_frames=None, seed=0):
        import torch
        self.torch, self.ctx, self.dtype, self.sigmoid = torch, ctx, dtype, sigmoid
        r = np.random.default_rng(seed)
        self.off = _offsets(lens, front)
        self.T, self.D, self.n = int(self.off[-1]) + behind, D, len(lens)
        self.max_frames = max(lens, default=0) if max_frames is None else max_frames
        g = r.normal(1.0, 2.0, (self.T, D))
        if not sigmoid:
            g = 1 / (1 + np.exp(-g)) * r.choice([1, 1, 1, -1], g.shape)
        self.g, self.x, self.dh = (_strided(torch, v, dtype, pad, shift) for v in (g, r.normal(size=(self.T, D)), r.normal(size=(self.T, D))))
        self.h, self.dg, self.dx = (_strided(torch, np.full((self.T, D), 5.0), dtype, pad, shift) for _ in range(3))
        f = lambda: torch.from_numpy(r.normal(size=(self.n, D)).astype(np.float32)).cuda()  # noqa: E731
        self.h0, self.dl = (f(), f()) if with_state else (None, None)
        self.hl, self.d0 = f(), f()
        self.offd = torch.from_numpy(self.off).cuda()
        self.mode = host.SCAN_SIGMOID if sigmoid else host.SCAN_VALUE
        self.states = torch.full((max(host.gated_scan_states_bytes(ctx, self.n, self.T, D), 4),), 255, dtype=torch.uint8, device="cuda")
        self.scratch = torch.full((max(host.gated_scan_scratch_bytes(ctx, self.n, self.T, self.max_frames, D), 4),), 255, dtype=torch.uint8,
                                  device="cuda")
        torch.cuda.synchronize()

    def run(self, ctx=None, back=True):
        ctx = ctx or self.ctx
        host.gated_scan(ctx, self.mode, self.g, self.x, self.offd, self.max_frames, self.h, h0=self.h0, h_last=self.hl,
                        states=self.states if back else None, scratch=self.scratch)
        if back:
            host.gated_scan_backward(ctx, self.mode, self.g, self.x, self.offd, self.max_frames, self.states, self.dh, self.dg, self.dx,
                                     dh_last=self.dl, dh0=self.d0, scratch=self.scratch)

    def check(self):
        self.ctx.sync()
        n = lambda t: None if t is None else t.double().cpu().numpy()  # noqa: E731
        f = R.scan(n(self.g), n(self.x), self.off, n(self.h0), self.sigmoid)
        b = R.scan_back(f, n(self.g), n(self.x), self.off, n(self.dh), n(self.dl), self.sigmoid)
        inside = np.zeros(self.T, bool)
        for u in range(self.n):
            inside[self.off[u]:self.off[u + 1]] = True
        for name, got, want, err in (("h", self.h, f["h"], f["eh"]), ("dx", self.dx, b["dx"], b["edx"]), ("dgate", self.dg, b["dg"], b["edg"])):
            got = n(got)
            tol = R.out_bound(want, err, self.dtype)
            bad = np.abs(got - want)[inside] > tol[inside]
            assert not bad.any(), (name, int(bad.sum()), float(np.max((np.abs(got - want) / (tol + 1e-300))[inside])))
            assert (got[~inside] == 5.0).all(), name                        # frames of no utterance are left as they were
        for name, got, want, err in (("h_last", self.hl, f["last"], f["elast"]), ("dh0", self.d0, b["d0"], b["e0"])):
            assert (np.abs(n(got) - want) <= R.out_bound(want, err, "f32")).all(), name


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens,D", [([1], 1), ([0], 3), ([1, 0, 2, 15, 16, 17], 39), ([33, 1, 64], 130), ([5, 7], 64), ([40] * 9, 6)])
def test_scan_and_gradients(ctx, dtype, sigmoid, lens, D):
    c = Case(ctx, lens, D, dtype, sigmoid)
    c.run()
    c.check()


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens,D,front,behind", [([700], 39, 0, 0), ([0, 300, 0, 64, 65, 1, 513, 0], 130, 5, 3), ([2000, 1], 2, 200, 70),
                                                 ([127, 128, 129], 64, 64, 64)])
def test_pieces_of_long_utterances(ctx, dtype, sigmoid, lens, D, front, behind):
    """max_frames 0 (unknown) makes the library cut the utterances; frames in front of the first and behind the last stay."""
    c = Case(ctx, lens, D, dtype, sigmoid, front=front, behind=behind, max_frames=0)
    assert host.gated_scan_scratch_bytes(ctx, c.n, c.T, 0, D) > 0 or sum(lens) < 200
    c.run()
    c.check()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("pad,shift", [(1, 0), (2, 1), (3, 3), (64, 2)])
def test_row_strides_and_odd_addresses(ctx, dtype, pad, shift):
    c = Case(ctx, [50, 3], 66, dtype, True, pad=pad, shift=shift)
    c.run()
    c.check()


def test_no_initial_state_and_nothing_wanted(ctx):
    c = Case(ctx, [20, 0, 3], 10, "f32", True, with_state=False)
    c.run()
    c.check()
    before = c.h.clone()
    c.h.zero_()
    c.torch.cuda.synchronize()
    host.gated_scan(ctx, c.mode, c.g, c.x, c.offd, c.max_frames, c.h)      # no h0, h_last, states, scratch
    ctx.sync()
    assert c.torch.equal(c.h[:23], before[:23])


def test_steps_of_one_frame_are_the_whole_scan(ctx):
    """h_last written over h0, one frame of every stream at a time: bit for bit the scan of the whole streams."""
    n, T, D = 7, 19, 48
    c = Case(ctx, [T] * n, D, "f32", True)
    c.run(back=False)
    state = c.h0.clone()
    ones = c.torch.arange(n + 1, dtype=c.torch.int64, device="cuda")
    for t in range(T):
        g, x = (v.view(n, T, D)[:, t].contiguous() for v in (c.g, c.x))
        h = c.torch.empty_like(x)
        c.torch.cuda.synchronize()
        host.gated_scan(ctx, c.mode, g, x, ones, 1, h, h0=state, h_last=state)
        ctx.sync()
        assert c.torch.equal(h, c.h.view(n, T, D)[:, t])
    assert c.torch.equal(state, c.hl)


@pytest.mark.parametrize("max_frames", [None, 0])
def test_state_written_over_the_one_read(ctx, max_frames):
    c = Case(ctx, [300, 0, 90], 20, "f32", False, max_frames=max_frames)
    c.run()
    ctx.sync()
    hl, d0 = c.hl.clone(), c.d0.clone()
    a, b = c.h0.clone(), c.dl.clone()
    c.torch.cuda.synchronize()
    host.gated_scan(ctx, c.mode, c.g, c.x, c.offd, c.max_frames, c.h, h0=a, h_last=a, states=c.states, scratch=c.scratch)
    host.gated_scan_backward(ctx, c.mode, c.g, c.x, c.offd, c.max_frames, c.states, c.dh, c.dg, c.dx, dh_last=b, dh0=b, scratch=c.scratch)
    ctx.sync()
    assert c.torch.equal(a, hl) and c.torch.equal(b, d0)


@pytest.mark.parametrize("max_frames", [None, 0])
def test_nan_and_infinity_stay_in_their_channel_and_utterance(ctx, max_frames):
    c = Case(ctx, [80, 80, 80], 34, "bf16", True, max_frames=max_frames)
    c.run()
    ctx.sync()
    clean = c.h.clone(), c.dx.clone(), c.dg.clone()
    c.x[100, 3] = float("nan")       # utterance 1
    c.x[100, 4] = float("inf")
    c.g[100, 5] = float("nan")
    c.torch.cuda.synchronize()
    c.run()
    ctx.sync()
    hit = c.torch.zeros_like(c.h, dtype=c.torch.bool)
    hit[80:160, 3:6] = True
    for now, was in zip((c.h, c.dx, c.dg), clean):
        assert c.torch.equal(now[~hit], was[~hit])
    assert c.torch.isnan(c.h[100:160, 3]).all() and c.torch.isinf(c.h[100, 4]) and c.torch.isnan(c.h[100:160, 5]).all()
    assert c.torch.isfinite(c.h[80:100, 3:6]).all()


def test_gates_above_one_and_zero_gates_across_pieces(ctx):
    """The product of a piece's gates overflows while the state is zero, or a zero gate ends it: no NaN appears."""
    c = Case(ctx, [400], 8, "f32", False, max_frames=0)
    c.g.fill_(8.0)
    c.x.zero_()
    c.h0.zero_()
    c.dh.zero_()
    c.dl.zero_()
    c.g[::50, 1] = 0.0
    c.torch.cuda.synchronize()
    c.run()
    ctx.sync()
    for v in (c.h, c.hl, c.dx, c.dg, c.d0):
        assert (v == 0).all()


def test_gradient_against_differences(ctx):
    """<h, dh> + <h_last, dh_last> moved by +-eps along a direction: x and h0 enter linearly (eps of any size), the gate through
    a sigmoid (the third derivative's eps^2 / 6 is below the bound at 2^-5; f32 rounding of the two sums is far below)."""
    c = Case(ctx, [37, 90], 24, "f32", True)
    torch = c.torch
    c.run()
    ctx.sync()
    grads = [v.clone().double() for v in (c.dg, c.dx, c.d0)]

    def value():
        torch.cuda.synchronize()
        c.run(back=False)
        ctx.sync()
        return float((c.h.double() * c.dh.double()).sum() + (c.hl.double() * c.dl.double()).sum())

    gen = torch.Generator(device="cuda").manual_seed(3)
    for what, grad, eps, rel in ((c.g, grads[0], 2.0 ** -5, 5e-3), (c.x, grads[1], 0.5, 1e-4), (c.h0, grads[2], 0.5, 1e-4)):
        v = torch.sign(grad).float() * torch.rand(what.shape, generator=gen, device="cuda")
        keep = what.clone()
        what.copy_(keep + eps * v)
        up = value()
        what.copy_(keep - eps * v)
        down = value()
        what.copy_(keep)
        want = float((grad * v.double()).sum())
        assert abs((up - down) / (2 * eps) - want) <= rel * abs(want)


@pytest.mark.parametrize("max_frames", [None, 0])
def test_captured_and_replayed(ctx, max_frames):
    """Forward and backward captured into one graph; every replay on new inputs equals the eager call bit for bit."""
    import torch
    stream = torch.cuda.Stream()
    side = host.Context(0, stream.cuda_stream)
    c = Case(ctx, [300, 17, 129], 36, "bf16", True, max_frames=max_frames)
    with torch.cuda.stream(stream):
        c.run(side)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            c.run(side)
    for k in range(3):
        c.x.normal_()
        c.g.normal_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in (c.h, c.hl, c.dg, c.dx, c.d0)]
        c.run()
        ctx.sync()
        assert all(torch.equal(a, b) for a, b in zip(got, (c.h, c.hl, c.dg, c.dx, c.d0))), k
    side.close()


def test_two_contexts_at_once(ctx):
    other = host.Context(0)
    a, b = Case(ctx, [500] * 20, 64, "f32", True, seed=1), Case(ctx, [900, 0, 30], 64, "f32", True, max_frames=0, seed=2)
    for _ in range(5):
        a.run()
        b.run(other)
    ctx.sync()
    other.sync()
    a.check()
    b.check()
    other.close()


def test_refusals(ctx):
    c = Case(ctx, [300], 20, "f32", False, max_frames=0)
    import torch
    with pytest.raises(ValueError):
        host.gated_scan(ctx, c.mode, c.g[:, :19], c.x, c.offd, 0, c.h, scratch=c.scratch)
    with pytest.raises(ValueError):
        host.gated_scan(ctx, c.mode, c.g.half(), c.x, c.offd, 0, c.h, scratch=c.scratch)
    with pytest.raises(ValueError):
        host.gated_scan(ctx, c.mode, c.g, c.x, c.offd.int(), 0, c.h, scratch=c.scratch)
    with pytest.raises(ValueError):
        host.gated_scan(ctx, c.mode, c.g, c.x, c.offd, 0, c.h, states=c.states[:100], scratch=c.scratch)
    with pytest.raises(ValueError):
        host.gated_scan(ctx, c.mode, c.g.cpu(), c.x, c.offd, 0, c.h, scratch=c.scratch)
    with pytest.raises(_capi.SrxError, match="scratch"):
        host.gated_scan(ctx, c.mode, c.g, c.x, c.offd, 0, c.h)
    with pytest.raises(_capi.SrxError, match="mode"):
        host.gated_scan(ctx, 7, c.g, c.x, c.offd, 0, c.h, scratch=c.scratch)
    lib, h = ctx.lib, ctx.h
    p = c.x.data_ptr()
    ok = [h, 0, 0, p, 20, p, 20, None, c.offd.data_ptr(), 1, 300, 300, 20, c.h.data_ptr(), 20, None, None, c.scratch.data_ptr(), 1 << 20]
    for i, v in ((1, 2), (2, 3), (3, None), (4, 19), (6, 19), (8, None), (9, -1), (10, -1), (11, -1), (12, 0), (13, None), (14, 19), (12, 1 << 21),
                 (10, 1 << 41), (3, p + 2)):
        a = list(ok)
        a[i] = v
        assert lib.srx_gated_scan_dev(*a) == _capi.SRX_ERR_INVALID, (i, v)
    assert lib.srx_gated_scan_scratch_bytes(h, 1, 10, 10, 0) == -1 and lib.srx_gated_scan_states_len(h, -1, 10, 3) == -1
    empty = torch.zeros(1, dtype=torch.int64, device="cuda")
    assert lib.srx_gated_scan_dev(h, 0, 0, None, 20, None, 20, None, empty.data_ptr(), 0, 0, 0, 20, None, 20, None, None, None, 0) == 0
