"""The learned layers together, as a recogniser runs and trains them: features -> a transform per speaker -> gated recurrence ->
8-bit output layer over the tied states -> Viterbi; and the gradients of a transform under a recurrence.  Nothing waits between the
calls; every stage is compared with its 64-bit form (tests/learned_ref.py).  No counterpart in the reference."""
import numpy as np
import pytest

from speechrecognition_amd import host, synth
from tests import learned_ref as R

pytestmark = pytest.mark.gpu


def _offsets(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int64)


def _within(got, want, tol):
    bad = ~(np.abs(got.astype(np.float64) - want) <= tol)
    assert not bad.any(), (int(bad.sum()), bad.shape, np.argwhere(bad)[:4].tolist())


def _features(ctx, lens, rng):
    cfg = host.mfcc_config()
    samples = rng.normal(size=sum(lens)).astype(np.float32) * 0.1
    plan = host.MfccPlan(ctx, cfg, host.mel_filterbank()[0])
    ceps, off = plan.write_features(samples, _offsets(lens))
    plan.close()
    return host.read_features(ctx, ceps, off), off


class Recogniser:
    """39 features -> 39 per speaker -> gate and value of D units -> recurrence -> G state scores."""

    def __init__(self, ctx, feats, off, D, G, rng):
        self.ctx, self.off, self.T, self.n, self.D, self.G = ctx, off, len(feats), len(off) - 1, D, G
        K = feats.shape[1]
        self.spk = (np.eye(K) + rng.normal(size=(self.n, K, K)) * 0.1).astype(np.float32)
        self.spk_b = rng.normal(size=(self.n, K)).astype(np.float32)
        self.wi = (rng.normal(size=(2, D, K)) * 0.2).astype(np.float32)
        self.wo = rng.normal(size=(G, D)).astype(np.float32)
        self.bo = rng.normal(size=G).astype(np.float32) - 20
        a, e = ctx.array, ctx.empty
        self.feats, self.offd = a(feats), a(off)
        self.d = [a(v) for v in (self.spk, self.spk_b, self.wi[:1], self.wi[1:], self.wo, self.bo)]
        self.all = a(np.array([0, self.T], np.int64))
        self.y, self.gate, self.x, self.h = e((self.T, K), np.float32), e((self.T, D), np.float32), e((self.T, D), np.float32), e((self.T, D), np.float32)
        k16 = (D + 15) // 16 * 16
        self.q, self.s, self.wq, self.ws = e((self.T, k16), np.int8), e(self.T, np.float32), e((G, k16), np.int8), e(G, np.float32)
        self.Tp = (self.T + 3) // 4 * 4
        self.emis = e((G, self.Tp), np.float32)
        self.scratch = e(max(host.gated_scan_scratch_bytes(ctx, self.n, self.T, int(np.diff(off).max()), D), 4), np.uint8)
        host.quantize_rows(ctx, self.d[4], self.wq, self.ws)

    def run(self):
        c, (spk, spk_b, wg, wx, _, bo) = self.ctx, self.d
        host.group_matmul(c, self.feats, spk, self.offd, self.y, bias=spk_b)
        host.group_matmul(c, self.y, wg, self.all, self.gate)
        host.group_matmul(c, self.y, wx, self.all, self.x)
        host.gated_scan(c, host.SCAN_SIGMOID, self.gate, self.x, self.offd, int(np.diff(self.off).max()), self.h, scratch=self.scratch)
        host.quantize_rows(c, self.h, self.q, self.s)
        host.matmul_i8(c, self.q, self.s, self.wq, self.ws, self.D, self.emis, bias=bo, by_state=True)

    def check(self):
        one = np.array([0, self.T])
        f, y, gate, x, h, q, s = (v.get() for v in (self.feats, self.y, self.gate, self.x, self.h, self.q, self.s))
        y64 = y.astype(np.float64)
        for got, (want, err) in ((y, R.group(f.astype(np.float64), self.spk, self.off, self.spk_b, "f32")), (gate, R.group(y64, self.wi[:1], one, None, "f32")),
                                 (x, R.group(y64, self.wi[1:], one, None, "f32"))):
            _within(got, want, R.out_bound(want, err, "f32"))
        ref = R.scan(gate.astype(np.float64), x.astype(np.float64), self.off, None, True)
        _within(h, ref["h"], R.out_bound(ref["h"], ref["eh"], "f32"))
        ws, wq = R.quantize(h)
        assert s.tobytes() == ws.tobytes() and (q[:, :self.D] == wq).all() and (q[:, self.D:] == 0).all()
        want, err = R.i8(q[:, :self.D], s, self.wq.get()[:, :self.D], self.ws.get(), self.bo)
        emis = self.emis.get()[:, :self.T].T
        _within(emis, want, R.out_bound(want, err, "f32"))
        return np.ascontiguousarray(emis)


def test_features_to_alignment(ctx, oracle):
    rng = np.random.default_rng(1)
    feats, off = _features(ctx, [32000, 9600, 21111, 48000, 14400], rng)
    G = 50
    r = Recogniser(ctx, feats, off, 100, G, rng)
    ntrs, trs, tieds = [], [], []
    for _ in range(r.n):
        ph = synth.phone_string(rng, 2, 24)
        ntr, tr, _ = host.build_training_hmm(ph)
        ntrs.append(ntr)
        trs.append(tr)
        tieds.append(rng.integers(0, G, len(ph)).astype(np.int32))
    hb = host.HmmBatch(ctx, off, ntrs, trs, tieds)
    r.run()
    path, final, status = hb.viterbi(r.emis, 1, r.Tp)
    ctx.sync()
    emis, path, final, status = r.check(), path.get(), final.get(), status.get()
    for u in range(r.n):
        want = oracle.viterbi(emis[off[u]:off[u + 1]], tieds[u], ntrs[u], trs[u], 1e10, 0)
        assert status[u] == want["status"] == 0
        assert final[u].tobytes() == want["final"].tobytes() and np.array_equal(path[off[u]:off[u + 1]], want["path"])


def test_two_contexts_side_by_side(ctx):
    """Two streams, each with its own buffers, queued without waiting: as one after the other."""
    rng = np.random.default_rng(2)
    feats, off = _features(ctx, [20000, 33000, 4000], rng)
    other = host.Context(0)
    a, b = Recogniser(ctx, feats, off, 72, 130, rng), Recogniser(other, feats[::-1].copy(), off, 264, 2000, rng)
    ctx.sync()
    other.sync()
    for _ in range(5):
        a.run()
        b.run()
    ctx.sync()
    other.sync()
    together = a.emis.get()[:, :a.T], b.emis.get()[:, :b.T]
    a.check()
    b.check()
    a.run()
    ctx.sync()
    b.run()
    other.sync()
    assert together[0].tobytes() == a.emis.get()[:, :a.T].tobytes() and together[1].tobytes() == b.emis.get()[:, :b.T].tobytes()
    del b
    other.close()


@pytest.mark.parametrize("lens,K,D", [([70, 0, 1, 130, 16], 39, 64), ([900, 30], 24, 100), ([5] * 60, 13, 7)])
def test_training_step(ctx, lens, K, D):
    """y = W_u x + b_u, h = recurrence of y with given gates, value = sum h c: all gradients against the whole chain in 64 bits.  An
    error e of y moves h by the recurrence of |gates| over e; one of lambda moves dW, db and dx by the products of magnitudes.
    Bounds are of first order: 1 % is left for the rest."""
    rng = np.random.default_rng(3)
    off, T, n = _offsets(lens), sum(lens), len(lens)
    x, c = (rng.normal(size=(T, k)).astype(np.float32) for k in (K, D))
    w, b = (rng.normal(size=(n, D, K)) / np.sqrt(K)).astype(np.float32), rng.normal(size=(n, D)).astype(np.float32)
    a = rng.uniform(-0.2, 1, (T, D)).astype(np.float32)
    h0, cl = (rng.normal(size=(n, D)).astype(np.float32) for _ in range(2))
    longest = max(lens)
    d = {k: ctx.array(v) for k, v in dict(x=x, c=c, w=w, b=b, a=a, h0=h0, cl=cl, off=off).items()}
    o = {k: ctx.empty(s, np.float32) for k, s in dict(y=(T, D), h=(T, D), hl=(n, D), da=(T, D), dy=(T, D), dh0=(n, D), dx=(T, K), dw=(n, D, K), db=(n, D)).items()}
    states = ctx.empty(max(host.gated_scan_states_bytes(ctx, n, T, D), 4), np.uint8)
    room = ctx.empty(max(host.gated_scan_scratch_bytes(ctx, n, T, longest, D), host.group_matmul_dw_scratch_bytes(ctx, n, T, K, D), 16), np.uint8)
    host.group_matmul(ctx, d["x"], d["w"], d["off"], o["y"], bias=d["b"])
    host.gated_scan(ctx, host.SCAN_VALUE, d["a"], o["y"], d["off"], longest, o["h"], h0=d["h0"], h_last=o["hl"], states=states, scratch=room)
    host.gated_scan_backward(ctx, host.SCAN_VALUE, d["a"], o["y"], d["off"], longest, states, d["c"], o["da"], o["dy"], dh_last=d["cl"], dh0=o["dh0"], scratch=room)
    host.group_matmul_dx(ctx, o["dy"], d["w"], d["off"], o["dx"])
    host.group_matmul_dw(ctx, o["dy"], d["x"], d["off"], o["dw"], dbias=o["db"], scratch=room)
    ctx.sync()
    got = {k: v.get() for k, v in o.items()}

    x, c, a, w = (v.astype(np.float64) for v in (x, c, a, w))
    y, ey = R.group(x, w, off, b, "f32")
    ey = R.out_bound(y, ey, "f32")
    f = R.scan(a, y, off, h0, False)
    moved = R.scan(np.abs(a), ey, off, None, False)
    back = R.scan_back(f, a, y, off, c, cl, False)
    lam, el = back["dx"], R.out_bound(back["dx"], back["edx"], "f32")
    bound = {k: R.out_bound(v, e, "f32") * 1.01 for k, v, e in (("y", y, ey), ("h", f["h"], f["eh"] + moved["h"]), ("hl", f["last"], f["elast"] + moved["last"]),
                                                              ("da", back["dg"], back["edg"] + np.abs(lam) * moved["prev"]), ("dy", lam, el),
                                                              ("dh0", back["d0"], back["e0"]))}
    for k, v in dict(y=y, h=f["h"], hl=f["last"], da=back["dg"], dy=lam, dh0=back["d0"]).items():
        _within(got[k], v, bound[k])
    dx, edx = R.group(lam, w.transpose(0, 2, 1), off, None, "f32")
    more, _ = R.group(el, np.abs(w).transpose(0, 2, 1), off, None, "f32")
    _within(got["dx"], dx, R.out_bound(dx, edx + more, "f32") * 1.01)
    dw, edw, db, edb = R.group_dw(lam, x, off, "f32")
    mw, _, mb, _ = R.group_dw(el, np.abs(x), off, "f32")
    _within(got["dw"], dw, R.out_bound(dw, edw + mw, "f32") * 1.01)
    _within(got["db"], db, R.out_bound(db, edb + mb, "f32") * 1.01)


def test_bf16_words_of_numpy(ctx):
    """numpy has no bf16: a uint16 buffer holds its words."""
    rng = np.random.default_rng(4)
    words = lambda *s: (rng.normal(size=s).astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)  # noqa: E731
    wide = lambda v: (v.astype(np.uint32) << 16).view(np.float32).astype(np.float64)  # noqa: E731
    x, w, off = words(90, 40), words(2, 72, 40), _offsets([33, 57])
    y, y32 = ctx.empty((90, 72), np.uint16), ctx.empty((90, 72), np.float32)
    xd, wd, od = ctx.array(x), ctx.array(w), ctx.array(off)
    host.group_matmul(ctx, xd, wd, od, y)
    host.group_matmul(ctx, xd, wd, od, y32)
    ctx.sync()
    want, err = R.group(wide(x), wide(w), off, None, "bf16")
    _within(wide(y.get()), want, R.out_bound(want, err, "bf16"))
    _within(y32.get(), want, R.out_bound(want, err, "f32"))
    with pytest.raises(ValueError):
        host.group_matmul(ctx, ctx.empty((90, 40), np.int32), wd, od, y)
