"""Emission scores held by torch go into the alignment and the decoder as those of a DevArray do."""
import numpy as np
import pytest
import torch

from speechrecognition_amd import host, synth
from tests.test_learned_wrappers import Ctx


def _batch(ctx):
    h = host.HmmBatch.__new__(host.HmmBatch)
    h.ctx, h.c, h.total_frames, h.n_utt = ctx, host.srx_hmm_batch(), 5, 1
    return h


def test_addresses_and_refusals():
    c = Ctx()
    out = [type("A", (), dict(ptr=v)) for v in (11, 12, 13)]
    e = torch.zeros(7, 8)
    got = _batch(c).viterbi(e, 1, 8, path_d=out[0], final_d=out[1], status_d=out[2])
    assert got == tuple(out) and c.last()[2:] == (e.data_ptr(), 1, 8, 1e10, 11, 12, 13)
    for bad in (e.half(), e.long(), torch.zeros(7, 8, device="meta")):
        c.device = -1 if bad.device.type == "cpu" else 0
        with pytest.raises(ValueError, match="emission"):
            _batch(c).viterbi(bad, 1, 8, path_d=out[0], final_d=out[1], status_d=out[2])


@pytest.mark.gpu
def test_alignment_and_decode(ctx):
    rng = np.random.default_rng(7)
    lens, G = [90, 41, 160], 37
    off = np.concatenate([[0], np.cumsum(lens)]).astype(np.int64)
    T = int(off[-1])
    ntrs, trs, tieds = [], [], []
    for _ in lens:
        ph = synth.phone_string(rng, 2, 14)
        ntr, tr, _ = host.build_training_hmm(ph)
        ntrs.append(ntr)
        trs.append(tr)
        tieds.append(rng.integers(0, G, len(ph)).astype(np.int32))
    hb = host.HmmBatch(ctx, off, ntrs, trs, tieds)
    k16, D = 112, 100
    xq, wq = (torch.randint(-127, 128, (n, k16), dtype=torch.int8, device="cuda") for n in (T, G))
    wq[:, D:] = 0
    xs, ws = torch.full((T,), 0.01, device="cuda"), torch.full((G,), 0.01, device="cuda")
    Tp = (T + 3) // 4 * 4
    emis = torch.zeros((G, Tp), device="cuda")
    torch.cuda.synchronize()
    host.matmul_i8(ctx, xq, xs, wq, ws, D, emis, by_state=True)
    a = [v.get() for v in hb.viterbi(emis, 1, Tp)]
    held = ctx.array(emis.cpu().numpy())
    b = [v.get() for v in hb.viterbi(held, 1, Tp)]
    assert all(x.tobytes() == y.tobytes() for x, y in zip(a, b)) and (a[2] == 0).all()
    states = np.concatenate([[0], np.cumsum(ntrs[0])]).astype(np.int32)
    to = np.concatenate([np.arange(s, s + n) for s, n in enumerate(ntrs[0])]).astype(np.int32)
    graph = host.GraphHmm(ctx, states, to, np.concatenate([trs[0][s, :n] for s, n in enumerate(ntrs[0])]).astype(np.float32), tieds[0])
    a, b = (graph.viterbi(e, 1, Tp, off[:2]) for e in (emis, held))
    assert all(x.tobytes() == y.tobytes() for x, y in zip(a, b)) and (a[3] == 0).all()
    with pytest.raises(ValueError):
        graph.viterbi(emis.half(), 1, Tp, off[:2])
    graph.close()
    with pytest.raises(ValueError):
        hb.viterbi(emis.cpu(), 1, Tp)
    with pytest.raises(ValueError):
        hb.viterbi(emis.double(), 1, Tp)
