"""Which stream a Python context launches on: the handle that it is given -- 0 is the default stream, torch's own -- or a stream
of its own."""
import ctypes

import pytest

from speechrecognition_amd import _capi, host


class Lib:
    def __init__(self):
        self.streams = []

    def srx_ctx_create(self, device, stream, out):
        self.streams.append(stream.value if isinstance(stream, ctypes.c_void_p) else stream)
        return 0

    def srx_ctx_destroy(self, h):
        pass


def test_handles_reach_the_library(monkeypatch):
    lib = Lib()
    monkeypatch.setattr(_capi, "load", lambda: lib)
    for given in (None, 0, 0x7000):
        host.Context(0, given)
    host.Context(0)
    assert lib.streams == [None, _capi.SRX_STREAM_DEFAULT, 0x7000, None]


@pytest.mark.gpu
def test_default_stream_is_in_order_with_torch(ctx):
    """Inputs made, codes taken and their copies read without a wait in between, behind work that keeps the stream busy."""
    import numpy as np
    import torch

    from tests import learned_ref as R
    assert torch.cuda.current_stream().cuda_stream == 0
    c = host.Context(0, 0)
    assert c.stream_handle() == 0 and ctx.stream_handle() != 0
    busy = torch.randn(4096, 4096, device="cuda")
    x = torch.zeros(500, 256, device="cuda")
    q, s = torch.zeros((500, 256), dtype=torch.int8, device="cuda"), torch.zeros(500, device="cuda")
    got, src = [], [np.random.default_rng(k).normal(size=(500, 256)).astype(np.float32) for k in range(4)]
    dev = [torch.from_numpy(v).cuda() for v in src]
    for v in dev:
        for _ in range(10):
            busy = torch.mm(busy, busy).clamp_(-1, 1)
        x.copy_(v)
        host.quantize_rows(c, x, q, s)
        got.append((q.clone(), s.clone()))
        q.zero_()
    for v, (codes, scale) in zip(src, got):
        ws, wq = R.quantize(v)
        assert scale.cpu().numpy().tobytes() == ws.tobytes() and (codes.cpu().numpy() == wq).all()
    c.sync()
    c.close()
