"""The learned layers' Python calls without a GPU: what reaches the C ABI, and what is refused before it."""
import numpy as np
import pytest
import torch

from speechrecognition_amd import _capi, host


class Lib:
    """Records calls; sizes as the library answers for a batch that is not cut."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*a):
            assert len(a) == len(_capi.SIGNATURES[name][1]), name
            self.calls.append((name, a))
            return 256 if name.endswith("_bytes") or name.endswith("_len") else 0
        return call


class Ctx:
    device, h = -1, None                          # (a CPU tensor's get_device() is -1)

    def __init__(self):
        self.lib = Lib()

    def last(self):
        return self.lib.calls[-1][1]


@pytest.fixture
def c():
    return Ctx()


def test_recurrence(c):
    g, x, h = (torch.zeros(5, 8)[:, :6] for _ in range(3))
    off, h0 = torch.tensor([0, 2, 5]), torch.zeros(2, 6)
    host.gated_scan(c, host.SCAN_SIGMOID, g, x, off, 3, h, h0=h0, h_last=h0)
    a = c.last()
    assert a[1:5] == (1, _capi.SRX_F32, g.data_ptr(), 8) and a[5:13] == (x.data_ptr(), 8, h0.data_ptr(), off.data_ptr(), 2, 5, 3, 6) and a[13:18] == (h.data_ptr(), 8, h0.data_ptr(), None, None)
    for bad in (dict(gate=g[:, :5]), dict(gate=g.half()), dict(gate=g.t()), dict(h=h[:4]), dict(off=off.int()), dict(off=torch.zeros(2, 3, dtype=torch.int64).t()),
                dict(h0=h0[:1]), dict(h0=h0.double()), dict(x=x.long()), dict(states=torch.zeros(3)), dict(x=torch.zeros(5, 1).expand(5, 6))):
        k = dict(gate=g, x=x, off=off, h=h, h0=h0, states=None)
        k.update(bad)
        with pytest.raises(ValueError):
            host.gated_scan(c, host.SCAN_VALUE, k["gate"], k["x"], k["off"], 3, k["h"], h0=k["h0"], states=k["states"])
    with pytest.raises(ValueError):               # the states are not optional here
        host.gated_scan_backward(c, host.SCAN_VALUE, g, x, off, 3, None, x, g, h)


def test_groups(c):
    x, w, off, y = torch.zeros(5, 6, dtype=torch.bfloat16), torch.zeros(2, 4, 6, dtype=torch.bfloat16), torch.tensor([0, 2, 5]), torch.zeros(5, 4)
    host.group_matmul(c, x, w, off, y)
    assert c.last()[1:] == (_capi.SRX_BF16, _capi.SRX_F32, x.data_ptr(), 6, w.data_ptr(), None, off.data_ptr(), 2, 5, 6, 4, y.data_ptr(), 4)
    dy = torch.zeros(5, 4, dtype=torch.bfloat16)
    host.group_matmul_dx(c, dy, w, off, x)
    assert c.last()[1:] == (_capi.SRX_BF16, _capi.SRX_BF16, dy.data_ptr(), 4, w.data_ptr(), off.data_ptr(), 2, 5, 6, 4, x.data_ptr(), 6)
    host.group_matmul_dw(c, dy, x, off, w)
    assert c.last()[1:3] == (2, 2) and c.last()[8:12] == (2, 5, 6, 4)
    for a in ((x, w[:1], off, y), (x, w.float(), off, y), (x, w.transpose(1, 2), off, y), (x, w, off[:2], y), (x, w, off, y[:, :3]), (x, w, off, y.double()),
              (x[:, :5], w, off, y), (x, torch.zeros(2, 4, 12, dtype=torch.bfloat16)[:, :, ::2], off, y)):
        with pytest.raises(ValueError):
            host.group_matmul(c, *a)
    with pytest.raises(ValueError):
        host.group_matmul(c, x, w, off, y, bias=torch.zeros(4))
    with pytest.raises(ValueError):
        host.group_matmul_dw(c, dy, x[:4], off, w)


def test_8_bit(c):
    x, q, s = torch.zeros(5, 20), torch.zeros(5, 32, dtype=torch.int8), torch.zeros(5)
    host.quantize_rows(c, x, q, s)
    assert c.last()[1:] == (_capi.SRX_F32, x.data_ptr(), 20, 5, 20, q.data_ptr(), 32, s.data_ptr())
    wq, ws = torch.zeros(7, 32, dtype=torch.int8), torch.zeros(7)
    y = torch.zeros(5, 7)
    host.matmul_i8(c, q, s, wq, ws, 20, y)
    assert c.last()[9:] == (5, 7, 20, y.data_ptr(), 7, 1)
    t = torch.zeros(7, 8)
    host.matmul_i8(c, q, s, wq, ws, 20, t, by_state=True)
    assert c.last()[9:] == (5, 7, 20, t.data_ptr(), 1, 8)
    host.matmul_i8(c, q, s, wq, ws, 20, t.t()[:5])
    assert c.last()[9:] == (5, 7, 20, t.data_ptr(), 1, 8)
    host.matmul_i8(c, q[:1], s[:1], wq, ws, 20, y[:1])
    assert c.last()[9:] == (1, 7, 20, y.data_ptr(), 7, 1)
    host.matmul_i8(c, q[:1], s[:1], wq, ws, 20, t[:, :1].t())
    assert c.last()[9:] == (1, 7, 20, t.data_ptr(), 1, 8)
    for bad in ((q, s, wq, ws, 33, y), (q, s[:4], wq, ws, 20, y), (q, s, wq, ws[:6], 20, y), (q.short(), s, wq, ws, 20, y), (q, s, wq, ws, 20, y[:4]), (q, s, wq, ws, 20, y.double())):
        with pytest.raises(ValueError):
            host.matmul_i8(c, *bad)
    for bad in (torch.zeros(6, 8), torch.zeros(7, 4), torch.zeros(8, 7).t()):
        with pytest.raises(ValueError):
            host.matmul_i8(c, q, s, wq, ws, 20, bad, by_state=True)
    with pytest.raises(ValueError):
        host.quantize_rows(c, x, q[:, :16], s)


def test_types_of_arrays(c):
    class Array(host.DevArray):
        def __init__(self, v):
            self.ctx, self.shape, self.dtype, self.v = c, v.shape, v.dtype, v
            self.ptr = type("P", (), dict(value=v.ctypes.data))

        def free(self):
            pass

    for t, code in ((np.float32, 0), (np.float16, 1), (np.uint16, 2)):
        x, w, off = Array(np.zeros((5, 6), t)), Array(np.zeros((1, 4, 6), t)), Array(np.array([0, 5]))
        y = Array(np.zeros((5, 4), t))
        host.group_matmul(c, x, w, off, y)
        assert c.last()[1:5] == (code, code, x.data_ptr(), 6)
    with pytest.raises(ValueError):
        host.group_matmul(c, Array(np.zeros((5, 6), np.int16)), w, off, y)
