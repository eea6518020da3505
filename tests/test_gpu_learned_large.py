"""The learned layers where a buffer passes 4 GiB and element numbers pass 32 bits, on values whose results are exact; and sizes that are
refused because no launch holds them.  No counterpart in the reference."""
import pytest

from speechrecognition_amd import _capi, host
from tests import learned_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture
def torch_():
    import torch
    yield torch
    torch.cuda.empty_cache()


def test_recurrence(ctx, torch_):
    """Gates of zero: h = x, dx = dh and dgate_t = dh_t x_(t-1), one product; the first frame of an utterance meets h0."""
    torch = torch_
    T, D = 1_100_003, 1024
    off = torch.tensor([0, 400_000, 400_000, T - 5], device="cuda")
    n, longest = 3, T - 5 - 400_000
    x = torch.empty((T, D), device="cuda").normal_()
    dh = torch.empty((T, D), device="cuda").normal_()
    gate, h, dx, dg = (torch.zeros((T, D), device="cuda") for _ in range(4))
    h0 = torch.randn((n, D), device="cuda")
    last = torch.zeros((n, D), device="cuda")
    states = torch.empty(host.gated_scan_states_bytes(ctx, n, T, D), dtype=torch.uint8, device="cuda")
    scratch = torch.empty(max(host.gated_scan_scratch_bytes(ctx, n, T, longest, D), 4), dtype=torch.uint8, device="cuda")
    assert x.numel() * 4 > 1 << 32
    torch.cuda.synchronize()
    host.gated_scan(ctx, host.SCAN_VALUE, gate, x, off, longest, h, h0=h0, h_last=last, states=states, scratch=scratch)
    host.gated_scan_backward(ctx, host.SCAN_VALUE, gate, x, off, longest, states, dh, dg, dx, scratch=scratch)
    ctx.sync()
    end = T - 5
    assert torch.equal(h[:end], x[:end]) and torch.equal(dx[:end], dh[:end])
    assert not h[end:].any() and not dx[end:].any() and not dg[end:].any()
    assert torch.equal(last[0], x[399_999]) and torch.equal(last[1], h0[1]) and torch.equal(last[2], x[end - 1])
    for lo, hi, u in ((0, 400_000, 0), (400_000, end, 2)):
        assert torch.equal(dg[lo + 1:hi], dh[lo + 1:hi] * x[lo:hi - 1]) and torch.equal(dg[lo], dh[lo] * h0[u])


@pytest.mark.parametrize("N", [64, 200])
def test_groups(ctx, torch_, N):
    """W selects: y_r = x_r's first N columns, times 1, 2, 3 by group; dW of ones counts rows."""
    torch = torch_
    T, K, E = 2_200_001, 1024, 3
    off = torch.tensor([0, 1_000_000, 1_000_001, T - 2], device="cuda")
    x = torch.empty((T, K), dtype=torch.bfloat16, device="cuda").normal_()
    w = torch.eye(N, K, device="cuda").expand(E, N, K) * torch.arange(1, E + 1, device="cuda")[:, None, None]
    w = w.to(torch.bfloat16).contiguous()
    y = torch.zeros((T, N), device="cuda")
    assert x.numel() * 2 > 1 << 32
    torch.cuda.synchronize()
    host.group_matmul(ctx, x, w, off, y)
    ctx.sync()
    for e in range(E):
        r = slice(int(off[e]), int(off[e + 1]))
        assert torch.equal(y[r], x[r, :N].float() * (e + 1))
    assert not y[T - 2:].any()
    dx, dy = x, y.to(torch.bfloat16)                         # (over the input: not read by this call)
    torch.cuda.synchronize()
    host.group_matmul_dx(ctx, dy, w, off, dx)
    ctx.sync()
    b = slice(1_000_001, T - 2)
    assert torch.equal(dx[b, :N].float(), (dy[b].float() * 3).to(torch.bfloat16).float()) and not dx[b, N:].any()
    x.fill_(1)
    dy = torch.ones((T, N), dtype=torch.bfloat16, device="cuda")
    dw, db = torch.zeros((E, N, K), device="cuda"), torch.zeros((E, N), device="cuda")
    scratch = torch.empty(max(host.group_matmul_dw_scratch_bytes(ctx, E, T, K, N), 16), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    host.group_matmul_dw(ctx, dy, x, off, dw, dbias=db, scratch=scratch)
    ctx.sync()
    for e in range(E):
        assert (dw[e] == int(off[e + 1] - off[e])).all() and (db[e] == int(off[e + 1] - off[e])).all()


@pytest.mark.parametrize("by_state", [False, True])
def test_8_bit(ctx, torch_, by_state):
    """Codes of one place each: y_rn = whether row r's place is output n's."""
    torch = torch_
    T, N, K = 2_100_001, 1000, 64
    place = torch.randint(0, K, (T,), device="cuda")
    q = torch.zeros((T, K), dtype=torch.int8, device="cuda")
    q[torch.arange(T, device="cuda"), place] = 1
    wplace = torch.arange(N, device="cuda") % K
    wq = torch.zeros((N, K), dtype=torch.int8, device="cuda")
    wq[torch.arange(N, device="cuda"), wplace] = 3
    ones = torch.ones(T, device="cuda")
    y = torch.zeros((N, T + 3) if by_state else (T, N), device="cuda")
    assert y.numel() * 4 > 1 << 32
    torch.cuda.synchronize()
    host.matmul_i8(ctx, q, ones, wq, ones[:N].contiguous(), K, y, by_state=by_state)
    ctx.sync()
    for r in (slice(0, 1000), slice(1_073_000, 1_075_000), slice(T - 1000, T)):
        want = (place[r, None] == wplace) * 3.0
        assert torch.equal(y[:, r].t() if by_state else y[r], want)
    assert int((y != 0).sum()) == int((place[:, None] == torch.arange(K, device="cuda")).sum(0).mul(torch.bincount(wplace, minlength=K)).sum())
    assert not by_state or not y[:, T:].any()


def test_quantised_rows(ctx, torch_):
    torch = torch_
    T, K = 1_100_003, 1000
    x = torch.empty((T, K), device="cuda").normal_()
    q = torch.zeros((T, 1008), dtype=torch.int8, device="cuda")
    s = torch.zeros(T, device="cuda")
    assert x.numel() * 4 > 1 << 32
    torch.cuda.synchronize()
    host.quantize_rows(ctx, x, q, s)
    ctx.sync()
    for r in (slice(0, 2000), slice(1_073_000, 1_075_000), slice(T - 2000, T)):
        ws, wq = R.quantize(x[r].cpu().numpy())
        assert s[r].cpu().numpy().tobytes() == ws.tobytes() and (q[r, :K].cpu().numpy() == wq).all() and not q[r, K:].any()
    assert (s > 0).all()


def test_sizes_that_no_launch_holds_are_refused(ctx, torch_):
    """Refused before anything is read: the addresses are those of small buffers."""
    torch = torch_
    b = torch.zeros(4096, device="cuda")
    p, lib, h, bad = b.data_ptr(), ctx.lib, ctx.h, _capi.SRX_ERR_INVALID
    big = 1 << 30
    assert lib.srx_quantize_rows_dev(h, 0, p, 16, 1 << 26, 16, p, 16, p) == bad
    assert lib.srx_matmul_i8_dev(h, 0, p, 16, p, p, 16, p, None, 1 << 40, 16, 16, p, 16, 1) == bad
    assert lib.srx_group_matmul_dev(h, 0, 0, p, 2, p, None, p, 1, 1 << 40, 2, 64, p, 64) == bad
    assert lib.srx_group_matmul_dev(h, 0, 0, p, 64, p, None, p, 1, 1 << 40, 64, 64, p, 64) == bad
    assert lib.srx_group_matmul_dx_dev(h, 0, 0, p, 64, p, p, 1, 1 << 40, 256, 64, p, 256) == bad
    assert lib.srx_gated_scan_dev(h, 0, 0, p, 64, p, 64, None, p, big, big, 1, 64, p, 64, None, None, None, 0) == bad
    assert lib.srx_gated_scan_dev(h, 0, 0, p, 64, p, 64, None, p, 1 << 23, 1 << 24, 1 << 23, 64, p, 64, None, None, p, 1 << 50) == bad
    ctx.sync()
