"""srx_quantize_rows_dev (codes and scales bit for bit) and srx_matmul_i8_dev (an exact sum: within the roundings of its
scales) against their definitions (tests/learned_ref.py).  No counterpart in the reference."""
import numpy as np
import pytest

from speechrecognition_amd import _capi, host
from tests import learned_ref as R

pytestmark = pytest.mark.gpu


def _t(dtype):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,K,pad,shift", [(1, 1, 0, 0), (5, 15, 0, 0), (6, 16, 3, 1), (33, 39, 0, 0), (9, 512, 8, 0), (4, 1000, 1, 3), (3, 2056, 0, 0), (2, 9000, 8, 8)])
def test_codes_and_scales(ctx, dtype, rows, K, pad, shift):
    import torch
    r = np.random.default_rng(K)
    v = r.normal(size=(rows, K)) * np.exp(r.uniform(-20 if dtype != "f16" else -5, 5, (rows, 1)))
    if rows > 4:
        v[2] = 0.0
        v[3] = np.arange(K) % 255 - 127          # whole codes at scale 1 (K > 254) and their halves: ties
        v[4] = (np.arange(K) % 509 - 254) / 2
        v[3, 0], v[4, 0] = 127, 127
    buf = torch.zeros(rows * (K + pad) + shift + 8, dtype=_t(dtype), device="cuda")
    x = buf[shift:shift + rows * (K + pad)].view(rows, K + pad)[:, :K]
    x.copy_(torch.from_numpy(v))
    k16 = (K + 15) // 16 * 16
    q = torch.full((rows + 1, k16 + 16), 77, dtype=torch.int8, device="cuda")
    s = torch.full((rows,), 5.0, device="cuda")
    torch.cuda.synchronize()
    host.quantize_rows(ctx, x, q[:rows], s)
    ctx.sync()
    ws, wq = R.quantize(x.float().cpu().numpy())
    got = q.cpu().numpy()
    assert s.cpu().numpy().tobytes() == ws.tobytes()
    assert (got[:rows, :K] == wq).all()
    assert (got[:rows, K:k16] == 0).all() and (got[:rows, k16:] == 77).all() and (got[rows] == 77).all()


def _operands(torch, rows, N, K, seed, pad=0):
    r = np.random.default_rng(seed)
    k16 = (K + 15) // 16 * 16 + pad
    xq, wq = (r.integers(-127, 128, (n, k16)).astype(np.int8) for n in (rows, N))
    xq[:, K:] = 99                                # behind K only one operand has to hold zeros
    wq[:, K:] = 0
    xs, ws, b = r.uniform(0.001, 2, rows).astype(np.float32), r.uniform(0.001, 2, N).astype(np.float32), r.normal(size=N).astype(np.float32)
    return [torch.from_numpy(v).cuda() for v in (xq, xs, wq, ws, b)]


@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("by_state", [False, True])
@pytest.mark.parametrize("rows,N,K", [(1, 1, 1), (1, 2000, 512), (4, 130, 39), (3, 2001, 2048), (17, 40, 129), (33, 300, 16), (130, 129, 400), (300, 520, 1025)])
def test_products(ctx, out, by_state, rows, N, K):
    import torch
    xq, xs, wq, ws, b = _operands(torch, rows, N, K, rows + N + K)
    xs, ws = (v * (0.01 if out == "f16" else 1) for v in (xs, ws))
    store = torch.full((N, rows + 3) if by_state else (rows, N + 5), 7.0, dtype=_t(out), device="cuda")
    y = store.t()[:rows] if by_state else store[:, :N]
    torch.cuda.synchronize()
    for bias in (b, None):
        host.matmul_i8(ctx, xq, xs, wq, ws, K, y, bias=bias)
        ctx.sync()
        n = lambda t: t.cpu().numpy()  # noqa: E731
        want, err = R.i8(n(xq)[:, :K], n(xs), n(wq)[:, :K], n(ws), None if bias is None else n(b))
        got = y.double().cpu().numpy()
        assert (np.abs(got - want) <= R.out_bound(want, err, out)).all()
        rest = store[:, rows:] if by_state else store[:, N:]
        assert (rest == 7.0).all()


def test_largest_sum_is_exact(ctx):
    """K at its limit with every code -127 or 127: the 32-bit sum does not overflow and is exact."""
    import torch
    K = _capi.SRX_I8_MAX_K
    xq, wq = torch.full((2, K), -127, dtype=torch.int8, device="cuda"), torch.full((33, K), 127, dtype=torch.int8, device="cuda")
    wq[1, ::2] = -127
    one = torch.ones(40, device="cuda")
    y = torch.zeros((2, 33), device="cuda")
    torch.cuda.synchronize()
    host.matmul_i8(ctx, xq, one[:2].contiguous(), wq, one[:33].contiguous(), K, y)
    ctx.sync()
    want = torch.full((2, 33), float(-127 * 127 * K), device="cuda")
    want[:, 1] = 0
    assert torch.equal(y, want)


def test_rows_without_a_scale(ctx):
    """Rows of zeros give the bias, rows that hold a NaN or an infinity give NaN, the others are not touched by them."""
    import torch
    x = torch.randn(40, 100, device="cuda")
    x[3] = 0
    x[5, 7] = float("nan")
    x[6, 9] = float("-inf")
    _, _, wq, ws, b = _operands(torch, 1, 50, 100, 0)
    q, s, y = torch.zeros((40, 112), dtype=torch.int8, device="cuda"), torch.zeros(40, device="cuda"), torch.zeros((40, 50), device="cuda")
    torch.cuda.synchronize()
    host.quantize_rows(ctx, x, q, s)
    host.matmul_i8(ctx, q, s, wq, ws, 100, y, bias=b)
    ctx.sync()
    assert torch.equal(y[3], b) and torch.isnan(y[5:7]).all()
    keep = [i for i in range(40) if i not in (5, 6)]
    assert torch.isfinite(y[keep]).all()


def test_captured_and_replayed(ctx):
    import torch
    stream = torch.cuda.Stream()
    side = host.Context(0, stream.cuda_stream)
    _, _, wq, ws, b = _operands(torch, 1, 200, 64, 1)
    x, q, s, y = torch.randn(5, 64, device="cuda"), torch.zeros((5, 64), dtype=torch.int8, device="cuda"), torch.zeros(5, device="cuda"), torch.zeros((5, 200), device="cuda")

    def both(c):
        host.quantize_rows(c, x, q, s)
        host.matmul_i8(c, q, s, wq, ws, 64, y, bias=b)

    with torch.cuda.stream(stream):
        both(side)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            both(side)
    for _ in range(3):
        x.normal_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        both(ctx)
        ctx.sync()
        assert torch.equal(got, y)
    side.close()


def test_refusals(ctx):
    import torch
    xq, xs, wq, ws, b = _operands(torch, 4, 20, 40, 0)
    x, y = torch.randn(4, 40, device="cuda"), torch.zeros((4, 20), device="cuda")
    with pytest.raises(ValueError):
        host.quantize_rows(ctx, x, xq[:, :40], xs)
    with pytest.raises(_capi.SrxError, match="16"):
        host.quantize_rows(ctx, x, torch.zeros((4, 49), dtype=torch.int8, device="cuda"), xs)
    with pytest.raises(ValueError):
        host.quantize_rows(ctx, x, xq, xs[:3])
    with pytest.raises(ValueError):
        host.matmul_i8(ctx, xq, xs, wq, ws, 49, y)
    with pytest.raises(ValueError):
        host.matmul_i8(ctx, xq, xs, wq, ws, 40, y[:, :19])
    with pytest.raises(_capi.SrxError, match="strides"):
        host.matmul_i8(ctx, xq, xs, wq, ws, 40, torch.zeros((4, 40), device="cuda")[:, ::2])
    with pytest.raises(ValueError):
        host.matmul_i8(ctx, xq.float(), xs, wq, ws, 40, y)
    lib, h = ctx.lib, ctx.h
    P = [t.data_ptr() for t in (xq, xs, wq, ws, b, y)]
    ok = [h, 0, P[0], 48, P[1], P[2], 48, P[3], P[4], 4, 20, 40, P[5], 20, 1]
    for i, v in ((1, 3), (2, None), (2, P[0] + 8), (3, 40), (3, 32), (4, None), (5, None), (6, 49), (7, None), (9, -1), (10, 0), (11, 0), (11, _capi.SRX_I8_MAX_K + 1),
                 (12, None), (13, 19), (14, 2)):
        a = list(ok)
        a[i] = v
        assert lib.srx_matmul_i8_dev(*a) == _capi.SRX_ERR_INVALID, (i, v)


@pytest.mark.parametrize("out,by_state,pad", [("f32", False, 0), ("f32", True, 3), ("bf16", False, 1), ("f16", True, 0)])
def test_many_large_tiles(ctx, out, by_state, pad):
    """Enough scores for the 256 x 256 tiles, in both layouts, on lines of memory and off them."""
    import torch
    rows, N, K = 33011, 2000, 200
    xq, xs, wq, ws, b = _operands(torch, rows, N, K, 3)
    xs, ws = xs * 0.01, ws * 0.01
    store = torch.full((N, rows + pad) if by_state else (rows, N + pad), 7.0, dtype=_t(out), device="cuda")
    y = store.t()[:rows] if by_state else store[:, :N]
    torch.cuda.synchronize()
    host.matmul_i8(ctx, xq, xs, wq, ws, K, y, bias=b)
    ctx.sync()
    v = (xq[:, :K].double() @ wq[:, :K].double().t()) * xs.double()[:, None] * ws.double()
    want = v + b.double()
    err = 3.01 * R.U * v.abs() + R.U * want.abs()
    assert (torch.abs(y.double() - want) <= err + R.HALF[out] * (want.abs() + err) + R.TINY[out]).all()
    assert ((store[:, rows:] if by_state else store[:, N:]) == 7.0).all()


@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("by_state", [False, True])
@pytest.mark.parametrize("rows,N,K", [(700, 1003, 400), (2101, 260, 129), (5000, 33, 39), (300, 2001, 1025), (3000, 1025, 16)])
def test_more_small_tiles_than_the_chip_holds(ctx, out, by_state, rows, N, K):
    """Sizes that take the 128- and 256-row tiles, in odd numbers."""
    import torch
    xq, xs, wq, ws, b = _operands(torch, rows, N, K, rows + N + K)
    xs, ws = (v * (0.01 if out == "f16" else 1) for v in (xs, ws))
    store = torch.full((N, rows + 3) if by_state else (rows, N + 5), 7.0, dtype=_t(out), device="cuda")
    torch.cuda.synchronize()
    host.matmul_i8(ctx, xq, xs, wq, ws, K, store if by_state else store[:, :N], bias=b, by_state=by_state)
    ctx.sync()
    want = torch.from_numpy((xq.cpu().numpy()[:, :K].astype(np.float64) @ wq.cpu().numpy()[:, :K].T.astype(np.float64))).cuda()
    want = want * xs.double()[:, None] * ws.double()
    y = want + b.double()
    err = 3.01 * R.U * want.abs() + R.U * y.abs()
    got = (store.t()[:rows] if by_state else store[:, :N]).double()
    assert bool(((got - y).abs() <= err + R.HALF[out] * (y.abs() + err) + R.TINY[out]).all())
    assert bool(((store[:, rows:] if by_state else store[:, N:]) == 7.0).all())


def test_misaligned_scales_are_refused(ctx):
    import torch
    xq, xs, wq, ws, b = _operands(torch, 4, 20, 40, 0)
    y = torch.zeros((4, 20), device="cuda")
    for i in range(3):
        p = [v.data_ptr() + (2 if k == i else 0) for k, v in enumerate((xs, ws, b))]
        assert ctx.lib.srx_matmul_i8_dev(ctx.h, 0, xq.data_ptr(), 48, p[0], wq.data_ptr(), 48, p[1], p[2], 4, 20, 40, y.data_ptr(), 20, 1) == _capi.SRX_ERR_INVALID
