"""srx_group_matmul_dev and its gradients against the products in 64 bits (tests/learned_ref.py), every element within the
bound of an f32 accumulation.  No counterpart in the reference."""
import numpy as np
import pytest

from speechrecognition_amd import _capi, host
from tests import learned_ref as R

pytestmark = pytest.mark.gpu


def _t(dtype):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]


def _strided(torch, a, dtype, pad, shift=0):
    rows, cols = a.shape
    buf = torch.full((rows * (cols + pad) + shift + 8,), -7.0, dtype=_t(dtype), device="cuda")
    v = buf[shift:shift + rows * (cols + pad)].view(rows, cols + pad)[:, :cols] if rows else buf[:0].view(0, cols)
    v.copy_(torch.from_numpy(np.ascontiguousarray(a)))
    return v


def _n(t):
    return t.double().cpu().numpy()


class Case:
    def __init__(self, ctx, lens, K, N, dtype, out=None, front=0, behind=0, pad=0, shift=0, bias=True, seed=0):
        import torch
        self.torch, self.ctx, self.dtype, self.out = torch, ctx, dtype, out or dtype
        r = np.random.default_rng(seed)
        self.off = np.concatenate([[front], front + np.cumsum(lens)]).astype(np.int64)
        self.E, self.K, self.N, self.T = len(lens), K, N, int(self.off[-1]) + behind
        self.x, self.dy = _strided(torch, r.normal(size=(self.T, K)), dtype, pad, shift), _strided(torch, r.normal(size=(self.T, N)), dtype, pad, shift)
        self.w = torch.from_numpy(r.normal(size=(self.E, N, K)) / np.sqrt(K)).cuda().to(_t(dtype))
        self.bias = torch.from_numpy(r.normal(size=(self.E, N)).astype(np.float32)).cuda() if bias else None
        self.y, self.dx = (_strided(torch, np.full((self.T, c), 5.0), self.out, pad, shift) for c in (N, K))
        self.dw = torch.full((self.E, N, K), 5.0, dtype=_t(self.out), device="cuda")
        self.db = torch.full((self.E, N), 5.0, device="cuda")
        self.offd = torch.from_numpy(self.off).cuda()
        need = host.group_matmul_dw_scratch_bytes(ctx, self.E, self.T, K, N)
        self.scratch = torch.full((max(need, 16),), 255, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()

    def run(self, ctx=None):
        ctx = ctx or self.ctx
        host.group_matmul(ctx, self.x, self.w, self.offd, self.y, bias=self.bias)
        host.group_matmul_dx(ctx, self.dy, self.w, self.offd, self.dx)
        host.group_matmul_dw(ctx, self.dy, self.x, self.offd, self.dw, dbias=self.db, scratch=self.scratch)

    def check(self):
        self.ctx.sync()
        x, dy, w = _n(self.x), _n(self.dy), _n(self.w)
        b = None if self.bias is None else _n(self.bias)
        inside = np.zeros(self.T, bool)
        for g in range(self.E):
            inside[self.off[g]:self.off[g + 1]] = True
        dw, edw, db, edb = R.group_dw(dy, x, self.off, self.dtype)
        for name, got, (want, err), kind in (("y", self.y, R.group(x, w, self.off, b, self.dtype), self.out),
                                             ("dx", self.dx, R.group(dy, w.transpose(0, 2, 1), self.off, None, self.dtype), self.out),
                                             ("dw", self.dw, (dw, edw), self.out), ("db", self.db, (db, edb), "f32")):
            got, tol = _n(got), R.out_bound(want, err, kind)
            if name in ("y", "dx"):
                assert (got[~inside] == 5.0).all(), name
                got, want, tol = got[inside], want[inside], tol[inside]
            bad = ~(np.abs(got - want) <= tol)
            assert not bad.any(), (name, int(bad.sum()), bad.shape, np.argwhere(bad)[:4].tolist())


SIZES = [([1], 1, 1), ([3, 0, 5], 39, 39), ([40, 1, 0, 200], 64, 130), ([129], 429, 33), ([7, 300], 24, 264), ([0, 0], 16, 16), ([260, 31], 96, 512)]


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("lens,K,N", SIZES)
def test_products_and_gradients(ctx, dtype, out, lens, K, N):
    c = Case(ctx, lens, K, N, dtype, out)
    c.run()
    c.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_of_no_group_stay(ctx, dtype):
    c = Case(ctx, [50, 0, 140, 3], 72, 200, dtype, front=37, behind=150)
    c.run()
    c.check()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pad,shift", [(1, 0), (8, 0), (8, 8), (3, 1), (4, 2), (16, 4)])
def test_row_strides_and_addresses(ctx, dtype, pad, shift):
    """Strides and addresses of whole 16 bytes and others take different loads, and give the same."""
    c = Case(ctx, [70, 150], 136, 272, dtype, pad=pad, shift=shift)
    c.run()
    c.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens,K,N", [([3000], 64, 40), ([1100, 0, 2500], 33, 128), ([513, 2000], 256, 264)])
def test_long_groups_are_cut_and_joined(ctx, dtype, lens, K, N):
    """Few tiles and many rows: dW is summed in parts."""
    c = Case(ctx, lens, K, N, dtype, "f32")
    assert host.group_matmul_dw_scratch_bytes(ctx, c.E, c.T, K, N) > 0
    c.run()
    c.check()
    first = c.dw.clone(), c.db.clone()
    c.run()
    c.ctx.sync()
    assert c.torch.equal(c.dw, first[0]) and c.torch.equal(c.db, first[1])


@pytest.mark.parametrize("E", [64, 65, 300, 4500])
def test_many_groups(ctx, E):
    r = np.random.default_rng(E)
    c = Case(ctx, r.integers(0, 5, E).tolist(), 20, 12, "f32", front=2, behind=1)
    c.run()
    c.check()


def test_equal_rows_of_a_group_are_equal(ctx):
    """The same input row anywhere in a group gives the same bits."""
    c = Case(ctx, [400], 128, 300, "bf16", "f32")
    c.x[:] = c.x[0]
    c.torch.cuda.synchronize()
    c.run()
    c.ctx.sync()
    assert (c.y == c.y[0]).all()


def test_nan_stays_in_its_row_and_group(ctx):
    c = Case(ctx, [150, 150], 64, 96, "bf16")
    c.run()
    c.ctx.sync()
    y, dw = c.y.clone(), c.dw.clone()
    c.x[20, 5] = float("nan")
    c.torch.cuda.synchronize()
    c.run()
    c.ctx.sync()
    keep = c.torch.arange(300, device="cuda") != 20
    assert c.torch.equal(c.y[keep], y[keep]) and c.torch.isnan(c.y[20]).all()
    assert c.torch.equal(c.dw[1], dw[1]) and c.torch.isnan(c.dw[0, :, 5]).all()
    assert c.torch.equal(c.dw[0, :, :5], dw[0, :, :5]) and c.torch.equal(c.dw[0, :, 6:], dw[0, :, 6:])


def test_gradient_against_differences(ctx):
    """<y, dy> is linear in x, w and bias: differences of any step are the gradients up to the sums' rounding."""
    c = Case(ctx, [60, 90], 40, 24, "f32")
    torch = c.torch
    c.run()
    c.ctx.sync()
    grads = c.dx.clone().double(), c.dw.clone().double(), c.db.clone().double()

    def value():
        torch.cuda.synchronize()
        host.group_matmul(ctx, c.x, c.w, c.offd, c.y, bias=c.bias)
        ctx.sync()
        return float((c.y.double() * c.dy.double()).sum())

    for what, g in zip((c.x, c.w, c.bias), grads):
        keep, v = what.clone(), torch.sign(g).float()
        what.copy_(keep + 0.5 * v)
        up = value()
        what.copy_(keep - 0.5 * v)
        down = value()
        what.copy_(keep)
        assert abs((up - down) - float((g * v.double()).sum())) <= 1e-4 * float(g.abs().sum())


def test_captured_and_replayed_with_other_offsets(ctx):
    """A captured call follows the offsets on the device: rows move between the groups from replay to replay."""
    import torch
    stream = torch.cuda.Stream()
    side = host.Context(0, stream.cuda_stream)
    c = Case(ctx, [2000, 100, 0, 500], 64, 72, "bf16")
    with torch.cuda.stream(stream):
        c.run(side)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            c.run(side)
    for lens in ([2000, 100, 0, 500], [0, 0, 2600, 0], [650, 650, 650, 650]):
        c.off = np.concatenate([[0], np.cumsum(lens)]).astype(np.int64)
        c.offd.copy_(torch.from_numpy(c.off))
        c.x.normal_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in (c.y, c.dx, c.dw, c.db)]
        c.check()
        c.run()
        ctx.sync()
        assert all(torch.equal(a, b) for a, b in zip(got, (c.y, c.dx, c.dw, c.db)))
    side.close()


def test_no_rows(ctx):
    c = Case(ctx, [0, 0, 0], 24, 40, "f16")
    c.run()
    c.check()
    assert (c.dw == 0).all() and (c.db == 0).all()


def test_refusals(ctx):
    c = Case(ctx, [20, 30], 24, 40, "bf16")
    bad = c.torch.zeros((2, 40, 25), dtype=c.torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        host.group_matmul(ctx, c.x, bad, c.offd, c.y)
    with pytest.raises(ValueError):
        host.group_matmul(ctx, c.x, c.w.half(), c.offd, c.y)
    with pytest.raises(ValueError):
        host.group_matmul(ctx, c.x, c.w, c.offd[:2], c.y)
    with pytest.raises(ValueError):
        host.group_matmul(ctx, c.x.t(), c.w, c.offd, c.y)
    with pytest.raises(_capi.SrxError, match="element types"):
        host.group_matmul(ctx, c.x, c.w, c.offd, c.y.half())
    with pytest.raises(ValueError):
        host.group_matmul_dx(ctx, c.dy[:, :39], c.w, c.offd, c.dx)
    with pytest.raises(ValueError):
        host.group_matmul_dw(ctx, c.dy, c.x, c.offd, c.dw, dbias=c.db.half())
    long = Case(ctx, [4000], 24, 40, "bf16")
    with pytest.raises(_capi.SrxError, match="scratch"):
        host.group_matmul_dw(ctx, long.dy, long.x, long.offd, long.dw)
    lib, h, p, o = ctx.lib, ctx.h, c.x.data_ptr(), c.offd.data_ptr()
    ok = [h, 2, 2, p, 24, c.w.data_ptr(), None, o, 2, 50, 24, 40, c.y.data_ptr(), 40]
    for i, v in ((1, 3), (2, 1), (3, None), (4, 23), (5, None), (7, None), (8, -1), (9, -1), (10, 0), (11, 0), (12, None), (13, 39), (10, 1 << 21), (3, p + 1)):
        a = list(ok)
        a[i] = v
        assert lib.srx_group_matmul_dev(*a) == _capi.SRX_ERR_INVALID, (i, v)
    assert lib.srx_group_matmul_dw_scratch_bytes(h, 1, 1, 0, 1) == -1


def _near(torch, got, want, mag, k, dtype):
    """The bound of learned_ref.product and out_bound, on the GPU in 64 bits."""
    err = R.U * (k + 1) * mag
    return bool((torch.abs(got.double() - want) <= err + R.HALF[dtype] * (want.abs() + err) + R.TINY[dtype]).all())


@pytest.mark.parametrize("dtype,pad", [("bf16", 0), ("f16", 5), ("f32", 0), ("bf16", 8)])
def test_many_large_tiles(ctx, dtype, pad):
    """Enough rows and columns for the 256 x 256 tiles (and, with odd strides, the 128 x 128 ones without direct loads): every
    row and weight against the products in 64 bits."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(5)
    lens, K, N = [9000, 0, 300, 20011, 3700], 136, 1032
    off = np.concatenate([[0], np.cumsum(lens)])
    T, E = int(off[-1]), len(lens)

    def rand(r, c):
        return torch.randn((r, c + pad), generator=g, device="cuda").to(_t(dtype))[:, :c]

    x, dy = rand(T, K), rand(T, N)
    w = torch.randn((E, N, K), generator=g, device="cuda").to(_t(dtype))
    y, dx = torch.zeros((T, N), dtype=_t(dtype), device="cuda"), torch.zeros((T, K), dtype=_t(dtype), device="cuda")
    dw, db = torch.zeros_like(w), torch.zeros((E, N), device="cuda")
    offd = torch.from_numpy(off).cuda()
    scratch = torch.full((max(host.group_matmul_dw_scratch_bytes(ctx, E, T, K, N), 16),), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    host.group_matmul(ctx, x, w, offd, y)
    host.group_matmul_dx(ctx, dy, w, offd, dx)
    host.group_matmul_dw(ctx, dy, x, offd, dw, dbias=db, scratch=scratch)
    ctx.sync()
    for e in range(E):
        r = slice(int(off[e]), int(off[e + 1]))
        X, D, W = x[r].double(), dy[r].double(), w[e].double()
        assert _near(torch, y[r], X @ W.t(), X.abs() @ W.abs().t(), K, dtype), ("y", e)
        assert _near(torch, dx[r], D @ W, D.abs() @ W.abs(), N, dtype), ("dx", e)
        assert _near(torch, dw[e], D.t() @ X, D.abs().t() @ X.abs(), lens[e], dtype), ("dw", e)
        assert _near(torch, db[e], D.sum(0), D.abs().sum(0), lens[e], "f32"), ("db", e)


@pytest.mark.parametrize("lens", [[70000, 3, 0, 1], [1] * 500 + [40000]])
def test_groups_of_very_different_sizes(ctx, lens):
    """One group with nearly all rows: the others' dW are right beside it, wherever the shares fall."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(6)
    K, N, T, E = 40, 72, sum(lens), len(lens)
    off = np.concatenate([[0], np.cumsum(lens)])
    x, dy = torch.randn((T, K), generator=g, device="cuda"), torch.randn((T, N), generator=g, device="cuda")
    dw, db = torch.full((E, N, K), 5.0, device="cuda"), torch.full((E, N), 5.0, device="cuda")
    offd = torch.from_numpy(off).cuda()
    scratch = torch.full((max(host.group_matmul_dw_scratch_bytes(ctx, E, T, K, N), 16),), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    host.group_matmul_dw(ctx, dy, x, offd, dw, dbias=db, scratch=scratch)
    ctx.sync()
    for e in range(E):
        D, X = dy[int(off[e]):int(off[e + 1])].double(), x[int(off[e]):int(off[e + 1])].double()
        assert _near(torch, dw[e], D.t() @ X, D.abs().t() @ X.abs(), lens[e], "f32"), e
        assert _near(torch, db[e], D.sum(0), D.abs().sum(0), lens[e], "f32"), e


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("f16", "f16"), ("bf16", "f32")])
@pytest.mark.parametrize("pad", [0, 1, 8])
@pytest.mark.parametrize("lens,K,N", [([2600, 0, 77, 1900], 39, 264), ([2600, 0, 77, 1900], 136, 257), ([9000, 0, 33, 1500, 8000], 40, 41), ([5000, 4], 1, 130)])
def test_more_small_tiles_than_the_chip_holds(ctx, dtype, out, pad, lens, K, N):
    """Sizes whose forward product takes the 128-row tiles, wide and narrow, with and without direct loads."""
    c = Case(ctx, lens, K, N, dtype, out, front=3, behind=70, pad=pad)
    c.run()
    c.check()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens,K,N", [([345], 1370, 1), ([800], 1000, 300), ([100, 0, 501, 3], 2056, 65)])
def test_long_reductions_of_few_tiles(ctx, dtype, lens, K, N):
    c = Case(ctx, lens, K, N, dtype, front=5, behind=9)
    c.run()
    c.check()


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("f16", "f16"), ("bf16", "f32")])
@pytest.mark.parametrize("K,N,pad", [(39, 39, 0), (39, 13, 1), (8, 3, 0), (16, 64, 0), (33, 7, 3), (64, 64, 0), (64, 1, 8), (100, 50, 0), (13, 60, 4), (128, 33, 0)])
def test_small_weights_and_many_rows(ctx, dtype, out, K, N, pad):
    c = Case(ctx, [9000, 0, 1, 129, 10001, 128, 1900], K, N, dtype, out, front=7, behind=200, pad=pad)
    c.run()
    c.check()


def test_misaligned_tables_are_refused(ctx):
    c = Case(ctx, [20, 30], 24, 40, "bf16")
    lib, h = ctx.lib, ctx.h
    x, w, b, o, y, dy, dx, dw, db = (v.data_ptr() for v in (c.x, c.w, c.bias, c.offd, c.y, c.dy, c.dx, c.dw, c.db))
    s = (c.scratch.data_ptr(), c.scratch.numel())
    for bias, off in ((b + 2, o), (b, o + 4)):
        assert lib.srx_group_matmul_dev(h, 2, 2, x, 24, w, bias, off, 2, 50, 24, 40, y, 40) == _capi.SRX_ERR_INVALID
        assert lib.srx_group_matmul_dw_dev(h, 2, 2, dy, 40, x, 24, off, 2, 50, 24, 40, dw, db + bias - b, *s) == _capi.SRX_ERR_INVALID
    assert lib.srx_group_matmul_dx_dev(h, 2, 2, dy, 40, w, o + 4, 2, 50, 24, 40, dx, 24) == _capi.SRX_ERR_INVALID
