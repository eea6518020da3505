"""Forms of the learned layers' kernels that sizes, types and alignment choose: 16-bit rows on whole lines of the recurrence, many rows to a
wave of the quantisation, shares of dW over whole numbers (sums that f32 holds exactly, so that one lost or doubled row shows); and the
memory between rows, which no call touches.  No counterpart in the reference."""
import numpy as np
import pytest

from speechrecognition_amd import host
from tests import learned_ref as R
from tests.test_gpu_group import Case as GroupCase
from tests.test_gpu_scan import Case as ScanCase

pytestmark = pytest.mark.gpu


def _t(dtype):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]


def untouched(*views):
    """What lies around the rows (-7 from the start) is as it was."""
    for v in views:
        around = v._base.clone()
        around.as_strided(v.size(), v.stride(), v.storage_offset()).fill_(-7.0)
        assert bool((around == -7.0).all())


@pytest.mark.parametrize("max_frames", [0, 1])             # cut into pieces, and whole
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D,pad", [(128, 0), (192, 0), (128, 64), (100, 28)])
@pytest.mark.parametrize("lens,front,behind", [([700, 0, 33, 1, 16, 255], 0, 0), ([513, 64, 0], 5, 40)])
def test_16_bit_rows_on_whole_lines(ctx, lens, front, behind, D, pad, dtype, sigmoid, max_frames):
    """Row strides of 64 elements, addresses of 128 bytes, more than 64 channels: pairs of channels, past the caches."""
    c = ScanCase(ctx, lens, D, dtype, sigmoid, front=front, behind=behind, pad=pad, max_frames=max_frames)
    assert all(v.data_ptr() % 128 == 0 and v.stride(0) % 64 == 0 for v in (c.g, c.x, c.dh, c.h, c.dg, c.dx))
    assert (host.gated_scan_scratch_bytes(ctx, c.n, c.T, max_frames, D) > 0) == (max_frames == 0)
    c.run()
    c.check()
    untouched(c.g, c.x, c.dh, c.h, c.dg, c.dx)


@pytest.mark.parametrize("dtype,D,pad,shift", [("f32", 66, 1, 3), ("f32", 20, 3, 0), ("f32", 96, 32, 0), ("f16", 66, 2, 2), ("bf16", 39, 2, 1), ("bf16", 130, 6, 0)])
@pytest.mark.parametrize("max_frames", [0, 1])
def test_recurrence_between_rows(ctx, dtype, D, pad, shift, max_frames):
    c = ScanCase(ctx, [300, 0, 17, 64], D, dtype, True, front=2, behind=3, pad=pad, shift=shift, max_frames=max_frames)
    c.run()
    c.check()
    untouched(c.g, c.x, c.dh, c.h, c.dg, c.dx)


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("f16", "f16"), ("bf16", "f32")])
@pytest.mark.parametrize("lens,K,N,pad,shift", [([2600, 0, 77, 1900], 39, 39, 1, 0), ([2600, 0, 77, 1900], 136, 264, 8, 8), ([2600, 0, 77, 1900], 136, 264, 3, 1),
                                                ([9, 0, 20], 100, 130, 5, 3), ([900, 40], 2, 130, 6, 1), ([6000, 0, 5000], 64, 1032, 8, 0)])
def test_products_between_rows(ctx, dtype, out, lens, K, N, pad, shift):
    c = GroupCase(ctx, lens, K, N, dtype, out, front=3, behind=70, pad=pad, shift=shift)
    c.run()
    c.check()
    untouched(c.x, c.dy, c.y, c.dx)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("more", [1, 3, 7])
@pytest.mark.parametrize("runs", [1, 2, 4, 8])
def test_codes_of_many_rows(ctx, dtype, more, runs):
    """From 16,384 rows on a wave takes 8, 4 or 2 of them; the last wave has fewer."""
    import torch
    rows, K = 16384 + more, runs * (256 if dtype == "f32" else 512) - 5
    k16 = (K + 15) // 16 * 16
    g = torch.Generator(device="cuda").manual_seed(rows + K)
    x = torch.randn((rows, K), generator=g, device="cuda") * torch.exp(torch.empty((rows, 1), device="cuda").uniform_(-5, 5, generator=g))
    x[5] = 0
    x[rows - 1, ::2] = 0
    x = x.to(_t(dtype))
    x[7, 3] = float("nan")
    x[rows - 2, K - 1] = float("inf")
    q, s = torch.full((rows + 1, k16), 77, dtype=torch.int8, device="cuda"), torch.full((rows + 1,), 5.0, device="cuda")
    torch.cuda.synchronize()
    host.quantize_rows(ctx, x, q[:rows], s[:rows])
    ctx.sync()
    v = x.float().cpu().numpy()
    with np.errstate(invalid="ignore"):
        ws, wq = R.quantize(v)
    got, gs = q.cpu().numpy(), s.cpu().numpy()
    ok = ~np.isnan(ws)
    assert gs[:rows][ok].tobytes() == ws[ok].tobytes() and np.isnan(gs[:rows][~ok]).all() and (~ok).sum() == 1 and gs[rows] == 5
    assert (got[:rows, :K] == wq).all() and (got[:rows, K:] == 0).all() and (got[rows] == 77).all()


@pytest.mark.parametrize("lens", [[70000, 3, 0, 1], [1] * 500 + [40000], [40000, 0, 5, 3000, 9001]])
@pytest.mark.parametrize("dtype,out,K,N,pad", [("f32", "f32", 40, 72, 0), ("f32", "f32", 41, 39, 1), ("f32", "f32", 1, 130, 0), ("f16", "f32", 512, 512, 0), ("bf16", "f32", 512, 512, 8),
                                               ("bf16", "bf16", 512, 256, 0), ("f16", "f32", 136, 200, 0), ("bf16", "f32", 129, 130, 3)])
def test_gradients_of_weights_over_whole_numbers(ctx, lens, dtype, out, K, N, pad):
    """Factors from -2 to 2: every sum is a whole number below 2^24, so dW and db are exact wherever the shares fall."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(len(lens) + K)
    T, E = sum(lens), len(lens)
    assert 4 * max(lens) < 1 << 24
    off = np.concatenate([[0], np.cumsum(lens)])
    x, dy = (torch.randint(-2, 3, (T, c + pad), generator=g, device="cuda").to(_t(dtype))[:, :c] for c in (K, N))
    dw, db = torch.full((E, N, K), 5.0, dtype=_t(out), device="cuda"), torch.full((E, N), 5.0, device="cuda")
    offd = torch.from_numpy(off).cuda()
    scratch = torch.full((max(host.group_matmul_dw_scratch_bytes(ctx, E, T, K, N), 16),), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    host.group_matmul_dw(ctx, dy, x, offd, dw, dbias=db, scratch=scratch)
    ctx.sync()
    big = [e for e in range(E) if lens[e] > 1]
    for e in big + [e for e in range(E) if lens[e] <= 1][::37]:
        D, X = dy[int(off[e]):int(off[e + 1])].double(), x[int(off[e]):int(off[e + 1])].double()
        want = D.t().contiguous() @ X
        assert torch.equal(dw[e], want.to(_t(out))), e
        assert torch.equal(db[e].double(), D.sum(0)), e


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lens,K,N", [([9000, 0, 300, 20011, 3700], 136, 1032), ([4097], 1024, 1024)])
def test_large_tiles_over_whole_numbers(ctx, dtype, lens, K, N):
    """The forward product and dx in 256 x 256 tiles, with the bias, as exact sums in f32."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(K)
    T, E = sum(lens), len(lens)
    off = np.concatenate([[0], np.cumsum(lens)])
    x, dy, w = (torch.randint(-2, 3, s, generator=g, device="cuda").to(_t(dtype)) for s in ((T, K), (T, N), (E, N, K)))
    bias = torch.randint(-9, 10, (E, N), generator=g, device="cuda").float()
    y, dx = torch.full((T, N), 0.5, device="cuda"), torch.full((T, K), 0.5, device="cuda")
    offd = torch.from_numpy(off).cuda()
    torch.cuda.synchronize()
    host.group_matmul(ctx, x, w, offd, y, bias=bias)
    host.group_matmul_dx(ctx, dy, w, offd, dx)
    ctx.sync()
    for e in range(E):
        r = slice(int(off[e]), int(off[e + 1]))
        W = w[e].double()
        assert torch.equal(y[r].double(), x[r].double() @ W.t().contiguous() + bias[e].double()), e
        assert torch.equal(dx[r].double(), dy[r].double() @ W), e
