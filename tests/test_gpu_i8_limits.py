"""Ends of the 8-bit layer's ranges: the largest sums that codes can make, and the most rows that a launch takes.  No counterpart in
the reference."""
import pytest

from speechrecognition_amd import _capi, host

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("by_state", [False, True])
@pytest.mark.parametrize("rows,N", [(2, 33), (520, 1100), (4096, 4096)])
def test_largest_sums_of_any_codes(ctx, rows, N, by_state, out):
    """K at its limit with codes of -128: 2^31, which 32 bits do not hold, beside the sums next to it.  The row counts take the three
    tiles.  Results are powers of two times 127 or 128 at most: exact in every type."""
    import torch
    K = _capi.SRX_I8_MAX_K
    xq, wq = (torch.full((n, K), -128, dtype=torch.int8, device="cuda") for n in (rows, N))
    xq[1::5] = 127                                    # 127 * -128 * K
    wq[2::7, ::2] = 0                                 # half of the sum
    one = torch.ones(max(rows, N), device="cuda")
    y = torch.zeros((N, rows) if by_state else (rows, N), dtype={"f32": torch.float32, "bf16": torch.bfloat16}[out], device="cuda")
    torch.cuda.synchronize()
    host.matmul_i8(ctx, xq, one[:rows], wq, one[:N], K, y, by_state=by_state)
    ctx.sync()
    a = torch.full((rows,), 128.0, dtype=torch.float64, device="cuda")
    a[1::5] = -127.0
    b = torch.full((N,), 128.0 * K, dtype=torch.float64, device="cuda")
    b[2::7] /= 2
    want = a[:, None] * b
    assert float(want.max()) == 2.0 ** 31
    assert torch.equal((y.t() if by_state else y).double(), want)
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype,z", [(_capi.SRX_F32, 4), (_capi.SRX_F16, 2), (_capi.SRX_BF16, 2)])
def test_more_rows_than_a_launch_takes_are_refused(ctx, dtype, z):
    """A wave to a row, four to a workgroup: refused before anything is read, the addresses are those of a small buffer."""
    import torch
    p = torch.zeros(4096, device="cuda").data_ptr()
    for K in (4096 // z + 1, 8192 // z, 8192 // z + 1):
        for rows in ((1 << 26) - 3, (1 << 26) - 1, 1 << 26):
            assert ctx.lib.srx_quantize_rows_dev(ctx.h, dtype, p, 1 << 20, rows, K, p, 1 << 20, p) == _capi.SRX_ERR_INVALID, (rows, K)
    ctx.sync()


def test_most_rows_that_a_launch_takes(ctx):
    """2^26 - 1 rows of one element: the codes are signs times 127."""
    import torch
    rows = (1 << 26) - 1
    x = torch.empty((rows, 1), device="cuda").normal_()
    q, s = torch.full((rows, 16), 7, dtype=torch.int8, device="cuda"), torch.zeros(rows, device="cuda")
    torch.cuda.synchronize()
    host.quantize_rows(ctx, x, q, s)
    ctx.sync()
    assert torch.equal(q[:, 0].float(), 127 * torch.sign(x[:, 0])) and not q[:, 1:].any() and torch.equal(s, x[:, 0].abs() / torch.full((1,), 127.0, device="cuda"))
    del x, q, s
    torch.cuda.empty_cache()
