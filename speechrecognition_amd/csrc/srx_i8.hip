// 8-bit matrix product with a scale for each row and each output, and the quantisation that makes its operands:
//
//   s_r = max_k |x_rk| / 127,  q_rk = round(x_rk / s_r) to the nearest whole number, ties to even   (s_r = 0: all codes 0)
//   y_rn = s_r s_n sum_k q_rk q_nk + b_n
//
// The sum is exact in 32 bits (K <= SRX_I8_MAX_K), so the only roundings are the scale's, the codes' and the output's few.
#include "srx_tile.h"

struct QuantArgs {
    const void *x;
    int64_t ld_x, rows, ld_q;
    int K;
    int8_t *q;
    float *scale;
};

// One wave per row: the maximum in a first sweep, the codes in a second that finds the row in cache.  HBM-bound.
template <class T>
__global__ __launch_bounds__(256) void k_quantize_rows(QuantArgs p) {
    const int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (row >= p.rows) return;
    const int lane = threadIdx.x & 63;
    const T *x = reinterpret_cast<const T *>(p.x) + row * p.ld_x;
    float m = 0.0f;
    for (int k = lane; k < p.K; k += 64) {
        const float v = fabsf(srx_to_f32<T>(x[k]));
        m = v > m || v != v ? v : m;   // a NaN stays
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const float v = __shfl_xor(m, o);
        m = v > m || v != v ? v : m;
    }
    const float s = m / 127.0f;
    if (lane == 0) p.scale[row] = s;
    const bool live = s > 0.0f && s < __builtin_huge_valf();
    int8_t *q = p.q + row * p.ld_q;
    const int end = (p.K + 15) / 16 * 16;   // zeros up to whole 16 bytes: the product reads them
    for (int k = lane; k < end; k += 64) {
        int c = 0;
        if (live && k < p.K) {
            const float r = rintf(srx_to_f32<T>(x[k]) / s);
            c = (int)(r > 127.0f ? 127.0f : r < -127.0f ? -127.0f : r);
        }
        q[k] = (int8_t)c;
    }
}

struct I8Args {
    const int8_t *p, *q;        // operands: i the output's adjacent index, j the other
    int64_t ld_p, ld_q;
    const float *sp, *sq, *bias;
    bool bias_i;                // bias by i (else by j)
    int64_t I, J;
    int K;
    void *y;
    int64_t ld_y;
    int64_t tiles_i, tiles_j;
};

template <class O, int WI, int WJ, int FI, int FJ>
__global__ __launch_bounds__(WI *WJ * 64) void k_matmul_i8(I8Args p) {
    typedef Tile<int8_t, WI, WJ, FI, FJ, false, false, true> T;
    __shared__ __attribute__((aligned(1024))) unsigned char smem[T::LDS];
    int64_t i0, j0;
    tile_of(blockIdx.x, p.tiles_i, p.tiles_j, i0, j0);
    i0 *= T::TI;
    j0 *= T::TJ;
    TileOperand P{p.p + i0 * p.ld_p, p.ld_p, (int)(p.I - i0 < T::TI ? p.I - i0 : T::TI)};
    TileOperand Q{p.q + j0 * p.ld_q, p.ld_q, (int)(p.J - j0 < T::TJ ? p.J - j0 : T::TJ)};
    typename T::acc_t acc[FI][FJ];
    float none[FJ];
    T::template product<false>(smem, P, Q, (p.K + 15) / 16 * 16, acc, none, false);
    O *y = reinterpret_cast<O *>(p.y);
    struct Held { float s[RUN<O>], b[RUN<O>]; };
    T::template write_out<RUN<O>>(
        smem, acc,
        [&](int i) {
            Held h;
#pragma unroll
            for (int e = 0; e < RUN<O>; e++) {
                h.s[e] = i + e < P.n ? p.sp[i0 + i + e] : 0.0f;
                h.b[e] = p.bias && p.bias_i && i + e < P.n ? p.bias[i0 + i + e] : 0.0f;
            }
            return h;
        },
        [&](int i, int j, const float (&v)[RUN<O>], const Held &h) {
            if (j >= Q.n || i >= P.n) return;
            const float sj = p.sq[j0 + j], bj = p.bias && !p.bias_i ? p.bias[j0 + j] : 0.0f;
            float f[RUN<O>];
#pragma unroll
            for (int e = 0; e < RUN<O>; e++) f[e] = __builtin_fmaf(v[e] * sj, h.s[e], p.bias_i ? h.b[e] : bj);
            store_run<O>(y + (j0 + j) * p.ld_y + i0 + i, f, P.n - i);
        });
}

// Few rows: tiles of 32 x 32
template <class O>
__global__ __launch_bounds__(THIN_WAVES * 64) void k_matmul_i8_thin(I8Args p) {
    __shared__ __attribute__((aligned(16))) unsigned char smem[THIN_LDS];
    const int64_t i0 = (blockIdx.x % p.tiles_i) * 32, j0 = (blockIdx.x / p.tiles_i) * 32;
    const TileOperand P{p.p + i0 * p.ld_p, p.ld_p, (int)(p.I - i0 < 32 ? p.I - i0 : 32)};
    const TileOperand Q{p.q + j0 * p.ld_q, p.ld_q, (int)(p.J - j0 < 32 ? p.J - j0 : 32)};
    O *y = reinterpret_cast<O *>(p.y);
    thin_product<int8_t>(smem, P, Q, (p.K + 15) / 16 * 16, [&](int i, int j, const float (&v)[4]) {
        if (j >= Q.n || i >= P.n) return;
        const float sj = p.sq[j0 + j], bj = p.bias && !p.bias_i ? p.bias[j0 + j] : 0.0f;
        float f[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const bool in = i + e < P.n;
            f[e] = __builtin_fmaf(v[e] * sj, in ? p.sp[i0 + i + e] : 0.0f, p.bias && p.bias_i && in ? p.bias[i0 + i + e] : bj);
        }
        store_four<O>(y + (j0 + j) * p.ld_y + i0 + i, f, P.n - i);
    });
}

// ------------------------------------------------------------------------------------------------ host side
static constexpr int64_t I8_MAX_ROWS = 1ll << 40;

extern "C" int srx_quantize_rows_dev(srx_ctx *ctx, int dtype, const void *x_dev, int64_t ld_x, int64_t rows, int K, int8_t *q_dev, int64_t ld_q, float *scale_dev) {
    const char *name = "srx_quantize_rows_dev";
    SRX_ENTER(ctx, name);
    SRX_REQUIRE(ctx, srx_dtype_size(dtype) != 0, "%s: element type %d", name, dtype);
    SRX_REQUIRE(ctx, rows >= 0 && rows < (1ll << 33) && K >= 1 && K <= SRX_I8_MAX_K, "%s: %lld rows of %d (at most %d)", name, (long long)rows, K, SRX_I8_MAX_K);
    if (rows == 0) return SRX_OK;
    SRX_REQUIRE(ctx, x_dev && q_dev && scale_dev, "%s: null argument", name);
    SRX_REQUIRE(ctx, ld_x >= K && ld_q >= (K + 15) / 16 * 16 && ld_q % 16 == 0 && srx_aligned(q_dev, 16),
                "%s: row strides %lld / %lld for %d columns (codes: whole 16 bytes, 16-byte aligned)", name, (long long)ld_x, (long long)ld_q, K);
    SRX_REQUIRE(ctx, srx_aligned(x_dev, srx_dtype_size(dtype)) && srx_aligned(scale_dev, 4), "%s: misaligned buffer", name);
    const QuantArgs p{x_dev, ld_x, rows, ld_q, K, q_dev, scale_dev};
    const dim3 g((unsigned)ceil_div64(rows, 4)), b(256);
    {
        SrxProf prof_(ctx, "k_quantize_rows");
        if (dtype == SRX_F32) hipLaunchKernelGGL(k_quantize_rows<float>, g, b, 0, ctx->stream, p);
        else if (dtype == SRX_F16) hipLaunchKernelGGL(k_quantize_rows<srx_f16>, g, b, 0, ctx->stream, p);
        else hipLaunchKernelGGL(k_quantize_rows<srx_bf16>, g, b, 0, ctx->stream, p);
    }
    SRX_LAUNCH_CHECK(ctx);
    return SRX_OK;
}

// Rows up to which the product is bound by reading the weights once
static constexpr int64_t I8_THIN_ROWS = 64;

template <class O, int WI, int WJ, int FI, int FJ>
static int i8_tile(srx_ctx *ctx, const char *name, I8Args &p) {
    typedef Tile<int8_t, WI, WJ, FI, FJ, false, false, true> T;
    p.tiles_i = ceil_div64(p.I, T::TI);
    p.tiles_j = ceil_div64(p.J, T::TJ);
    SRX_REQUIRE(ctx, p.tiles_i * p.tiles_j < (1ll << 31), "%s: too many tiles", name);
    SrxProf prof_(ctx, "k_matmul_i8");
    hipLaunchKernelGGL((k_matmul_i8<O, WI, WJ, FI, FJ>), dim3((unsigned)(p.tiles_i * p.tiles_j)), dim3(T::NT), 0, ctx->stream, p);
    return SRX_OK;
}

template <class O>
static int i8_launch(srx_ctx *ctx, const char *name, I8Args &p, int64_t rows) {
    if (rows <= I8_THIN_ROWS) {
        p.tiles_i = ceil_div64(p.I, 32);
        p.tiles_j = ceil_div64(p.J, 32);
        SrxProf prof_(ctx, "k_matmul_i8_thin");
        hipLaunchKernelGGL((k_matmul_i8_thin<O>), dim3((unsigned)(p.tiles_i * p.tiles_j)), dim3(THIN_WAVES * 64), 0, ctx->stream, p);
        return SRX_OK;
    }
    if (tile_large(ceil_div64(p.I, 256) * ceil_div64(p.J, 256), ceil_div64(p.I, 128) * ceil_div64(p.J, 128), ctx->num_cus))
        return i8_tile<O, 4, 2, 2, 4>(ctx, name, p);
    return i8_tile<O, 2, 2, 2, 2>(ctx, name, p);
}

extern "C" int srx_matmul_i8_dev(srx_ctx *ctx, int out_dtype, const int8_t *xq_dev, int64_t ld_xq, const float *xs_dev, const int8_t *wq_dev, int64_t ld_wq,
                                 const float *ws_dev, const float *bias_dev, int64_t rows, int N, int K, void *y_dev, int64_t stride_r, int64_t stride_n) {
    const char *name = "srx_matmul_i8_dev";
    SRX_ENTER(ctx, name);
    SRX_REQUIRE(ctx, srx_dtype_size(out_dtype) != 0, "%s: element type %d", name, out_dtype);
    SRX_REQUIRE(ctx, rows >= 0 && rows <= I8_MAX_ROWS && N >= 1 && N <= (1 << 24) && K >= 1 && K <= SRX_I8_MAX_K, "%s: %lld x %d x %d (K at most %d)", name,
                (long long)rows, N, K, SRX_I8_MAX_K);
    if (rows == 0) return SRX_OK;
    SRX_REQUIRE(ctx, xq_dev && xs_dev && wq_dev && ws_dev && y_dev, "%s: null argument", name);
    const int k16 = (K + 15) / 16 * 16;
    SRX_REQUIRE(ctx, ld_xq >= k16 && ld_wq >= k16 && ld_xq % 16 == 0 && ld_wq % 16 == 0 && ld_xq <= (1 << 22) && ld_wq <= (1 << 22) && srx_aligned(xq_dev, 16) && srx_aligned(wq_dev, 16),
                "%s: code rows of %lld / %lld bytes for K = %d (whole 16 bytes, 16-byte aligned, at most 4 MiB)", name, (long long)ld_xq, (long long)ld_wq, K);
    SRX_REQUIRE(ctx, (stride_n == 1 && stride_r >= N) || (stride_r == 1 && stride_n >= rows), "%s: output strides %lld, %lld (one of them 1)", name, (long long)stride_r,
                (long long)stride_n);
    SRX_REQUIRE(ctx, srx_aligned(y_dev, srx_dtype_size(out_dtype)), "%s: misaligned buffer", name);
    I8Args p{};
    p.K = K;
    p.bias = bias_dev;
    p.y = y_dev;
    if (stride_n == 1) {   // i = output, j = row
        p.p = wq_dev; p.ld_p = ld_wq; p.sp = ws_dev; p.I = N; p.bias_i = true;
        p.q = xq_dev; p.ld_q = ld_xq; p.sq = xs_dev; p.J = rows;
        p.ld_y = stride_r;
    } else {
        p.p = xq_dev; p.ld_p = ld_xq; p.sp = xs_dev; p.I = rows; p.bias_i = false;
        p.q = wq_dev; p.ld_q = ld_wq; p.sq = ws_dev; p.J = N;
        p.ld_y = stride_n;
    }
    int rc = out_dtype == SRX_F32 ? i8_launch<float>(ctx, name, p, rows) : out_dtype == SRX_F16 ? i8_launch<srx_f16>(ctx, name, p, rows) : i8_launch<srx_bf16>(ctx, name, p, rows);
    if (rc != SRX_OK) return rc;
    SRX_LAUNCH_CHECK(ctx);
    return SRX_OK;
}
