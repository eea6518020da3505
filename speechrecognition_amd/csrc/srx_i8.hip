// 8-bit matrix product with a scale for each row and each output, and the quantisation that makes its operands:
//
//   s_r = max_k |x_rk| / 127,  q_rk = round(x_rk / s_r) to the nearest whole number, ties to even   (s_r = 0: all codes 0)
//   y_rn = s_r s_n sum_k q_rk q_nk + b_n
//
// The sum is exact in 32 bits (K <= SRX_I8_MAX_K, see full_sum), so the only roundings are the scale's, the codes' and the output's few.
#include "srx_tile.h"

struct QuantArgs {
    const void *x;
    int64_t ld_x, rows, ld_q;
    int K;
    int8_t *q;
    float *scale;
};

// A code is x / s rounded to a whole number, ties to even.  x times the hardware's reciprocal of s lies within 127 * 2^-22 = 3e-5
// of the f32 quotient, so both round alike unless the product is nearly a half: only a run that holds such a value (one code in
// 5,000) forms the quotients.  A division costs about ten instructions, and there is one per element.
__device__ __forceinline__ int code_exact(float x, float s) {
    const float c = rintf(x / s);
    return (int)(c > 127.0f ? 127.0f : c < -127.0f ? -127.0f : c);   // (only a scale below the normal range can leave the range)
}

// |x| as a whole number that orders as it does, NaN above infinity above all others; two of a 16-bit type at a time
template <class T>
struct Magnitude {
    static constexpr int N = 16 / 4;
    typedef uint16_t two __attribute__((ext_vector_type(2)));
    typedef std::conditional_t<sizeof(T) == 4, uint32_t, two> part;
    part m;
    __device__ __forceinline__ void start() { m = {}; }
    template <class R>
    __device__ __forceinline__ void take(const R &run) {
        part p[N];
        __builtin_memcpy(p, &run, 16);
#pragma unroll
        for (int i = 0; i < N; i++) {
            if constexpr (sizeof(T) == 4) m = max(m, p[i] & 0x7fffffffu);
            else m = __builtin_elementwise_max(m, p[i] & (uint16_t)0x7fff);
        }
    }
    __device__ __forceinline__ float of_wave() const {   // the largest of all lanes
        uint32_t v;
        if constexpr (sizeof(T) == 4) v = m; else v = m.x > m.y ? m.x : m.y;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o));
        if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, v);
        else return srx_to_f32<T>(__builtin_bit_cast(T, (uint16_t)v));
    }
};

// A wave takes R rows, each in NV runs of 16 bytes per lane, and reads them once; NV = 0: one row of any length, its maximum in a
// first sweep and the codes in a second.  131,072 x 1,024 bf16: 95 us, 403 MB, 4.2 TB/s.  HBM-bound: 3 bytes per element of a 16-bit type; several short rows per wave because
// one row's loads (2 KB at 1,024 columns) do not cover their latency.
template <class T, int NV, int R>
__global__ __launch_bounds__(256) void k_quantize_rows(QuantArgs p) {
    const int64_t row0 = ((int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * R;
    if (row0 >= p.rows) return;
    const int lane = threadIdx.x & 63;
    constexpr int V = RUN<T>;
    const int end = (p.K + 15) / 16 * 16;   // zeros up to whole 16 bytes: the product reads them
    typedef typename SrxVec<T, V>::type run;
    auto load = [&](int64_t row, int k) {
        const T *x = reinterpret_cast<const T *>(p.x) + row * p.ld_x;
        run v;
        if (k + V <= p.K) __builtin_memcpy(&v, x + k, 16);
        else
#pragma unroll
            for (int e = 0; e < V; e++) v[e] = k + e < p.K ? x[k + e] : (T)0;
        return v;
    };
    struct Scale { float s, rs; bool live, fast; };
    auto scale = [&](int64_t row, float m) {
        const float s = m / 127.0f;
        if (lane == 0) p.scale[row] = s;
        const float rs = __builtin_amdgcn_rcpf(s);   // infinite for a subnormal s: its codes all take the division
        return Scale{s, rs, s > 0.0f && s < __builtin_huge_valf(), rs < __builtin_huge_valf()};
    };
    auto store = [&](int64_t row, int k, const run &v, const Scale &f) {
        if (k >= end) return;
        constexpr float whole = 12582912.0f;   // 3 * 2^22: added, it leaves the nearest whole number in the low bits
        uint32_t c[V];
        float off = 0.0f;
#pragma unroll
        for (int e = 0; e < V; e++) {
            const float x = srx_to_f32<T>(v[e]), t = __builtin_fmaf(x, f.rs, whole);
            off = fmaxf(off, fabsf(__builtin_fmaf(x, f.rs, whole - t)));
            c[e] = __builtin_bit_cast(uint32_t, t);
        }
        if (!f.live || !f.fast || off > 0.4999f) {
#pragma unroll
            for (int e = 0; e < V; e++) c[e] = f.live ? (uint32_t)code_exact(srx_to_f32<T>(v[e]), f.s) : 0u;
        }
        uint32_t w[V / 4];
#pragma unroll
        for (int e = 0; e < V / 4; e++)
            w[e] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[4 * e + 3], c[4 * e + 2], 0x0c0c0400u),
                                         __builtin_amdgcn_perm(c[4 * e + 1], c[4 * e], 0x0c0c0400u), 0x05040100u);
        __builtin_memcpy(p.q + row * p.ld_q + k, w, V);   // (end is a multiple of V)
    };
    if constexpr (NV > 0) {
        run held[R][NV];
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int i = 0; i < NV; i++) held[r][i] = load(row0 + r < p.rows ? row0 + r : p.rows - 1, (i * 64 + lane) * V);
#pragma unroll
        for (int r = 0; r < R; r++) {
            if (row0 + r >= p.rows) return;
            Magnitude<T> m;
            m.start();
#pragma unroll
            for (int i = 0; i < NV; i++) m.take(held[r][i]);
            const Scale f = scale(row0 + r, m.of_wave());
#pragma unroll
            for (int i = 0; i < NV; i++) store(row0 + r, (i * 64 + lane) * V, held[r][i], f);
        }
    } else {
        Magnitude<T> m;
        m.start();
        for (int k = lane * V; k < p.K; k += 64 * V) m.take(load(row0, k));
        const Scale f = scale(row0, m.of_wave());
        for (int k = lane * V; k < end; k += 64 * V) store(row0, k, load(row0, k), f);
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

// Sums lie in (-2^31, 2^31], since a product of two codes lies in [-127 * 128, 128 * 128] and there are at most 2^17 of them.  The one
// that 32 bits do not hold, 2^31, needs all of the 2^17 products at their largest, and comes out as -2^31, which no other sum is.
static_assert(SRX_I8_MAX_K == 1 << 17, "full_sum");
__device__ __forceinline__ void full_sum(int K, float (&v)[4]) {
    if (K < SRX_I8_MAX_K) return;   // (the same for all lanes)
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = v[e] == -0x1p31f ? 0x1p31f : v[e];
}

struct ScaleBias { float s, b; };
__device__ __forceinline__ ScaleBias from_lane(const ScaleBias &v, int l) { return {__shfl(v.s, l), __shfl(v.b, l)}; }

// Scales and bias on a tile's way out.  131,072 x 1,024 -> 2,000 f32: 440 to 470 us; the outputs alone (1,049 MB) are 152 us at the rate of a
// fill, the products 255 us at the library's best rate, and within a CU one follows the other.  The sum alone runs at 2,400 TOP/s (time per
// further K).
template <class O, int WI, int WJ, int FI, int FJ>
__global__ __launch_bounds__(WI *WJ * 64, 2) void k_matmul_i8(I8Args p) {
    typedef Tile<int8_t, WI, WJ, FI, FJ, false, false, TO_LDS> T;
    __shared__ __attribute__((aligned(1024))) unsigned char smem[T::LDS];
    struct Held { ScaleBias i[RUN<O>], j[FJ]; };
    int64_t i0, j0;
    tile_of(blockIdx.x, p.tiles_i, p.tiles_j, i0, j0);
    i0 *= T::TI;
    j0 *= T::TJ;
    const TileOperand P{p.p + i0 * p.ld_p, p.ld_p, (int)(p.I - i0 < T::TI ? p.I - i0 : T::TI), 0};
    const TileOperand Q{p.q + j0 * p.ld_q, p.ld_q, (int)(p.J - j0 < T::TJ ? p.J - j0 : T::TJ), 0};
    Held held;
    const int i = T::template lane_i<O>();
#pragma unroll
    for (int e = 0; e < RUN<O>; e++) held.i[e] = {i + e < P.n ? p.sp[i0 + i + e] : 0.0f, p.bias && p.bias_i && i + e < P.n ? p.bias[i0 + i + e] : 0.0f};
#pragma unroll
    for (int c = 0; c < FJ; c++) {
        const int j = T::lane_j(c);
        held.j[c] = {j < Q.n ? p.sq[j0 + j] : 0.0f, p.bias && !p.bias_i && j < Q.n ? p.bias[j0 + j] : 0.0f};
    }
    typename T::acc_t acc[FI][FJ];
    float none[FJ];
    T::template product<false>(smem, P, Q, (p.K + 15) / 16 * 16, acc, none, false);
    T::template write_out<O>(
        smem, acc, held,
        [&](const float (&sum)[4], const ScaleBias &j, f32x4_t &r) {
            float v[4] = {sum[0], sum[1], sum[2], sum[3]};
            full_sum(p.K, v);
            r = {v[0] * j.s, v[1] * j.s, v[2] * j.s, v[3] * j.s};
        },
        [&](const float (&v)[RUN<O>], const ScaleBias (&i)[RUN<O>], auto &&j, float (&r)[RUN<O>]) {
#pragma unroll
            for (int e = 0; e < RUN<O>; e++) r[e] = __builtin_fmaf(v[e], i[e].s, i[e].b);
            if (!p.bias_i) {
                const float b = j().b;
#pragma unroll
                for (int e = 0; e < RUN<O>; e++) r[e] += b;
            }
        },
        TileOut<O, T::TI>(reinterpret_cast<O *>(p.y) + j0 * p.ld_y + i0, p.ld_y, P.n, Q.n, P.n == T::TI && Q.n == T::TJ));
}

// Few rows: tiles of 32 x 32
template <class O>
__global__ __launch_bounds__(THIN_WAVES * 64) void k_matmul_i8_thin(I8Args p) {
    __shared__ __attribute__((aligned(16))) unsigned char smem[THIN_LDS];
    const int64_t i0 = (blockIdx.x % p.tiles_i) * 32, j0 = (blockIdx.x / p.tiles_i) * 32;
    const TileOperand P{p.p + i0 * p.ld_p, p.ld_p, (int)(p.I - i0 < 32 ? p.I - i0 : 32), 0};
    const TileOperand Q{p.q + j0 * p.ld_q, p.ld_q, (int)(p.J - j0 < 32 ? p.J - j0 : 32), 0};
    O *y = reinterpret_cast<O *>(p.y);
    thin_product<int8_t>(smem, P, Q, (p.K + 15) / 16 * 16, [&](int i, int j, const float (&sum)[4]) {
        if (j >= Q.n || i >= P.n) return;
        float v[4] = {sum[0], sum[1], sum[2], sum[3]};
        full_sum(p.K, v);
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
static constexpr int64_t I8_MAX_ROWS = 1ll << 40, QUANT_MAX_ROWS = 1ll << 26;

// Several rows to a wave from this many rows on: fewer are better spread over the chip, one to a wave
static constexpr int64_t QUANT_MANY = 16384;

template <class T, int NV, int R>
static int quant_rows(srx_ctx *ctx, const char *name, const QuantArgs &p) {
    const int64_t blocks = ceil_div64(p.rows, 4 * R);
    SRX_REQUIRE(ctx, srx_grid_fits(blocks, 256), "%s: %lld rows of %d: no launch holds one wave to each", name, (long long)p.rows, p.K);
    SrxProf prof_(ctx, "k_quantize_rows");
    hipLaunchKernelGGL((k_quantize_rows<T, NV, R>), dim3((unsigned)blocks), dim3(256), 0, ctx->stream, p);
    return SRX_OK;
}
template <class T>
static int quant_launch(srx_ctx *ctx, const char *name, const QuantArgs &p) {
    const int runs = (int)ceil_div64(p.K, 64 * RUN<T>);
    const bool many = p.rows >= QUANT_MANY;
    if (runs == 1) return many ? quant_rows<T, 1, 8>(ctx, name, p) : quant_rows<T, 1, 1>(ctx, name, p);
    if (runs == 2) return many ? quant_rows<T, 2, 4>(ctx, name, p) : quant_rows<T, 2, 1>(ctx, name, p);
    if (runs <= 4) return many ? quant_rows<T, 4, 2>(ctx, name, p) : quant_rows<T, 4, 1>(ctx, name, p);
    if (runs <= 8) return quant_rows<T, 8, 1>(ctx, name, p);
    return quant_rows<T, 0, 1>(ctx, name, p);
}

extern "C" int srx_quantize_rows_dev(srx_ctx *ctx, int dtype, const void *x_dev, int64_t ld_x, int64_t rows, int K, int8_t *q_dev, int64_t ld_q, float *scale_dev) {
    const char *name = "srx_quantize_rows_dev";
    SRX_ENTER(ctx, name);
    SRX_REQUIRE(ctx, srx_dtype_size(dtype) != 0, "%s: element type %d", name, dtype);
    SRX_REQUIRE(ctx, rows >= 0 && rows < QUANT_MAX_ROWS && K >= 1 && K <= SRX_I8_MAX_K, "%s: %lld rows of %d (less than %lld of at most %d)", name, (long long)rows, K, (long long)QUANT_MAX_ROWS,
                SRX_I8_MAX_K);
    if (rows == 0) return SRX_OK;
    SRX_REQUIRE(ctx, x_dev && q_dev && scale_dev, "%s: null argument", name);
    SRX_REQUIRE(ctx, ld_x >= K && ld_q >= (K + 15) / 16 * 16 && ld_q % 16 == 0 && srx_aligned(q_dev, 16),
                "%s: row strides %lld / %lld for %d columns (codes: whole 16 bytes, 16-byte aligned)", name, (long long)ld_x, (long long)ld_q, K);
    SRX_REQUIRE(ctx, srx_aligned(x_dev, srx_dtype_size(dtype)) && srx_aligned(scale_dev, 4), "%s: misaligned buffer", name);
    const QuantArgs p{x_dev, ld_x, rows, ld_q, K, q_dev, scale_dev};
    const int rc = dtype == SRX_F32 ? quant_launch<float>(ctx, name, p) : dtype == SRX_F16 ? quant_launch<srx_f16>(ctx, name, p) : quant_launch<srx_bf16>(ctx, name, p);
    if (rc != SRX_OK) return rc;
    SRX_LAUNCH_CHECK(ctx);
    return SRX_OK;
}

// 32 x 32 tiles for few rows (the product is bound by reading the weights once), and where even these are no more than the chip
// holds at a time (4 rows x 512 -> 2,000 f32: 5 us)
static constexpr int64_t I8_THIN_ROWS = 64;

template <class O, int WI, int WJ, int FI, int FJ>
static int i8_tile(srx_ctx *ctx, const char *name, I8Args &p) {
    typedef Tile<int8_t, WI, WJ, FI, FJ, false, false, TO_LDS> T;
    p.tiles_i = ceil_div64(p.I, T::TI);
    p.tiles_j = ceil_div64(p.J, T::TJ);
    SRX_REQUIRE(ctx, srx_grid_fits(p.tiles_i * p.tiles_j, T::NT), "%s: too many tiles", name);
    SrxProf prof_(ctx, "k_matmul_i8");
    hipLaunchKernelGGL((k_matmul_i8<O, WI, WJ, FI, FJ>), dim3((unsigned)(p.tiles_i * p.tiles_j)), dim3(T::NT), 0, ctx->stream, p);
    return SRX_OK;
}

template <class O>
static int i8_launch(srx_ctx *ctx, const char *name, I8Args &p, int64_t rows) {
    if (rows <= I8_THIN_ROWS || ceil_div64(p.I, 32) * ceil_div64(p.J, 32) <= 2 * (int64_t)ctx->num_cus) {
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
    SRX_REQUIRE(ctx, (stride_n == 1 && stride_r >= N && stride_r <= (1 << 26)) || (stride_r == 1 && stride_n >= rows && stride_n <= (1 << 26)), "%s: output strides %lld, %lld (one of them 1, the other at most 2^26 and no less than what it crosses)", name, (long long)stride_r,
                (long long)stride_n);
    SRX_REQUIRE(ctx, srx_aligned(y_dev, srx_dtype_size(out_dtype)) && srx_aligned(xs_dev, 4) && srx_aligned(ws_dev, 4) && srx_aligned(bias_dev, 4), "%s: misaligned buffer", name);
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
