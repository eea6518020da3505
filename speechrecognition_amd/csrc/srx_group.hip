// Matrix products whose weights change from group to group of rows, and their gradients:
//
//   y_r  = W_e x_r + b_e          rows r of group e: row_off[e] <= r < row_off[e+1];  W [E][N][K]
//   dx_r = W_e^T dy_r
//   dW_e = sum over r of dy_r x_r^T,   db_e = sum over r of dy_r
//
// The tile of srx_tile.h with i the output's adjacent index, so that a lane stores four neighbours; j is the row (forward, dx) or
// the output unit (dW).  Groups are ragged and known on the device only: row tile number t of the launch belongs to the group e
// with row_off[e] / TJ + e <= t < row_off[e+1] / TJ + e + 1, a closed form that needs no table (the range holds at least the
// ceil(rows / TJ) tiles that group e needs; the spare ones leave at once).
#include <type_traits>

#include "srx_tile.h"

struct GroupArgs {
    const void *x, *w, *dy;
    void *y;
    const float *bias;
    float *dbias;
    int64_t ld_x, ld_dy, ld_y;
    const int64_t *off;
    int64_t total;
    int E, K, N;
    int64_t tiles_i, tiles_j;   // of the launch
    float *part;                // dW split over rows: [S][E][N][K] then [S][E][N], f32
    int splits;
};

__device__ __forceinline__ int64_t group_clamp(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : v > hi ? hi : v; }

// The group of row tile t and the tile's rows; false: a spare tile.  64 candidates at a time: E = 1,000 takes two loads.
template <int TJ>
__device__ __forceinline__ bool group_rows(const GroupArgs &p, int64_t t, int &e, int64_t &r0, int &rows) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = p.E;
    while (n > 1) {
        const int step = (n + 63) / 64, idx = lo + lane * step;
        const bool ok = lane * step < n && group_clamp(p.off[idx], 0, p.total) / TJ + idx <= t;
        const int c = __popcll(__ballot(ok));
        if (c == 0) break;
        const int first = (c - 1) * step;
        n = n - first < step ? n - first : step;
        lo += first;
    }
    e = lo;
    const int64_t a = group_clamp(p.off[e], 0, p.total), b = group_clamp(p.off[e + 1], a, p.total);
    const int64_t j = t - (a / TJ + e);
    r0 = a + j * TJ;
    if (j < 0 || r0 >= b) return false;
    rows = b - r0 < TJ ? (int)(b - r0) : TJ;
    return true;
}

// forward (DX false): i = output unit, reduction over K; dx: i = input unit, reduction over N, W read along its columns
template <class El, class O, bool DX, int WI, int WJ, int FI, int FJ, bool DMA>
__global__ __launch_bounds__(WI *WJ * 64) void k_group(GroupArgs p) {
    typedef Tile<El, WI, WJ, FI, FJ, DX, false, DMA> T;
    __shared__ __attribute__((aligned(1024))) unsigned char smem[T::LDS];
    int64_t ti, tj;
    tile_of(blockIdx.x, p.tiles_i, p.tiles_j, ti, tj);
    const int i0 = (int)ti * T::TI;
    int e, rows;
    int64_t r0;
    if (!group_rows<T::TJ>(p, tj, e, r0, rows)) return;
    const int I = DX ? p.K : p.N, R = DX ? p.N : p.K;
    const El *w = reinterpret_cast<const El *>(p.w) + (int64_t)e * p.N * p.K;
    const int64_t ldq = DX ? p.ld_dy : p.ld_x;
    TileOperand P, Q;
    P.base = DX ? w + i0 : w + (int64_t)i0 * p.K;
    P.ld = p.K;
    P.n = I - i0 < T::TI ? I - i0 : T::TI;
    Q.base = reinterpret_cast<const El *>(DX ? p.dy : p.x) + r0 * ldq;
    Q.ld = ldq;
    Q.n = rows;
    typename T::acc_t acc[FI][FJ];
    float none[FJ];
    T::template product<false>(smem, P, Q, R, acc, none, false);
    O *y = reinterpret_cast<O *>(p.y);
    const float *bias = !DX && p.bias ? p.bias + (int64_t)e * p.N : nullptr;
    struct Held { float b[RUN<O>]; };
    T::template write_out<RUN<O>>(
        smem, acc,
        [&](int i) {
            Held h;
#pragma unroll
            for (int q = 0; q < RUN<O>; q++) h.b[q] = bias && i0 + i + q < I ? bias[i0 + i + q] : 0.0f;
            return h;
        },
        [&](int i, int j, const float (&v)[RUN<O>], const Held &h) {
            if (j >= rows || i0 + i >= I) return;
            float f[RUN<O>];
#pragma unroll
            for (int q = 0; q < RUN<O>; q++) f[q] = v[q] + h.b[q];
            store_run<O>(y + (r0 + j) * p.ld_y + i0 + i, f, I - i0 - i);
        });
}

// forward, few rows per group: tiles of 32 x 32
template <class El, class O>
__global__ __launch_bounds__(THIN_WAVES * 64) void k_group_thin(GroupArgs p) {
    __shared__ __attribute__((aligned(16))) unsigned char smem[THIN_LDS];
    const int i0 = (int)(blockIdx.x % p.tiles_i) * 32;
    int e, rows;
    int64_t r0;
    if (!group_rows<32>(p, blockIdx.x / p.tiles_i, e, r0, rows)) return;
    const El *w = reinterpret_cast<const El *>(p.w) + ((int64_t)e * p.N + i0) * p.K;
    const TileOperand P{w, p.K, p.N - i0 < 32 ? p.N - i0 : 32};
    const TileOperand Q{reinterpret_cast<const El *>(p.x) + r0 * p.ld_x, p.ld_x, rows};
    O *y = reinterpret_cast<O *>(p.y);
    const float *bias = p.bias ? p.bias + (int64_t)e * p.N : nullptr;
    thin_product<El>(smem, P, Q, p.K, [&](int i, int j, const float (&v)[4]) {
        if (j >= rows || i0 + i >= p.N) return;
        float f[4];
#pragma unroll
        for (int q = 0; q < 4; q++) f[q] = v[q] + (bias && i0 + i + q < p.N ? bias[i0 + i + q] : 0.0f);
        store_four<O>(y + (r0 + j) * p.ld_y + i0 + i, f, p.N - i0 - i);
    });
}

// dW (i = input unit k, j = output unit n, reduction over the group's rows) and db with it, taken by the tiles of i = 0 from the
// fragments that they hold anyway.  blockIdx.y: the group; blockIdx.z: the part of its rows.
template <class El, class O, int WI, int WJ, int FI, int FJ, bool DMA>
__global__ __launch_bounds__(WI *WJ * 64) void k_group_dw(GroupArgs p) {
    typedef Tile<El, WI, WJ, FI, FJ, true, true, DMA> T;
    __shared__ __attribute__((aligned(1024))) unsigned char smem[T::LDS];
    int64_t ti, tj;
    tile_of(blockIdx.x, p.tiles_i, p.tiles_j, ti, tj);
    const int i0 = (int)ti * T::TI, j0 = (int)tj * T::TJ;
    const int e = blockIdx.y, z = blockIdx.z;
    const int64_t a = group_clamp(p.off[e], 0, p.total), b = group_clamp(p.off[e + 1], a, p.total);
    const int64_t per = ((b - a + p.splits - 1) / p.splits + T::KS - 1) / T::KS * T::KS;
    const int64_t lo = a + z * per < b ? a + z * per : b, hi = lo + per < b ? lo + per : b;
    TileOperand P, Q;
    P.base = reinterpret_cast<const El *>(p.x) + lo * p.ld_x + i0;
    P.ld = p.ld_x;
    P.n = p.K - i0 < T::TI ? p.K - i0 : T::TI;
    Q.base = reinterpret_cast<const El *>(p.dy) + lo * p.ld_dy + j0;
    Q.ld = p.ld_dy;
    Q.n = p.N - j0 < T::TJ ? p.N - j0 : T::TJ;
    typename T::acc_t acc[FI][FJ];
    float sums[FJ];
    const bool want = p.dbias != nullptr && i0 == 0 && __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % WI == 0;
    T::template product<true>(smem, P, Q, hi - lo, acc, sums, want);
    const bool split = p.splits > 1;
    if (want) {
        const int lane = threadIdx.x & 63, wj = (threadIdx.x >> 6) / WI;
        float *db = split ? p.part + (int64_t)p.splits * p.E * p.N * p.K + ((int64_t)z * p.E + e) * p.N : p.dbias + (int64_t)e * p.N;
#pragma unroll
        for (int f = 0; f < FJ; f++) {
            const float s = sums[f] + __shfl_xor(sums[f], 32);
            const int j = j0 + (wj * FJ + f) * 32 + (lane & 31);
            if (lane < 32 && j < p.N) db[j] = s;
        }
    }
    const auto out = [&](auto *o) {
        typedef std::remove_reference_t<decltype(*o)> Out;
        T::template write_out<RUN<Out>>(
            smem, acc, [](int) { return 0; },
            [&](int i, int j, const float (&v)[RUN<Out>], int) {
                if (j0 + j < p.N && i0 + i < p.K) store_run<Out>(o + (int64_t)(j0 + j) * p.K + i0 + i, v, p.K - i0 - i);
            });
    };
    if (split) out(p.part + ((int64_t)z * p.E + e) * p.N * p.K);
    else out(reinterpret_cast<O *>(p.y) + (int64_t)e * p.N * p.K);
}

// The parts of dW and db, added in their order
template <class O>
__global__ __launch_bounds__(256) void k_group_join(GroupArgs p) {
    const int64_t nw = (int64_t)p.E * p.N * p.K, nb = p.dbias ? (int64_t)p.E * p.N : 0;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < nw + nb; i += (int64_t)gridDim.x * 256) {
        const float *q = i < nw ? p.part + i : p.part + (int64_t)p.splits * nw + (i - nw);
        const int64_t step = i < nw ? nw : (int64_t)p.E * p.N;
        float s = 0.0f;
        for (int z = 0; z < p.splits; z++) s += q[z * step];
        if (i < nw) reinterpret_cast<O *>(p.y)[i] = srx_from_f32<O>(s);
        else p.dbias[i - nw] = s;
    }
}

// ------------------------------------------------------------------------------------------------ host side
static constexpr int64_t GROUP_MAX_ROWS = 1ll << 40;
static constexpr int GROUP_MAX_DIM = 1 << 20;

static int group_check(srx_ctx *ctx, const char *name, int in_dtype, int out_dtype, int E, int64_t total, int K, int N) {
    SRX_REQUIRE(ctx, srx_dtype_size(in_dtype) != 0 && (out_dtype == in_dtype || out_dtype == SRX_F32), "%s: element types %d -> %d (out: the same or f32)", name,
                in_dtype, out_dtype);
    SRX_REQUIRE(ctx, E >= 0 && total >= 0 && K >= 1 && N >= 1, "%s: bad size", name);
    SRX_REQUIRE(ctx, total <= GROUP_MAX_ROWS && K <= GROUP_MAX_DIM && N <= GROUP_MAX_DIM && E <= (1 << 20), "%s: %lld rows in %d groups of %d x %d is too large", name,
                (long long)total, E, N, K);
    return SRX_OK;
}

// Rows of an average group up to which the forward product is bound by reading W once
static constexpr int64_t THIN_ROWS = 32;

template <class El, class O, bool DX, int WI, int WJ, int FI, int FJ, bool DMA>
static int group_tile(srx_ctx *ctx, const char *name, GroupArgs &p) {
    typedef Tile<El, WI, WJ, FI, FJ, DX, false, DMA> T;
    p.tiles_i = ceil_div64(DX ? p.K : p.N, T::TI);
    p.tiles_j = p.total / T::TJ + p.E;
    SRX_REQUIRE(ctx, p.tiles_i * p.tiles_j < (1ll << 31), "%s: too many tiles", name);
    SrxProf prof_(ctx, DX ? "k_group_dx" : "k_group");
    hipLaunchKernelGGL((k_group<El, O, DX, WI, WJ, FI, FJ, DMA>), dim3((unsigned)(p.tiles_i * p.tiles_j)), dim3(T::NT), 0, ctx->stream, p);
    return SRX_OK;
}

template <class El, class O, bool DX>
static int group_launch(srx_ctx *ctx, const char *name, GroupArgs &p) {
    constexpr int Z = sizeof(El);
    const int I = DX ? p.K : p.N;
    if constexpr (!DX)
        if (p.total <= THIN_ROWS * p.E) {
            p.tiles_i = ceil_div64(p.N, 32);
            p.tiles_j = p.total / 32 + p.E;
            SRX_REQUIRE(ctx, p.tiles_i * p.tiles_j < (1ll << 31), "%s: too many tiles", name);
            SrxProf prof_(ctx, "k_group_thin");
            hipLaunchKernelGGL((k_group_thin<El, O>), dim3((unsigned)(p.tiles_i * p.tiles_j)), dim3(THIN_WAVES * 64), 0, ctx->stream, p);
            return SRX_OK;
        }
    if (I <= 64) return group_tile<El, O, DX, 1, 4, 2, 1, false>(ctx, name, p);
    // W is read along its columns (extent K) by dx, along its rows (K) by the forward product
    const bool dma = tile_dma(p.w, p.K, p.K, Z) && (DX ? tile_dma(p.dy, p.ld_dy, p.N, Z) : tile_dma(p.x, p.ld_x, p.K, Z));
    if (!dma) return group_tile<El, O, DX, 2, 2, 2, 2, false>(ctx, name, p);
    if (tile_large(ceil_div64(I, 256) * (p.total / 256 + (p.E + 1) / 2), ceil_div64(I, 128) * (p.total / 128 + (p.E + 1) / 2), ctx->num_cus))
        return group_tile<El, O, DX, 4, 2, 2, 4, true>(ctx, name, p);
    return group_tile<El, O, DX, 2, 2, 2, 2, true>(ctx, name, p);
}

template <bool DX>
static int group_types(srx_ctx *ctx, const char *name, int in, int out, GroupArgs &p) {
    int rc;
    if (in == SRX_F32) rc = group_launch<float, float, DX>(ctx, name, p);
    else if (in == SRX_F16) rc = out == SRX_F32 ? group_launch<srx_f16, float, DX>(ctx, name, p) : group_launch<srx_f16, srx_f16, DX>(ctx, name, p);
    else rc = out == SRX_F32 ? group_launch<srx_bf16, float, DX>(ctx, name, p) : group_launch<srx_bf16, srx_bf16, DX>(ctx, name, p);
    if (rc != SRX_OK) return rc;
    SRX_LAUNCH_CHECK(ctx);
    return SRX_OK;
}

extern "C" int srx_group_matmul_dev(srx_ctx *ctx, int in_dtype, int out_dtype, const void *x_dev, int64_t ld_x, const void *w_dev, const float *bias_dev,
                                    const int64_t *row_off_dev, int n_groups, int64_t total_rows, int K, int N, void *y_dev, int64_t ld_y) {
    const char *name = "srx_group_matmul_dev";
    SRX_ENTER(ctx, name);
    int rc = group_check(ctx, name, in_dtype, out_dtype, n_groups, total_rows, K, N);
    if (rc != SRX_OK || n_groups == 0 || total_rows == 0) return rc;
    SRX_REQUIRE(ctx, x_dev && w_dev && row_off_dev && y_dev, "%s: null argument", name);
    SRX_REQUIRE(ctx, ld_x >= K && ld_y >= N, "%s: a row stride below its %d / %d columns", name, K, N);
    SRX_REQUIRE(ctx, srx_aligned(x_dev, srx_dtype_size(in_dtype)) && srx_aligned(w_dev, srx_dtype_size(in_dtype)) && srx_aligned(y_dev, srx_dtype_size(out_dtype)),
                "%s: misaligned buffer", name);
    GroupArgs p{};
    p.x = x_dev; p.ld_x = ld_x; p.w = w_dev; p.bias = bias_dev; p.y = y_dev; p.ld_y = ld_y;
    p.off = row_off_dev; p.total = total_rows; p.E = n_groups; p.K = K; p.N = N;
    return group_types<false>(ctx, name, in_dtype, out_dtype, p);
}

extern "C" int srx_group_matmul_dx_dev(srx_ctx *ctx, int in_dtype, int out_dtype, const void *dy_dev, int64_t ld_dy, const void *w_dev,
                                       const int64_t *row_off_dev, int n_groups, int64_t total_rows, int K, int N, void *dx_dev, int64_t ld_dx) {
    const char *name = "srx_group_matmul_dx_dev";
    SRX_ENTER(ctx, name);
    int rc = group_check(ctx, name, in_dtype, out_dtype, n_groups, total_rows, K, N);
    if (rc != SRX_OK || n_groups == 0 || total_rows == 0) return rc;
    SRX_REQUIRE(ctx, dy_dev && w_dev && row_off_dev && dx_dev, "%s: null argument", name);
    SRX_REQUIRE(ctx, ld_dy >= N && ld_dx >= K, "%s: a row stride below its %d / %d columns", name, N, K);
    SRX_REQUIRE(ctx, srx_aligned(dy_dev, srx_dtype_size(in_dtype)) && srx_aligned(w_dev, srx_dtype_size(in_dtype)) && srx_aligned(dx_dev, srx_dtype_size(out_dtype)),
                "%s: misaligned buffer", name);
    GroupArgs p{};
    p.dy = dy_dev; p.ld_dy = ld_dy; p.w = w_dev; p.y = dx_dev; p.ld_y = ld_dx;
    p.off = row_off_dev; p.total = total_rows; p.E = n_groups; p.K = K; p.N = N;
    return group_types<true>(ctx, name, in_dtype, out_dtype, p);
}

// Tiles of dW, and the parts that the rows of a group are cut into where there are fewer tiles than fill the chip: the cheapest by
// rounds of tiles (see tile_large), at least DW_MIN_ROWS rows of an average group to a part.  The sum of the parts costs about
// DW_JOIN of a round of an average group's rows for each part's E N K.
struct DwPlan { bool large; int splits; };
static constexpr int64_t DW_MIN_ROWS = 512, DW_CUS = 256;

static DwPlan group_dw_plan(int E, int64_t total, int K, int N) {
    const int64_t nl = E * ceil_div64(K, 256) * ceil_div64(N, 256), ns = E * ceil_div64(K, 128) * ceil_div64(N, 128);
    int64_t most = total / E / DW_MIN_ROWS;
    most = most < 1 ? 1 : most > 64 ? 64 : most;
    DwPlan best{false, 1};
    double cost = 1e300;
    // a round of whole groups of R rows, large tiles: about R * 28 ns (8,192 rows: 230 us); a part's write and read again at
    // 4 TB/s
    const double R = (double)total / E * 28e-9, part = 8.0 * E * N * (double)K / 4e12;
    for (int64_t s = 1; s <= most; s++) {
        const double join = s > 1 ? s * part + 4e-6 : 0.0;
        const double l = (double)ceil_div64(nl * s, DW_CUS) * R / s + join, m = 0.63 * (double)ceil_div64(ns * s, 2 * DW_CUS) * R / s + join;
        if (l < cost) { cost = l; best = {true, (int)s}; }
        if (m < cost) { cost = m; best = {false, (int)s}; }
    }
    return best;
}

extern "C" int64_t srx_group_matmul_dw_scratch_bytes(const srx_ctx *ctx, int n_groups, int64_t total_rows, int K, int N) {
    if (!ctx || n_groups < 0 || n_groups > (1 << 20) || total_rows < 0 || total_rows > GROUP_MAX_ROWS || K < 1 || N < 1 || K > GROUP_MAX_DIM || N > GROUP_MAX_DIM) return -1;
    if (n_groups == 0) return 0;
    const int64_t s = group_dw_plan(n_groups, total_rows, K, N).splits;
    return s == 1 ? 0 : s * n_groups * N * ((int64_t)K + 1) * (int64_t)sizeof(float);
}

template <class El, class O, int WI, int WJ, int FI, int FJ, bool DMA>
static int group_dw_tile(srx_ctx *ctx, const char *name, GroupArgs &p) {
    typedef Tile<El, WI, WJ, FI, FJ, true, true, DMA> T;
    p.tiles_i = ceil_div64(p.K, T::TI);
    p.tiles_j = ceil_div64(p.N, T::TJ);
    SRX_REQUIRE(ctx, p.tiles_i * p.tiles_j < (1ll << 31) && p.E <= 65535, "%s: too many tiles", name);
    SrxProf prof_(ctx, "k_group_dw");
    hipLaunchKernelGGL((k_group_dw<El, O, WI, WJ, FI, FJ, DMA>), dim3((unsigned)(p.tiles_i * p.tiles_j), (unsigned)p.E, (unsigned)p.splits), dim3(T::NT), 0, ctx->stream, p);
    return SRX_OK;
}

template <class El, class O>
static int group_dw_launch(srx_ctx *ctx, const char *name, GroupArgs &p, bool large) {
    const bool dma = tile_dma(p.x, p.ld_x, p.K, sizeof(El)) && tile_dma(p.dy, p.ld_dy, p.N, sizeof(El));
    const int rc = !dma ? group_dw_tile<El, O, 2, 2, 2, 2, false>(ctx, name, p)
                 : large ? group_dw_tile<El, O, 2, 4, 4, 2, true>(ctx, name, p) : group_dw_tile<El, O, 2, 2, 2, 2, true>(ctx, name, p);
    if (rc == SRX_OK && p.splits > 1) {
        const int64_t n = ceil_div64((int64_t)p.E * p.N * (p.K + 1ll), 256);
        SrxProf prof_(ctx, "k_group_join");
        hipLaunchKernelGGL((k_group_join<O>), dim3((unsigned)(n < 4096 ? n : 4096)), dim3(256), 0, ctx->stream, p);
    }
    return rc;
}

extern "C" int srx_group_matmul_dw_dev(srx_ctx *ctx, int in_dtype, int out_dtype, const void *dy_dev, int64_t ld_dy, const void *x_dev, int64_t ld_x,
                                       const int64_t *row_off_dev, int n_groups, int64_t total_rows, int K, int N, void *dw_dev, float *dbias_dev,
                                       void *scratch_dev, int64_t scratch_bytes) {
    const char *name = "srx_group_matmul_dw_dev";
    SRX_ENTER(ctx, name);
    int rc = group_check(ctx, name, in_dtype, out_dtype, n_groups, total_rows, K, N);
    if (rc != SRX_OK || n_groups == 0) return rc;
    SRX_REQUIRE(ctx, row_off_dev && dw_dev && (total_rows == 0 || (dy_dev && x_dev)), "%s: null argument", name);
    SRX_REQUIRE(ctx, ld_dy >= N && ld_x >= K, "%s: a row stride below its %d / %d columns", name, N, K);
    SRX_REQUIRE(ctx, srx_aligned(dy_dev, srx_dtype_size(in_dtype)) && srx_aligned(x_dev, srx_dtype_size(in_dtype)) && srx_aligned(dw_dev, srx_dtype_size(out_dtype)),
                "%s: misaligned buffer", name);
    GroupArgs p{};
    p.dy = dy_dev; p.ld_dy = ld_dy; p.x = x_dev; p.ld_x = ld_x; p.y = dw_dev; p.dbias = dbias_dev;
    p.off = row_off_dev; p.total = total_rows; p.E = n_groups; p.K = K; p.N = N;
    const DwPlan plan = group_dw_plan(n_groups, total_rows, K, N);
    p.splits = plan.splits;
    const int64_t need = srx_group_matmul_dw_scratch_bytes(ctx, n_groups, total_rows, K, N);
    if (need) {
        SRX_REQUIRE(ctx, scratch_dev && scratch_bytes >= need && srx_aligned(scratch_dev, 16), "%s: scratch of %lld bytes, %lld needed, 16-byte aligned (srx_group_matmul_dw_scratch_bytes)",
                    name, (long long)(scratch_dev ? scratch_bytes : 0), (long long)need);
        p.part = reinterpret_cast<float *>(scratch_dev);
    }
    if (in_dtype == SRX_F32) rc = group_dw_launch<float, float>(ctx, name, p, plan.large);
    else if (in_dtype == SRX_F16) rc = out_dtype == SRX_F32 ? group_dw_launch<srx_f16, float>(ctx, name, p, plan.large) : group_dw_launch<srx_f16, srx_f16>(ctx, name, p, plan.large);
    else rc = out_dtype == SRX_F32 ? group_dw_launch<srx_bf16, float>(ctx, name, p, plan.large) : group_dw_launch<srx_bf16, srx_bf16>(ctx, name, p, plan.large);
    if (rc != SRX_OK) return rc;
    SRX_LAUNCH_CHECK(ctx);
    return SRX_OK;
}
