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
//
// Measured, 8 groups, 65,536 rows, 1,024 x 1,024 bf16 (137 GFLOP each): forward 170 us, dx 194, dW 217 + 20; 16 groups, 32,768 rows, 512 ->
// 2,048 bf16: 105 us (69 GFLOP, 202 MB moved, half of it outputs); 5 groups, 10,007 rows, 429 -> 500 f16: 22, 21, 23 + 12 us.
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
    float *part;                // dW's parts: two slots of TI * TJ + TJ floats per workgroup, and behind them a DwCut of each
};

// The tile that a workgroup of k_group_dw has begun and left to those after it, in `parts` parts with its own (0: it has not)
struct alignas(16) DwCut { int e, i0, j0, parts; };

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

__device__ __forceinline__ void pass_four(const float (&v)[4], Nothing, f32x4_t &r) { r = {v[0], v[1], v[2], v[3]}; }

// forward (DX false): i = output unit, reduction over K; dx: i = input unit, reduction over N, W read along its columns
template <class El, class O, bool DX, int WI, int WJ, int FI, int FJ, TileLoads HOW>
__global__ __launch_bounds__(WI *WJ * 64, 2) void k_group(GroupArgs p) {
    typedef Tile<El, WI, WJ, FI, FJ, DX, false, HOW> T;
    __shared__ __attribute__((aligned(1024))) unsigned char smem[T::LDS];
    struct Held {
        float i[RUN<O>];   // bias
        Nothing j[FJ];
    };
    const int I = DX ? p.K : p.N;
    int64_t ti, tj, r0;
    tile_of(blockIdx.x, p.tiles_i, p.tiles_j, ti, tj);
    int e, rows;
    if (!group_rows<T::TJ>(p, tj, e, r0, rows)) return;
    const int i0 = (int)ti * T::TI, ni = I - i0 < T::TI ? I - i0 : T::TI;
    Held held;
    const int i = T::template lane_i<O>();
#pragma unroll
    for (int q = 0; q < RUN<O>; q++) held.i[q] = !DX && p.bias && i + q < ni ? p.bias[(int64_t)e * p.N + i0 + i + q] : 0.0f;
    const El *w = reinterpret_cast<const El *>(p.w) + (int64_t)e * p.N * p.K;
    const int64_t ldq = DX ? p.ld_dy : p.ld_x;
    const TileOperand P{DX ? w + i0 : w + (int64_t)i0 * p.K, p.K, ni, i0};
    const TileOperand Q{reinterpret_cast<const El *>(DX ? p.dy : p.x) + r0 * ldq, ldq, rows, 0};
    typename T::acc_t acc[FI][FJ];
    float none[FJ];
    T::template product<false>(smem, P, Q, DX ? p.N : p.K, acc, none, false);
    T::template write_out<O>(
        smem, acc, held, pass_four,
        [](const float (&v)[RUN<O>], const float (&bias)[RUN<O>], auto &&, float (&r)[RUN<O>]) {
#pragma unroll
            for (int q = 0; q < RUN<O>; q++) r[q] = v[q] + bias[q];
        },
        TileOut<O, T::TI>(reinterpret_cast<O *>(p.y) + r0 * p.ld_y + i0, p.ld_y, ni, rows, ni == T::TI && rows == T::TJ));
}

// Few outputs (up to 64) and a short reduction (up to NKS k-steps of 32 bytes): a transform of a frame's features.  W stays in a
// wave's registers while it goes through SMALL_ROWS rows of the group, 32 at a time, straight from memory into fragments, the next
// rows on their way behind the products; the outputs go out as they lie in the accumulators (the rows' lines are whole in L2).
// No LDS and no barrier.  1,000 speakers, 499,674 rows of 39 -> 39 f32 (156 MB): 56 us; 81 us through LDS tiles of 64 x 128, 61 and 64 us
// with 128 and 256 rows to a wave.
static constexpr int SMALL_ROWS = 64, SMALL_OUT = 64, SMALL_BYTES = 256;

template <class El, class O, bool DX, int NKS>
__global__ __launch_bounds__(256, 2) void k_group_small(GroupArgs p) {
#if defined(__HIP_DEVICE_COMPILE__)   // (the compiler's host pass does not know all of the builtins)
    constexpr int Z = sizeof(El), EPC = 16 / Z;
    const int lane = threadIdx.x & 63, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int e, rows;
    int64_t r0;
    if (!group_rows<SMALL_ROWS>(p, (int64_t)blockIdx.x * 4 + wave, e, r0, rows)) return;
    constexpr unsigned OUTSIDE = 0x80000000u;
    const int I = DX ? p.K : p.N, R = DX ? p.N : p.K, last = R % EPC ? R / EPC : -1;   // outputs; reduction; the chunk that its end cuts
    const int64_t ldb = (DX ? p.ld_dy : p.ld_x) * Z;
    const auto in = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(reinterpret_cast<const char *>(DX ? p.dy : p.x) + r0 * ldb), 0, (unsigned)((rows - 1) * ldb + R * Z), 0x00020000);
    const auto wr = __builtin_amdgcn_make_buffer_rsrc(const_cast<El *>(reinterpret_cast<const El *>(p.w) + (int64_t)e * p.N * p.K), 0, (unsigned)((int64_t)p.N * p.K * Z), 0x00020000);
    // a chunk of a row at byte `row`: read in front of the row's end where that cuts it (then to be moved), zeros behind
    auto run = [&](auto &from, unsigned row, int c) __attribute__((always_inline)) {
        const int over = c * EPC + EPC - R;
        return __builtin_bit_cast(i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(from, over >= EPC ? OUTSIDE : row + c * 16 - (over > 0 ? over * Z : 0), 0, 0));
    };
    auto whole = [&](i32x4_t (&v)[NKS]) __attribute__((always_inline)) {
#pragma unroll
        for (int ks = 0; ks < NKS; ks++)
            if (last >> 1 == ks) v[ks] = drop_front(v[ks], ks * 2 + h == last ? (EPC - R % EPC) * Z : 0);   // (the same branch for all lanes)
    };
    i32x4_t w[2][NKS], x[NKS];
#pragma unroll
    for (int ks = 0; ks < NKS; ks++) x[ks] = run(in, (unsigned)((lane & 31) * ldb), ks * 2 + h);
#pragma unroll
    for (int f = 0; f < 2; f++) {
        const int i = f * 32 + (lane & 31);
#pragma unroll
        for (int ks = 0; ks < NKS; ks++) {
            if constexpr (!DX) w[f][ks] = run(wr, i < I ? (unsigned)(i * R * Z) : OUTSIDE, ks * 2 + h);
            else {
                El el[EPC];
#pragma unroll
                for (int q = 0; q < EPC; q++) {
                    const int n = (ks * 2 + h) * EPC + q;
                    const unsigned o = n < R && i < I ? (unsigned)((n * I + i) * Z) : OUTSIDE;
                    if constexpr (Z == 4) el[q] = __builtin_bit_cast(El, __builtin_amdgcn_raw_buffer_load_b32(wr, o, 0, 0));
                    else el[q] = __builtin_bit_cast(El, __builtin_amdgcn_raw_buffer_load_b16(wr, o, 0, 0));
                }
                __builtin_memcpy(&w[f][ks], el, 16);
            }
        }
        if constexpr (!DX) whole(w[f]);
    }
    float bias[2][16];
#pragma unroll
    for (int f = 0; f < 2; f++)
#pragma unroll
        for (int q = 0; q < 16; q++) {
            const int i = f * 32 + q / 4 * 8 + h * 4 + q % 4;
            bias[f][q] = !DX && p.bias && i < I ? p.bias[(int64_t)e * I + i] : 0.0f;
        }
    O *out = reinterpret_cast<O *>(p.y) + r0 * p.ld_y;
    for (int row = 0; row < rows; row += 32) {
        i32x4_t next[NKS];
#pragma unroll
        for (int ks = 0; ks < NKS; ks++) next[ks] = run(in, (unsigned)((row + 32 + (lane & 31)) * ldb), ks * 2 + h);
        whole(x);
        const int j = row + (lane & 31);
#pragma unroll
        for (int f = 0; f < 2; f++) {
            typename MxType<El>::acc acc;
#pragma unroll
            for (int q = 0; q < 16; q++) acc[q] = 0;
#pragma unroll
            for (int ks = 0; ks < NKS; ks++) MxType<El>::mma(acc, w[f][ks], x[ks]);
#pragma unroll
            for (int b = 0; b < 4; b++) {
                const int i = f * 32 + b * 8 + h * 4;
                float v[4];
#pragma unroll
                for (int q = 0; q < 4; q++) v[q] = acc[4 * b + q] + bias[f][4 * b + q];
                if (j < rows && i < I) store_four<O>(out + (int64_t)j * p.ld_y + i, v, I - i);
            }
        }
#pragma unroll
        for (int ks = 0; ks < NKS; ks++) x[ks] = next[ks];
    }
#endif
}

// forward, few rows per group: tiles of 32 x 32.  Bound by reading W: 16 rows over 8 groups of 1,024 x 1,024 bf16 (16.8 MB) 7 us with the
// launch.
template <class El, class O>
__global__ __launch_bounds__(THIN_WAVES * 64) void k_group_thin(GroupArgs p) {
    __shared__ __attribute__((aligned(16))) unsigned char smem[THIN_LDS];
    const int i0 = (int)(blockIdx.x % p.tiles_i) * 32;
    int e, rows;
    int64_t r0;
    if (!group_rows<32>(p, blockIdx.x / p.tiles_i, e, r0, rows)) return;
    const El *w = reinterpret_cast<const El *>(p.w) + ((int64_t)e * p.N + i0) * p.K;
    const TileOperand P{w, p.K, p.N - i0 < 32 ? p.N - i0 : 32, 0};
    const TileOperand Q{reinterpret_cast<const El *>(p.x) + r0 * p.ld_x, p.ld_x, rows, 0};
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

// dW (i = input unit k, j = output unit n, reduction over the group's rows), and db with it, taken by the tiles of i = 0 from the
// fragments that they hold anyway.
//
// Groups differ in rows, so tiles differ in work: the workgroups share the slabs instead.  In the order (group, tile, slab) every
// workgroup takes a run of equal length; a tile that one workgroup has to itself goes to its place, the two that its run may cut
// leave their part in f32 in its scratch (slot 0: begun by another, slot 1: left to another), and k_group_join adds the parts in
// their order.  A group of no rows counts as one slab, so that its tiles are written (zeros).  (Whole tiles on a grid of their own: the
// longest group sets the time.  Tiles of 4 x 2 waves 226 us, of 2 x 4 waves 243 us, at 65,536 rows; shares of at least DW_SLABS slabs,
// 8 or more leave a small product to too few workgroups: 10,007 rows 31 us -> 40.)
template <int KS>
__device__ __forceinline__ int64_t dw_slabs(const GroupArgs &p, int e) {
    const int64_t a = group_clamp(p.off[e], 0, p.total), b = group_clamp(p.off[e + 1], a, p.total);
    return b > a ? (b - a + KS - 1) / KS : 1;
}

// The same number in every lane, known to the compiler as such: operand addresses are scalar
__device__ __forceinline__ int64_t uniform64(int64_t v) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)v), hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)((uint64_t)v >> 32));
    return (int64_t)((uint64_t)hi << 32 | lo);
}

// total: slabs of all groups' tiles; len: those of each of the G runs; e: the group in which run `me` begins, and `before`: the
// slabs of the groups before it (of one tile).  Every thread of the workgroup counts a run of groups; sh: a number per thread.
template <int KS, int NT>
__device__ __forceinline__ void dw_find(const GroupArgs &p, int64_t *sh, int64_t tiles, int64_t me, int64_t G, int64_t &total, int64_t &len, int &e, int64_t &before) {
    const int t = threadIdx.x, each = (p.E + NT - 1) / NT;
    const int g0 = t * each < p.E ? t * each : p.E, g1 = g0 + each < p.E ? g0 + each : p.E;
    int64_t mine = 0;
    for (int g = g0; g < g1; g++) mine += dw_slabs<KS>(p, g);
    sh[t] = mine;
    __syncthreads();
    int64_t front = 0, all = 0;
    for (int i = 0; i * each < p.E; i++) {
        const int64_t v = sh[i];
        if (i < t) front += v;
        all += v;
    }
    __syncthreads();
    total = uniform64(all) * tiles;
    len = (total + G - 1) / G;
    const int64_t at = me * len / tiles;   // in slabs of groups
    if (g0 < g1 && front <= at && at < front + mine) {
        int g = g0;
        int64_t f = front;
        for (; g + 1 < g1; g++) {
            const int64_t n = dw_slabs<KS>(p, g);
            if (f + n > at) break;
            f += n;
        }
        sh[0] = g;
        sh[1] = f;
    }
    __syncthreads();
    e = (int)uniform64(sh[0]);
    before = uniform64(sh[1]);
    __syncthreads();
}

template <class El, class O, int WI, int WJ, int FI, int FJ, TileLoads HOW>
__global__ __launch_bounds__(WI *WJ * 64, 2) void k_group_dw(GroupArgs p) {
    typedef Tile<El, WI, WJ, FI, FJ, true, true, HOW> T;
    __shared__ __attribute__((aligned(1024))) unsigned char smem[T::LDS];
    constexpr int64_t SLOT = T::TI * T::TJ + T::TJ;   // (whole lines: a multiple of 128 bytes)
    struct Held { Nothing i[1], j[FJ]; };
    const int64_t tiles = p.tiles_i * p.tiles_j;
    // workgroups of one XCD take neighbouring runs: the tiles of the same rows share its L2
    const int64_t G = gridDim.x, x = blockIdx.x % 8, q8 = G / 8, r8 = G % 8;
    const int64_t me = x * q8 + (x < r8 ? x : r8) + blockIdx.x / 8;
    int64_t total, len, before;
    int e;
    dw_find<T::KS, T::NT>(p, reinterpret_cast<int64_t *>(smem), tiles, me, G, total, len, e, before);
    int64_t at = me * len;
    const int64_t end = at + len < total ? at + len : total;
    DwCut cut{0, 0, 0, 0};
    while (at < end) {
        int64_t n = dw_slabs<T::KS>(p, e);
        while (at >= (before + n) * tiles) {
            before += n;
            e++;
            n = dw_slabs<T::KS>(p, e);
        }
        const int64_t in = at - before * tiles, tile = in / n, s0 = in - tile * n;
        const int64_t s1 = s0 + (end - at) < n ? s0 + (end - at) : n;
        const int64_t a = group_clamp(p.off[e], 0, p.total), b = group_clamp(p.off[e + 1], a, p.total);
        const int64_t lo = a + s0 * T::KS < b ? a + s0 * T::KS : b, hi = a + s1 * T::KS < b ? a + s1 * T::KS : b;
        const int64_t tj = tile / p.tiles_i;
        const int i0 = (int)(tile - tj * p.tiles_i) * T::TI, j0 = (int)tj * T::TJ;
        const TileOperand P{reinterpret_cast<const El *>(p.x) + lo * p.ld_x + i0, p.ld_x, p.K - i0 < T::TI ? p.K - i0 : T::TI, i0};
        const TileOperand Q{reinterpret_cast<const El *>(p.dy) + lo * p.ld_dy + j0, p.ld_dy, p.N - j0 < T::TJ ? p.N - j0 : T::TJ, j0};
        const int slot = s0 > 0 ? 0 : s1 < n ? 1 : -1;   // -1: the whole reduction
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const bool wants = p.dbias != nullptr && i0 == 0 && wave % WI == 0;
        typename T::acc_t acc[FI][FJ];
        float sums[FJ];
        T::template product<true>(smem, P, Q, hi - lo, acc, sums, wants);
        float *part = p.part + (me * 2 + (slot > 0)) * SLOT;
        if (slot > 0) cut = {e, i0, j0, (int)(1 + (n - s1 + len - 1) / len)};
        if (wants) {
            const int lane = threadIdx.x & 63;
#pragma unroll
            for (int f = 0; f < FJ; f++) {
                const float v = sums[f] + __shfl_xor(sums[f], 32);
                const int j = (wave / WI * FJ + f) * 32 + (lane & 31);
                if (lane < 32) {
                    if (slot >= 0) part[T::TI * T::TJ + j] = v;
                    else if (j0 + j < p.N) p.dbias[(int64_t)e * p.N + j0 + j] = v;
                }
            }
        }
        const auto same = [](const auto &v, const Nothing (&)[1], auto &&, auto &r) {
#pragma unroll
            for (int q = 0; q < (int)(sizeof(v) / sizeof(v[0])); q++) r[q] = v[q];
        };
        if (slot >= 0) T::template write_out<float>(smem, acc, Held{}, pass_four, same, TileOut<float, T::TI, false>(part, T::TI, T::TI, T::TJ, true));
        else
            T::template write_out<O>(smem, acc, Held{}, pass_four, same,
                                     TileOut<O, T::TI>(reinterpret_cast<O *>(p.y) + ((int64_t)e * p.N + j0) * p.K + i0, p.K, P.n, Q.n, P.n == T::TI && Q.n == T::TJ));
        at += s1 - s0;
        lds_barrier();   // (the next product's loads go where columns were taken from)
    }
    if (p.part && threadIdx.x == 0) reinterpret_cast<DwCut *>(p.part + G * 2 * SLOT)[me] = cut;
}

// Adds the parts of the tile that workgroup blockIdx.x of k_group_dw's G has left to others: its slot 1, then slot 0 of those that
// follow it.  blockIdx.y: as many of the tile's columns as 256 threads take in fours.
template <int TI>
static constexpr int JOIN_COLS = 1024 / TI;

template <class O, int TI, int TJ>
__global__ __launch_bounds__(256) void k_group_join(GroupArgs p, int64_t G) {
    constexpr int64_t SLOT = TI * TJ + TJ;
    const int64_t g = blockIdx.x;
    const DwCut cut = reinterpret_cast<const DwCut *>(p.part + G * 2 * SLOT)[g];
    if (cut.parts == 0) return;
    const int e = cut.e, i0 = cut.i0, j0 = cut.j0, parts = cut.parts;
    const float *slot = p.part + (g * 2 + 1) * SLOT;
    constexpr int ROWS = JOIN_COLS<TI>;
    for (int c = threadIdx.x; c < ROWS * (TI / 4); c += 256) {
        const int j = blockIdx.y * ROWS + c / (TI / 4), i = c % (TI / 4) * 4;
        if (j0 + j >= p.N || i0 + i >= p.K) continue;
        f32x4_t v = *reinterpret_cast<const f32x4_t *>(slot + j * TI + i);
#pragma unroll 4
        for (int q = 1; q < parts; q++) v += *reinterpret_cast<const f32x4_t *>(slot + (2 * q - 1) * SLOT + j * TI + i);
        const float f[4] = {v[0], v[1], v[2], v[3]};
        store_four<O>(reinterpret_cast<O *>(p.y) + ((int64_t)e * p.N + j0 + j) * p.K + i0 + i, f, p.K - i0 - i);
    }
    if (p.dbias && i0 == 0 && (int)threadIdx.x < ROWS) {
        const int j = blockIdx.y * ROWS + threadIdx.x;
        if (j0 + j < p.N) {
            float v = slot[TI * TJ + j];
            for (int q = 1; q < parts; q++) v += slot[(2 * q - 1) * SLOT + TI * TJ + j];
            p.dbias[(int64_t)e * p.N + j0 + j] = v;
        }
    }
}

// ------------------------------------------------------------------------------------------------ host side
static constexpr int64_t GROUP_MAX_ROWS = 1ll << 40;
static constexpr int GROUP_MAX_DIM = 1 << 20;
static constexpr int64_t GROUP_MAX_LD = 1 << 21;   // (a tile's 128 rows of f32 stay inside 32 bits)

static int group_check(srx_ctx *ctx, const char *name, int in_dtype, int out_dtype, int E, int64_t total, int K, int N) {
    SRX_REQUIRE(ctx, srx_dtype_size(in_dtype) != 0 && (out_dtype == in_dtype || out_dtype == SRX_F32), "%s: element types %d -> %d (out: the same or f32)", name,
                in_dtype, out_dtype);
    SRX_REQUIRE(ctx, E >= 0 && total >= 0 && K >= 1 && N >= 1, "%s: bad size", name);
    SRX_REQUIRE(ctx, total <= GROUP_MAX_ROWS && K <= GROUP_MAX_DIM && N <= GROUP_MAX_DIM && E <= (1 << 20), "%s: %lld rows in %d groups of %d x %d is too large", name,
                (long long)total, E, N, K);
    return SRX_OK;
}

// 32 x 32 tiles: for groups of few rows on average (the product is bound by reading W once), and where even these tiles are no
// more than the chip holds at a time (two to a CU): the larger ones would leave most of it idle, each with a long reduction
// before it (345 rows x 1,370 -> 1 f32: 66 us as 3 tiles of 128 rows, 15 us as 11 of 32 with 8 waves to a reduction).  The groups'
// sizes are on the device, so the rule sees their mean: many groups of one row beside a long one lose (500 x 1 and 15,000 rows, 512 ->
// 512 bf16: 163 us, 63 in the larger tiles).
static constexpr int64_t THIN_ROWS = 32;
static bool group_thin(const srx_ctx *ctx, int64_t total, int E, int N) {
    return total <= THIN_ROWS * E || (total / 32 + E) * ceil_div64(N, 32) <= 2 * (int64_t)ctx->num_cus;
}

template <class El, class O, bool DX, int WI, int WJ, int FI, int FJ, TileLoads HOW>
static int group_tile(srx_ctx *ctx, const char *name, GroupArgs &p) {
    typedef Tile<El, WI, WJ, FI, FJ, DX, false, HOW> T;
    p.tiles_i = ceil_div64(DX ? p.K : p.N, T::TI);
    p.tiles_j = p.total / T::TJ + p.E;
    SRX_REQUIRE(ctx, srx_grid_fits(p.tiles_i * p.tiles_j, T::NT), "%s: too many tiles", name);
    SrxProf prof_(ctx, DX ? "k_group_dx" : "k_group");
    hipLaunchKernelGGL((k_group<El, O, DX, WI, WJ, FI, FJ, HOW>), dim3((unsigned)(p.tiles_i * p.tiles_j)), dim3(T::NT), 0, ctx->stream, p);
    return SRX_OK;
}

template <class El, class O, bool DX, int NKS>
static int group_small(srx_ctx *ctx, const char *name, GroupArgs &p) {
    const int64_t blocks = ceil_div64(p.total / SMALL_ROWS + p.E, 4);
    SRX_REQUIRE(ctx, srx_grid_fits(blocks, 256), "%s: too many tiles", name);
    SrxProf prof_(ctx, DX ? "k_group_dx" : "k_group");
    hipLaunchKernelGGL((k_group_small<El, O, DX, NKS>), dim3((unsigned)blocks), dim3(256), 0, ctx->stream, p);
    return SRX_OK;
}

template <class El, class O, bool DX>
static int group_launch(srx_ctx *ctx, const char *name, GroupArgs &p) {
    constexpr int Z = sizeof(El);
    const int I = DX ? p.K : p.N;
    if constexpr (!DX)
        if (p.K < 16 / Z || group_thin(ctx, p.total, p.E, p.N)) {
            p.tiles_i = ceil_div64(p.N, 32);
            p.tiles_j = p.total / 32 + p.E;
            SRX_REQUIRE(ctx, srx_grid_fits(p.tiles_i * p.tiles_j, THIN_WAVES * 64), "%s: too many tiles", name);
            SrxProf prof_(ctx, "k_group_thin");
            hipLaunchKernelGGL((k_group_thin<El, O>), dim3((unsigned)(p.tiles_i * p.tiles_j)), dim3(THIN_WAVES * 64), 0, ctx->stream, p);
            return SRX_OK;
        }
    if constexpr (DX)
        if (p.N < 16 / Z || p.K < 16 / Z) return group_tile<El, O, DX, 2, 2, 2, 2, BY_ELEMENT>(ctx, name, p);
    const int64_t bytes = (int64_t)(DX ? p.N : p.K) * Z;
    if (I <= SMALL_OUT && bytes <= SMALL_BYTES) {
        if (bytes <= 64) return group_small<El, O, DX, 2>(ctx, name, p);
        if (bytes <= 128) return group_small<El, O, DX, 4>(ctx, name, p);
        if (bytes <= 192) return group_small<El, O, DX, 6>(ctx, name, p);
        return group_small<El, O, DX, 8>(ctx, name, p);
    }
    if (I <= 64) return group_tile<El, O, DX, 1, 4, 2, 1, BY_RUN>(ctx, name, p);
    // W is read along its columns (extent K) by dx, along its rows (K) by the forward product
    const bool dma = tile_dma(p.w, p.K, p.K, Z) && (DX ? tile_dma(p.dy, p.ld_dy, p.N, Z) : tile_dma(p.x, p.ld_x, p.K, Z));
    if (!dma) return group_tile<El, O, DX, 2, 2, 2, 2, BY_RUN>(ctx, name, p);
    // f32 products take the matrix cores eight times as long for the same bytes, so that nothing is gained by reading operands less often,
    // and two workgroups to a CU hide each other's first loads and stores: 32,768 rows of 1,024 -> 1,024 558 us, 723 in 256 x 256 tiles
    if constexpr (Z == 2)
        if (tile_large(ceil_div64(I, 256) * (p.total / 256 + (p.E + 1) / 2), ceil_div64(I, 128) * (p.total / 128 + (p.E + 1) / 2), ctx->num_cus))
            return group_tile<El, O, DX, 4, 2, 2, 4, TO_LDS>(ctx, name, p);
    return group_tile<El, O, DX, 2, 2, 2, 2, TO_LDS>(ctx, name, p);
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
    SRX_REQUIRE(ctx, ld_x >= K && ld_y >= N && ld_x <= GROUP_MAX_LD && ld_y <= GROUP_MAX_LD, "%s: row strides %lld, %lld for %d / %d columns", name, (long long)ld_x, (long long)ld_y, K, N);
    SRX_REQUIRE(ctx, srx_aligned(x_dev, srx_dtype_size(in_dtype)) && srx_aligned(w_dev, srx_dtype_size(in_dtype)) && srx_aligned(y_dev, srx_dtype_size(out_dtype)) &&
                         srx_aligned(bias_dev, 4) && srx_aligned(row_off_dev, 8),
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
    SRX_REQUIRE(ctx, ld_dy >= N && ld_dx >= K && ld_dy <= GROUP_MAX_LD && ld_dx <= GROUP_MAX_LD, "%s: row strides %lld, %lld for %d / %d columns", name, (long long)ld_dy, (long long)ld_dx, N, K);
    SRX_REQUIRE(ctx, srx_aligned(dy_dev, srx_dtype_size(in_dtype)) && srx_aligned(w_dev, srx_dtype_size(in_dtype)) && srx_aligned(dx_dev, srx_dtype_size(out_dtype)) &&
                         srx_aligned(row_off_dev, 8),
                "%s: misaligned buffer", name);
    GroupArgs p{};
    p.dy = dy_dev; p.ld_dy = ld_dy; p.w = w_dev; p.y = dx_dev; p.ld_y = ld_dx;
    p.off = row_off_dev; p.total = total_rows; p.E = n_groups; p.K = K; p.N = N;
    return group_types<true>(ctx, name, in_dtype, out_dtype, p);
}

// dW: workgroups (as many as the chip holds at a time, fewer where a share would be below DW_SLABS slabs) and the size of a part
static constexpr int64_t DW_SLABS = 4;

static int64_t dw_groups(const srx_ctx *ctx, int E, int64_t total, int K, int N, int tile, int ks) {
    const int64_t slabs = (total / ks + E) * ceil_div64(K, tile) * ceil_div64(N, tile), most = (int64_t)ctx->num_cus * (tile == 256 ? 1 : 2);
    const int64_t g = ceil_div64(slabs, DW_SLABS);
    return g < 1 ? 1 : g < most ? g : most;
}
static int64_t dw_bytes(int64_t groups, int tile) { return groups < 2 ? 0 : groups * (2 * (tile * tile + tile) * (int64_t)sizeof(float) + (int64_t)sizeof(DwCut)); }
// 256 x 256 tiles where they cover no more than 128 x 128 ones do, and there is work for more than a slab or two each
static bool dw_large(const srx_ctx *ctx, int E, int64_t total, int K, int N) {
    return ceil_div64(K, 256) * ceil_div64(N, 256) * 4 * 4 <= ceil_div64(K, 128) * ceil_div64(N, 128) * 5 &&
           (total / 64 + E) * ceil_div64(K, 256) * ceil_div64(N, 256) >= 8 * (int64_t)ctx->num_cus;
}

extern "C" int64_t srx_group_matmul_dw_scratch_bytes(const srx_ctx *ctx, int n_groups, int64_t total_rows, int K, int N) {
    if (!ctx || n_groups < 0 || n_groups > (1 << 20) || total_rows < 0 || total_rows > GROUP_MAX_ROWS || K < 1 || N < 1 || K > GROUP_MAX_DIM || N > GROUP_MAX_DIM) return -1;
    if (n_groups == 0) return 0;
    const int64_t large = dw_bytes(dw_groups(ctx, n_groups, total_rows, K, N, 256, 32), 256), small = dw_bytes(dw_groups(ctx, n_groups, total_rows, K, N, 128, 32), 128);
    return dw_large(ctx, n_groups, total_rows, K, N) && large > small ? large : small;   // (the larger slab counts of f32 bound the other types')
}

template <class El, class O, int WI, int WJ, int FI, int FJ, TileLoads HOW>
static int group_dw_tile(srx_ctx *ctx, const char *name, GroupArgs &p) {
    typedef Tile<El, WI, WJ, FI, FJ, true, true, HOW> T;
    p.tiles_i = ceil_div64(p.K, T::TI);
    p.tiles_j = ceil_div64(p.N, T::TJ);
    const int64_t G = dw_groups(ctx, p.E, p.total, p.K, p.N, T::TI, T::KS);
    {
        SrxProf prof_(ctx, "k_group_dw");
        hipLaunchKernelGGL((k_group_dw<El, O, WI, WJ, FI, FJ, HOW>), dim3((unsigned)G), dim3(T::NT), 0, ctx->stream, p);
    }
    if (G > 1) {
        SrxProf prof_(ctx, "k_group_join");
        hipLaunchKernelGGL((k_group_join<O, T::TI, T::TJ>), dim3((unsigned)(G - 1), T::TJ / JOIN_COLS<T::TI>), dim3(256), 0, ctx->stream, p, G);
    }
    return SRX_OK;
}

template <class El, class O>
static int group_dw_launch(srx_ctx *ctx, const char *name, GroupArgs &p) {
    constexpr int Z = sizeof(El);
    if (p.N < 16 / Z || p.K < 16 / Z) return group_dw_tile<El, O, 2, 2, 2, 2, BY_ELEMENT>(ctx, name, p);
    if (!tile_dma(p.x, p.ld_x, p.K, Z) || !tile_dma(p.dy, p.ld_dy, p.N, Z)) return group_dw_tile<El, O, 2, 2, 2, 2, BY_RUN>(ctx, name, p);
    if constexpr (Z == 2)   // (f32: within 2 % of each other)
        if (dw_large(ctx, p.E, p.total, p.K, p.N)) return group_dw_tile<El, O, 4, 2, 2, 4, TO_LDS>(ctx, name, p);
    return group_dw_tile<El, O, 2, 2, 2, 2, TO_LDS>(ctx, name, p);
}

extern "C" int srx_group_matmul_dw_dev(srx_ctx *ctx, int in_dtype, int out_dtype, const void *dy_dev, int64_t ld_dy, const void *x_dev, int64_t ld_x,
                                       const int64_t *row_off_dev, int n_groups, int64_t total_rows, int K, int N, void *dw_dev, float *dbias_dev,
                                       void *scratch_dev, int64_t scratch_bytes) {
    const char *name = "srx_group_matmul_dw_dev";
    SRX_ENTER(ctx, name);
    int rc = group_check(ctx, name, in_dtype, out_dtype, n_groups, total_rows, K, N);
    if (rc != SRX_OK || n_groups == 0) return rc;
    SRX_REQUIRE(ctx, row_off_dev && dw_dev && (total_rows == 0 || (dy_dev && x_dev)), "%s: null argument", name);
    SRX_REQUIRE(ctx, ld_dy >= N && ld_x >= K && ld_dy <= GROUP_MAX_LD && ld_x <= GROUP_MAX_LD, "%s: row strides %lld, %lld for %d / %d columns", name, (long long)ld_dy, (long long)ld_x, N, K);
    SRX_REQUIRE(ctx, srx_aligned(dy_dev, srx_dtype_size(in_dtype)) && srx_aligned(x_dev, srx_dtype_size(in_dtype)) && srx_aligned(dw_dev, srx_dtype_size(out_dtype)) &&
                         srx_aligned(dbias_dev, 4) && srx_aligned(row_off_dev, 8),
                "%s: misaligned buffer", name);
    GroupArgs p{};
    p.dy = dy_dev; p.ld_dy = ld_dy; p.x = x_dev; p.ld_x = ld_x; p.y = dw_dev; p.dbias = dbias_dev;
    p.off = row_off_dev; p.total = total_rows; p.E = n_groups; p.K = K; p.N = N;
    const int64_t need = srx_group_matmul_dw_scratch_bytes(ctx, n_groups, total_rows, K, N);
    if (need) {
        SRX_REQUIRE(ctx, scratch_dev && scratch_bytes >= need && srx_aligned(scratch_dev, 16), "%s: scratch of %lld bytes, %lld needed, 16-byte aligned (srx_group_matmul_dw_scratch_bytes)",
                    name, (long long)(scratch_dev ? scratch_bytes : 0), (long long)need);
        p.part = reinterpret_cast<float *>(scratch_dev);
    }
    if (in_dtype == SRX_F32) rc = group_dw_launch<float, float>(ctx, name, p);
    else if (in_dtype == SRX_F16) rc = out_dtype == SRX_F32 ? group_dw_launch<srx_f16, float>(ctx, name, p) : group_dw_launch<srx_f16, srx_f16>(ctx, name, p);
    else rc = out_dtype == SRX_F32 ? group_dw_launch<srx_bf16, float>(ctx, name, p) : group_dw_launch<srx_bf16, srx_bf16>(ctx, name, p);
    if (rc != SRX_OK) return rc;
    SRX_LAUNCH_CHECK(ctx);
    return SRX_OK;
}
