// One workgroup's tile of a matrix product on the matrix cores, for f32, f16, bf16 and 8-bit operands:
//
//   D[i][j] = sum over k of P[i][k] Q[j][k],   i < TI, j < TJ
//
// Each operand lies in memory either with its reduction index adjacent ("rows": P[i][k] at base + i * ld + k) or with its other
// index adjacent ("columns": at base + k * ld + i), so that the three products of a linear layer -- x W^T, dy W and dy^T x --
// read their operands where they lie.
//
// All types share one layout.  A slab is 128 bytes of reduction per row (64 16-bit, 32 f32, 128 8-bit elements), staged in LDS in
// 16-byte chunks, double buffered; a k-step is 32 bytes: a lane's fragment is one chunk, its half-wave picks the chunk, which is
// the operand layout of v_mfma 32x32x16 (16 bit) and 32x32x32 (8 bit).  f32 runs four 32x32x2 on the chunk's four elements; any
// order of k is right as long as both operands have the same.
//
// Rows slab: chunk c of row r at r * 128 + ((c ^ (r & 7)) << 4): the eight lanes that LDS serves together read eight different
// bank groups.  Columns slab: [k][TX] with the column's 32-byte pairs moved by (k & 3): 16-bit fragments come through
// ds_read_b64_tr_b16 (each group of 16 lanes reads 4 k x 16 columns and gets them transposed), f32 ones element by element.
//
// Result layout: lane l holds column j = l & 31, rows 8 b + 4 (l >> 5) + 0..3 for b = 0..3: four adjacent i for one j.
#pragma once
#include "srx_dtype.h"

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x16_t __attribute__((ext_vector_type(16)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef short s16x8_t __attribute__((ext_vector_type(8)));
typedef srx_f16 f16x8_t __attribute__((ext_vector_type(8)));
typedef srx_bf16 bf16x8_t __attribute__((ext_vector_type(8)));

template <class El> struct MxType;
template <> struct MxType<float> {
    typedef f32x16_t acc;
    static __device__ __forceinline__ void mma(acc &c, i32x4_t p, i32x4_t q) {
        const f32x4_t a = __builtin_bit_cast(f32x4_t, p), b = __builtin_bit_cast(f32x4_t, q);
#pragma unroll
        for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    }
};
template <> struct MxType<srx_f16> {
    typedef f32x16_t acc;
    static __device__ __forceinline__ void mma(acc &c, i32x4_t p, i32x4_t q) {
        c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, p), __builtin_bit_cast(f16x8_t, q), c, 0, 0, 0);
    }
};
template <> struct MxType<srx_bf16> {
    typedef f32x16_t acc;
    static __device__ __forceinline__ void mma(acc &c, i32x4_t p, i32x4_t q) {
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, p), __builtin_bit_cast(bf16x8_t, q), c, 0, 0, 0);
    }
};
template <> struct MxType<int8_t> {
    typedef i32x16_t acc;
    static __device__ __forceinline__ void mma(acc &c, i32x4_t p, i32x4_t q) { c = __builtin_amdgcn_mfma_i32_32x32x32_i8(p, q, c, 0, 0, 0); }
};

// An operand's part that a tile needs: `n` rows (or columns), element (0, k = 0) at base
struct TileOperand {
    const void *base;
    int64_t ld;   // elements
    int n;
};

typedef __attribute__((address_space(3))) unsigned char *lds_bytes;

// All loads of the wave have landed, all its LDS reads are done, and so have everybody else's
__device__ __forceinline__ void tile_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// COLS: the operand's layout (see above); TX its extent in the tile; NT threads
template <class El, bool COLS, int TX, int NT>
struct TileLoader {
    static constexpr int Z = sizeof(El), EPC = 16 / Z, KS = 128 / Z;      // elements per chunk, per slab
    static constexpr int CHUNKS = TX * 8, PER = CHUNKS / NT;
    static constexpr int CPR = COLS ? TX * Z / 16 : 8;                    // chunks per slab row
    static_assert(CHUNKS % NT == 0 && (!COLS || CPR >= 8), "tile shape");
    static constexpr unsigned OUTSIDE = 0x80000000u;                      // past every bound: reads zeros

    const char *base;
    int64_t ldb;         // bytes per row of memory
    int n;
    int64_t K;
    unsigned off[PER];   // chunk's byte offset from the slab's first row / column
    int kin[PER];        // rows: first k of the chunk in its slab; columns: its k
    int col[PER];        // rows: its row; columns: its first column

    __device__ __forceinline__ void init(const TileOperand &o, int64_t K_, int t) {
        base = reinterpret_cast<const char *>(o.base);
        ldb = o.ld * Z;
        n = o.n;
        K = K_;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int s = t + i * NT, r = s / CPR, cs = s % CPR;
            if constexpr (COLS) {
                const int c = cs ^ ((r & 3) << 1);
                kin[i] = r;
                col[i] = c * EPC;
                off[i] = (unsigned)(r * ldb) + c * 16;
                if (col[i] >= n) off[i] = OUTSIDE;
            } else {
                const int c = cs ^ (r & 7);
                kin[i] = c * EPC;
                col[i] = r;
                off[i] = (unsigned)(r * ldb) + c * 16;
            }
        }
    }
    // Straight into LDS, 16 bytes a lane, through a buffer descriptor whose bound makes everything outside the operand read
    // as zeros.  Host's condition: base and ld are whole chunks, so is the extent along a chunk (n or K); a slab's span < 2 GiB.
    __device__ __forceinline__ void dma(int64_t k0, lds_bytes dst, int wave) const {
        const int64_t left = K - k0;
        const char *b = COLS ? base + k0 * ldb : base;
        const int64_t rows = COLS ? (left < KS ? left : KS) : n;
        const unsigned bound = rows > 0 ? (unsigned)((rows - 1) * ldb + (COLS ? (int64_t)n : K) * Z) : 0u;
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(b), 0, bound, 0x00020000);
#pragma unroll
        for (int i = 0; i < PER; i++) {
            unsigned o = off[i];
            if constexpr (!COLS) o = kin[i] < left ? o + (unsigned)(k0 * Z) : OUTSIDE;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)(dst + (i * NT + wave * 64) * 16), 16, o, 0, 0, 0);
        }
    }
    // Any alignment and size: whole chunks by one (unaligned) 16-byte load, the rest element by element
    __device__ __forceinline__ void load(int64_t k0, i32x4_t (&v)[PER]) const {
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int64_t k = k0 + kin[i];
            const int64_t have = COLS ? (k < K ? (int64_t)n - col[i] : 0) : (col[i] < n ? K - k : 0);
            const char *p = COLS ? base + k * ldb + (int64_t)col[i] * Z : base + (int64_t)col[i] * ldb + k * Z;
            i32x4_t r = {0, 0, 0, 0};
            if (have >= EPC) __builtin_memcpy(&r, p, 16);
            else if (have > 0) {
                El e[EPC];
#pragma unroll
                for (int q = 0; q < EPC; q++) e[q] = q < have ? reinterpret_cast<const El *>(p)[q] : (El)0;
                __builtin_memcpy(&r, e, 16);
            }
            v[i] = r;
        }
    }
    __device__ __forceinline__ void store(const i32x4_t (&v)[PER], lds_bytes dst, int t) const {
#pragma unroll
        for (int i = 0; i < PER; i++) *reinterpret_cast<__attribute__((address_space(3))) i32x4_t *>(dst + (t + i * NT) * 16) = v[i];
    }
};

// A lane's fragments of one operand, `first`: the wave's first row / column in the tile
template <class El, bool COLS, int TX>
struct TileReader {
    unsigned at[4];
    __device__ __forceinline__ void init(int first, int lane) {
        const int h = lane >> 5;
        if constexpr (!COLS) {
#pragma unroll
            for (int ks = 0; ks < 4; ks++) at[ks] = (first + (lane & 31)) * 128 + (((ks * 2 + h) ^ (lane & 7)) << 4);
        } else if constexpr (sizeof(El) == 2) {
            const int q = lane & 15, k = q >> 2;
            const unsigned c = (first + ((lane >> 4) & 1) * 16 + (q & 3) * 4) * 2;
            at[0] = (8 * h + k) * TX * 2 + (c ^ (k << 5));            // fragments 0, 2, ..
            at[1] = (8 * h + k) * TX * 2 + ((c + 64) ^ (k << 5));     // fragments 1, 3, ..
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) at[e] = (4 * h + e) * TX * 4 + ((unsigned)((first + (lane & 31)) * 4) ^ (e << 5));
        }
    }
    __device__ __forceinline__ i32x4_t read(lds_bytes slab, int ks, int f) const {
        typedef __attribute__((address_space(3))) i32x4_t *vec_ptr;
        if constexpr (!COLS) {
            return *reinterpret_cast<vec_ptr>(slab + at[ks] + f * 32 * 128);
        } else if constexpr (sizeof(El) == 2) {
            typedef __attribute__((address_space(3))) s16x4_t *half_ptr;
            const lds_bytes p = slab + at[f & 1] + (f >> 1) * 128 + ks * 16 * TX * 2;
            const s16x4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((half_ptr)p);
            const s16x4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((half_ptr)(p + 4 * TX * 2));
            return __builtin_bit_cast(i32x4_t, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            i32x4_t r;
#pragma unroll
            for (int e = 0; e < 4; e++) r[e] = *reinterpret_cast<__attribute__((address_space(3))) int *>(slab + at[e] + f * 128 + ks * 8 * TX * 4);
            return r;
        }
    }
};

// WI x WJ waves of FI x FJ fragments of 32 x 32.  DMA: see TileLoader::dma for what the host has to have checked.
template <class El, int WI_, int WJ_, int FI_, int FJ_, bool PC, bool QC, bool DMA>
struct Tile {
    static constexpr int WI = WI_, WJ = WJ_, FI = FI_, FJ = FJ_;
    static constexpr int NT = WI * WJ * 64, TI = WI * FI * 32, TJ = WJ * FJ * 32;
    static constexpr int KS = 128 / sizeof(El);
    static constexpr int STAGE = (TI + TJ) * 128, LDS = 2 * STAGE;
    typedef typename MxType<El>::acc acc_t;

    // SUM: also sums[f] += sum over k of Q[j][k] for the lane's column of fragment f, its half-wave's part (sum_on: wanted)
    template <bool SUM>
    static __device__ __forceinline__ void product(unsigned char *smem, const TileOperand &P, const TileOperand &Q, int64_t K, acc_t (&acc)[FI][FJ],
                                                   float (&sums)[FJ], bool sum_on) {
        const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
        const int wi = wave % WI, wj = wave / WI;
        const lds_bytes lds = (lds_bytes)smem;
        TileLoader<El, PC, TI, NT> lp;
        TileLoader<El, QC, TJ, NT> lq;
        TileReader<El, PC, TI> rp;
        TileReader<El, QC, TJ> rq;
        lp.init(P, K, t);
        lq.init(Q, K, t);
        rp.init(wi * FI * 32, lane);
        rq.init(wj * FJ * 32, lane);
#pragma unroll
        for (int i = 0; i < FI; i++)
#pragma unroll
            for (int j = 0; j < FJ; j++)
#pragma unroll
                for (int e = 0; e < 16; e++) acc[i][j][e] = 0;
#pragma unroll
        for (int j = 0; j < FJ; j++) sums[j] = 0.0f;
        const int64_t slabs = (K + KS - 1) / KS;
        if (slabs <= 0) return;
        i32x4_t vp[DMA ? 1 : lp.PER], vq[DMA ? 1 : lq.PER];
        if constexpr (DMA) {
            lp.dma(0, lds, wave);
            lq.dma(0, lds + TI * 128, wave);
        } else {
            lp.load(0, vp);
            lq.load(0, vq);
            lp.store(vp, lds, t);
            lq.store(vq, lds + TI * 128, t);
        }
        tile_barrier();
        for (int64_t s = 0; s < slabs; s++) {
            const lds_bytes cur = lds + (s & 1) * STAGE, nxt = lds + ((s + 1) & 1) * STAGE;
            const bool more = s + 1 < slabs;
            if (more) {
                if constexpr (DMA) {
                    lp.dma((s + 1) * KS, nxt, wave);
                    lq.dma((s + 1) * KS, nxt + TI * 128, wave);
                } else {
                    lp.load((s + 1) * KS, vp);
                    lq.load((s + 1) * KS, vq);
                }
            }
#pragma unroll
            for (int ks = 0; ks < 4; ks++) {
                i32x4_t a[FI], b[FJ];
#pragma unroll
                for (int i = 0; i < FI; i++) a[i] = rp.read(cur, ks, i);
#pragma unroll
                for (int j = 0; j < FJ; j++) b[j] = rq.read(cur + TI * 128, ks, j);
#pragma unroll
                for (int i = 0; i < FI; i++)
#pragma unroll
                    for (int j = 0; j < FJ; j++) MxType<El>::mma(acc[i][j], a[i], b[j]);
                if constexpr (SUM)
                    if (sum_on) {
#pragma unroll
                        for (int j = 0; j < FJ; j++) {
                            El e[16 / sizeof(El)];
                            __builtin_memcpy(e, &b[j], 16);
#pragma unroll
                            for (int q = 0; q < (int)(16 / sizeof(El)); q++) sums[j] += (float)e[q];
                        }
                    }
            }
            if constexpr (!DMA)
                if (more) {
                    lp.store(vp, nxt, t);
                    lq.store(vq, nxt + TI * 128, t);
                }
            tile_barrier();
        }
    }

    // f(i, j, v): v[0..3] are D[i .. i+3][j], i a multiple of 4, both counted within the tile
    template <class F>
    static __device__ __forceinline__ void each(const acc_t (&acc)[FI][FJ], F &&f) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int i0 = (wave % WI) * FI * 32 + 4 * (lane >> 5), j0 = (wave / WI) * FJ * 32 + (lane & 31);
#pragma unroll
        for (int j = 0; j < FJ; j++)
#pragma unroll
            for (int i = 0; i < FI; i++)
#pragma unroll
                for (int b = 0; b < 4; b++) {
                    const decltype(acc[0][0][0] + acc[0][0][0]) v[4] = {acc[i][j][4 * b], acc[i][j][4 * b + 1], acc[i][j][4 * b + 2], acc[i][j][4 * b + 3]};
                    f(i0 + i * 32 + b * 8, j0 + j * 32, v);
                }
    }
};

// v[0..3] to p[0..3], the first `n` of them; whole and aligned quadruples as one store
template <class O>
__device__ __forceinline__ void store4(O *p, const float (&v)[4], int64_t n, bool aligned) {
    if (n >= 4 && aligned) *reinterpret_cast<typename SrxVec<O, 4>::type *>(p) = srx_pack<O, 4>(v);
    else
        for (int e = 0; e < 4; e++)
            if (e < n) p[e] = srx_from_f32<O>(v[e]);
}

// Workgroups go to the eight XCDs in turn, and each XCD has an L2 of its own: work item w of n for workgroup b, such that an
// XCD works on a run of neighbouring items (which share their operands)
__device__ __forceinline__ int64_t xcd_item(int64_t b, int64_t n) {
    const int64_t q = n / 8, r = n % 8, x = b % 8, i = b / 8;
    return x * q + (x < r ? x : r) + i;
}
