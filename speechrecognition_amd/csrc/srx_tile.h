// One workgroup's tile of a matrix product on the matrix cores, for f32, f16, bf16 and 8-bit operands:
//
//   D[i][j] = sum over k of P[i][k] Q[j][k],   i < TI, j < TJ
//
// Each operand lies in memory either with its reduction index adjacent ("rows": P[i][k] at base + i * ld + k) or with its other
// index adjacent ("columns": at base + k * ld + i), so that the three products of a linear layer -- x W^T, dy W and dy^T x --
// read their operands where they lie.
//
// All types share one layout.  A slab is SLAB = 128 bytes of reduction per row (64 16-bit, 32 f32, 128 8-bit elements), staged in
// LDS in 16-byte chunks, double buffered; a k-step is 32 bytes: a lane's fragment is one chunk, its half-wave picks the chunk, which is
// the operand layout of v_mfma 32x32x16 (16 bit) and 32x32x32 (8 bit).  f32 runs four 32x32x2 on the chunk's four elements; any
// order of k is right as long as both operands have the same.
//
// Bank conflicts: LDS has 64 banks of 4 bytes and serves 256 bytes, 16 lanes of a 16-byte read, together.  Rows slab: chunk c of row r
// at r * 128 + ((c ^ (r >> 1 & 7)) << 4): 16 neighbouring rows' chunks cover all banks.  Columns slab: [k][TX]; 16-bit fragments come
// through ds_read_b64_tr_b16 (each group of 16 lanes reads 4 k x 16 columns and gets them transposed), 32 lanes 4 k x 64 bytes
// together, so the columns' 64-byte parts are moved by k & 3; f32 ones come element by element, both half-waves' k together, so
// their 128-byte parts are moved by bit 2 of k (turned()).
//
// Bound by the matrix cores and what stands beside them: a workgroup of 256 x 256 fills a CU's LDS and half its registers, so its first
// loads and its stores run beside nobody's products (8 groups, 65,536 rows, 1,024 x 1,024 bf16: matrix cores busy 0.49 of the time,
// forward 170 us or 810 TFLOP/s; 16,384 x 4,096 x 4,096: 1,087).  Tried and slower: slabs of 64 bytes four or five deep (10 %),
// touching the slab after next for the L2 (15 %), four waves of 128 x 128.  Workgroups that stay and take tile after tile were slower
// on the f32 39 -> 39 transform (113 us, 86 then; loads wait behind the stores of the tile before them: the counter of memory
// operations is in order) and are not measured on these tiles.
//
// Result layout: lane l holds column j = l & 31, rows 8 b + 4 (l >> 5) + 0..3 for b = 0..3: four adjacent i for one j.
#pragma once
#include <type_traits>

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

// An operand's part that a tile needs: `n` rows (or columns), element (0, k = 0) at base; columns: `before` more in front of it
struct TileOperand {
    const void *base;
    int64_t ld;   // elements
    int n, before;
};

typedef __attribute__((address_space(3))) unsigned char *lds_bytes;

static constexpr int SLAB = 128, KSTEPS = SLAB / 32;

// How 16-byte chunks come in.  TO_LDS: straight from memory, where every chunk is aligned and whole.  BY_RUN: through registers, any
// address and extent of at least a chunk: the chunk that an extent's end cuts is read as the last 16 bytes in front of that end and
// moved into place, so that every load is one instruction that is always issued (10,007 rows of 429 -> 500 f16, dx and dW: 21 and 23 us;
// 32 and 31 where the last chunk comes element by element, in a branch; a second slab ahead in registers costs 5 to 15 % more).
// BY_ELEMENT: extents below a chunk.
enum TileLoads { BY_ELEMENT, BY_RUN, TO_LDS };

// All loads of the wave have landed, all its LDS accesses are done, and so have everybody else's
__device__ __forceinline__ void tile_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// v without its first `bytes` (0 .. 15, even), zeros behind
__device__ __forceinline__ i32x4_t drop_front(i32x4_t v, int bytes) {
    const bool two = bytes & 8, one = bytes & 4, half = bytes & 2;
    v = two ? i32x4_t{v[2], v[3], 0, 0} : v;
    v = one ? i32x4_t{v[1], v[2], v[3], 0} : v;
    const uint32_t a = v[0], b = v[1], c = v[2], d = v[3];
    return half ? i32x4_t{(int)(a >> 16 | b << 16), (int)(b >> 16 | c << 16), (int)(c >> 16 | d << 16), (int)(d >> 16)} : v;
}

// Columns slab: the column chunk that lies at chunk c of row k (and the other way round)
template <class El, int TX>
__device__ __forceinline__ int turned(int k, int c) {
    if (sizeof(El) == 4) return c ^ ((k >> 2 & 1) << 3);
    return TX >= 128 ? c ^ ((k & 3) << 2) : c ^ ((k >> 1 & 1) << 2);   // (64 columns: two rows to 256 bytes)
}

// COLS: the operand's layout (see above); TX its extent in the tile; NT threads
template <class El, bool COLS, int TX, int NT, TileLoads HOW>
struct TileLoader {
    static constexpr int Z = sizeof(El), EPC = 16 / Z, KS = SLAB / Z;     // elements per chunk, per slab
    static constexpr int CHUNKS = TX * SLAB / 16, PER = CHUNKS / NT;
    static constexpr int CPR = COLS ? TX * Z / 16 : SLAB / 16;            // chunks per slab row
    static constexpr int STEP = NT / CPR;                                 // a thread's chunks: the same of every STEP-th slab row
    static_assert(CHUNKS % NT == 0 && (!COLS || CPR >= 8) && NT % CPR == 0 && STEP % (COLS ? 8 : 16) == 0, "tile shape");
    static constexpr unsigned OUTSIDE = 0x80000000u;                      // past every bound: reads zeros

    const char *base;
    int64_t ldb;         // bytes per row of memory
    int n, before;
    int64_t K;
    unsigned off, step;  // the first chunk's byte offset from the slab's first row / column; bytes to the next one
    int kin;             // rows: first k of the chunks in the slab; columns: k of the first chunk
    int col;             // rows: row of the first chunk; columns: first column of the chunks

    __device__ __forceinline__ void init(const TileOperand &o, int64_t K_, int t) {
        before = COLS && HOW == BY_RUN ? o.before : 0;   // (a chunk that is read from further left stays inside the descriptor)
        base = reinterpret_cast<const char *>(o.base) - (int64_t)before * Z;
        ldb = o.ld * Z;
        n = o.n;
        K = K_;
        step = (unsigned)(STEP * ldb);
        const int r = t / CPR, c = COLS ? turned<El, TX>(r, t % CPR) : t % CPR ^ (r >> 1 & 7);
        off = (unsigned)(r * ldb) + c * 16;
        if constexpr (COLS) {
            kin = r;
            col = c * EPC;
            off += before * Z;
            if (col >= n) off = OUTSIDE;
            else if (HOW == BY_RUN && col + EPC > n) off -= (col + EPC - n) * Z;
        } else {
            kin = c * EPC;
            col = r;
        }
    }
    // A buffer descriptor whose bound makes everything outside the operand read as zeros.  Host's condition: a slab's span < 2 GiB.
    struct Slab { __amdgpu_buffer_rsrc_t r; int left; unsigned at; };
    __device__ __forceinline__ Slab slab(int64_t k0) const {
        const int64_t left = K - k0;
        const char *b = COLS ? base + k0 * ldb : base;
        const int64_t rows = COLS ? (left < KS ? left : KS) : n;
        const unsigned bound = rows > 0 ? (unsigned)((rows - 1) * ldb + (COLS ? (int64_t)(before + n) : K) * Z) : 0u;
        return {__builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(b), 0, bound, 0x00020000), left < 0 ? 0 : left < KS ? (int)left : KS, COLS ? 0u : (unsigned)(k0 * Z)};
    }
    // Host's condition: base and ld are whole chunks, and so is the extent along a chunk (n or K)
    __device__ __forceinline__ void dma(const Slab &s, int i, lds_bytes dst, int wave) const {
        const unsigned o = COLS ? off : kin < s.left ? off + s.at : OUTSIDE;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(s.r, (__attribute__((address_space(3))) void *)(dst + (i * NT + wave * 64) * 16), 16, o + i * step, 0, 0, 0);
    }
    // BY_RUN.  Host's condition: the extent along a chunk is no less than one (columns: with those in front)
    __device__ __forceinline__ void load(const Slab &s, i32x4_t (&v)[PER]) const {
        const int over = kin + EPC - s.left;
        const unsigned o = COLS ? off : over >= EPC ? OUTSIDE : off + s.at - (over > 0 ? over * Z : 0);
#pragma unroll
        for (int i = 0; i < PER; i++) v[i] = __builtin_bit_cast(i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(s.r, o + i * step, 0, 0));
    }
    __device__ __forceinline__ void place(int64_t k0, i32x4_t (&v)[PER]) const {
        const int64_t left = K - k0;
        if (COLS ? n % EPC != 0 : left > 0 && left < KS && left % EPC != 0) {   // (the same for all lanes)
            const int over = COLS ? col + EPC - n : kin + EPC - (int)left;
#pragma unroll
            for (int i = 0; i < PER; i++) v[i] = drop_front(v[i], over > 0 && over < EPC ? over * Z : 0);
        }
    }
    // BY_ELEMENT: any size
    __device__ __forceinline__ void load_elements(int64_t k0, i32x4_t (&v)[PER]) const {
        const El *p = reinterpret_cast<const El *>(base + k0 * (COLS ? ldb : Z) + off);
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int64_t left = K - k0 - kin - (COLS ? i * STEP : 0);
            const int64_t have = COLS ? (left > 0 ? n - col : 0) : (col + i * STEP < n ? left : 0);
            El e[EPC];
#pragma unroll
            for (int q = 0; q < EPC; q++) e[q] = q < have ? p[(int64_t)i * STEP * ldb / Z + q] : (El)0;
            __builtin_memcpy(&v[i], e, 16);
        }
    }
    __device__ __forceinline__ void store(const i32x4_t (&v)[PER], lds_bytes dst, int t) const {
#pragma unroll
        for (int i = 0; i < PER; i++) *reinterpret_cast<__attribute__((address_space(3))) i32x4_t *>(dst + (t + i * NT) * 16) = v[i];
    }
};

__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// A lane's fragments of one operand, `first`: the wave's first row / column in the tile
template <class El, bool COLS, int TX>
struct TileReader {
    unsigned at[4];   // rows: by k-step; columns: by fragment
    __device__ __forceinline__ void init(int first, int lane) {
        const int h = lane >> 5, l = lane & 31;
        if constexpr (!COLS) {
#pragma unroll
            for (int ks = 0; ks < KSTEPS; ks++) at[ks] = (first + l) * SLAB + (((ks * 2 + h) ^ (l >> 1 & 7)) << 4);
        } else {
            const int q = lane & 15, k = sizeof(El) == 2 ? 8 * h + (q >> 2) : 4 * h;
#pragma unroll
            for (int f = 0; f < 4; f++) {
                const int byte = sizeof(El) == 2 ? (first + f * 32 + (l >> 4) * 16 + (q & 3) * 4) * 2 : (first + f * 32 + l) * 4;
                at[f] = k * TX * (int)sizeof(El) + (turned<El, TX>(k, byte >> 4) << 4 | (byte & 15));
            }
        }
    }
    __device__ __forceinline__ i32x4_t read(lds_bytes slab, int ks, int f) const {
        typedef __attribute__((address_space(3))) i32x4_t *vec_ptr;
        if constexpr (!COLS) {
            return *reinterpret_cast<vec_ptr>(slab + at[ks] + f * 32 * SLAB);
        } else if constexpr (sizeof(El) == 2) {
            typedef __attribute__((address_space(3))) s16x4_t *half_ptr;
            const lds_bytes p = slab + at[f] + ks * 16 * TX * 2;
            const s16x4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((half_ptr)p);
            const s16x4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((half_ptr)(p + 4 * TX * 2));
            return __builtin_bit_cast(i32x4_t, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            i32x4_t r;
#pragma unroll
            for (int e = 0; e < 4; e++) r[e] = *reinterpret_cast<__attribute__((address_space(3))) int *>(slab + at[f] + e * TX * 4 + ks * 8 * TX * 4);
            return r;
        }
    }
};

// Elements per 16-byte run of an output type
template <class O>
static constexpr int RUN = 16 / sizeof(O);

// Lane l's value
__device__ __forceinline__ float from_lane(float v, int l) { return __shfl(v, l); }
struct Nothing {};
__device__ __forceinline__ Nothing from_lane(Nothing, int) { return {}; }

// WI x WJ waves of FI x FJ fragments of 32 x 32.  HOW: see TileLoader for what the host has to have checked.
template <class El, int WI_, int WJ_, int FI_, int FJ_, bool PC, bool QC, TileLoads HOW>
struct Tile {
    static constexpr bool DMA = HOW == TO_LDS;
    static constexpr int WI = WI_, WJ = WJ_, FI = FI_, FJ = FJ_;
    static constexpr int NT = WI * WJ * 64, TI = WI * FI * 32, TJ = WJ * FJ * 32;
    static constexpr int KS = SLAB / sizeof(El);
    static constexpr int STAGE = (TI + TJ) * SLAB, LDS = 2 * STAGE;
    typedef typename MxType<El>::acc acc_t;

    // acc = the tile's sums.  SUM: sums[f] = sum over k of Q[j][k] for the lane's column of fragment f, its half-wave's part, where
    // sum_on.  LDS is free on return.
    template <bool SUM>
    static __device__ __forceinline__ void product(unsigned char *smem, const TileOperand &P, const TileOperand &Q, int64_t K, acc_t (&acc)[FI][FJ], float (&sums)[FJ],
                                                   bool sum_on) {
#if defined(__HIP_DEVICE_COMPILE__)   // (the compiler's host pass does not know all of the builtins)
        const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
        const int wi = wave % WI, wj = wave / WI;
        const lds_bytes lds = (lds_bytes)smem;
        TileLoader<El, PC, TI, NT, HOW> lp;
        TileLoader<El, QC, TJ, NT, HOW> lq;
        TileReader<El, PC, TI> rp;
        TileReader<El, QC, TJ> rq;
        rp.init(wi * FI * 32, lane);
        rq.init(wj * FJ * 32, lane);
        // Two slabs of LDS.  While slab s is multiplied, slab s + 1 is on its way (DMA: into the other half; otherwise: into
        // registers).  Fragments are read one k-step ahead of their products; the barrier at a slab's end stands before its last
        // k-step's products, when everything of the slab has been read, so that the next slab's first fragments and the loads of
        // the slab after that one go out behind it.
        constexpr int EACH = TileLoader<El, PC, TI, NT, HOW>::PER + TileLoader<El, QC, TJ, NT, HOW>::PER;
        i32x4_t vp[DMA ? 1 : lp.PER], vq[DMA ? 1 : lq.PER];
        auto ahead = [&](int64_t s, int stage) __attribute__((always_inline)) {
            if constexpr (DMA) {
                const lds_bytes to = lds + stage * STAGE;
                const auto sp = lp.slab(s * KS);
                const auto sq = lq.slab(s * KS);
#pragma unroll
                for (int i = 0; i < lp.PER; i++) lp.dma(sp, i, to, wave);
#pragma unroll
                for (int i = 0; i < lq.PER; i++) lq.dma(sq, i, to + TI * SLAB, wave);
            } else if constexpr (HOW == BY_RUN) {
                lp.load(lp.slab(s * KS), vp);
                lq.load(lq.slab(s * KS), vq);
            } else {
                lp.load_elements(s * KS, vp);
                lq.load_elements(s * KS, vq);
            }
        };
        auto settle = [&](int64_t s, int stage) __attribute__((always_inline)) {   // registers into LDS
            if constexpr (!DMA) {
                const lds_bytes to = lds + stage * STAGE;
                if constexpr (HOW == BY_RUN) {
                    lp.place(s * KS, vp);
                    lq.place(s * KS, vq);
                }
                lp.store(vp, to, t);
                lq.store(vq, to + TI * SLAB, t);
            }
        };
        i32x4_t a[2][FI], b[2][FJ];
        auto fetch = [&](int stage, int ks, int to) __attribute__((always_inline)) {
            const lds_bytes from = lds + stage * STAGE;
#pragma unroll
            for (int i = 0; i < FI; i++) a[to][i] = rp.read(from, ks, i);
#pragma unroll
            for (int j = 0; j < FJ; j++) b[to][j] = rq.read(from + TI * SLAB, ks, j);
        };
        auto multiply = [&](int of, auto &&between) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < FI; i++)
#pragma unroll
                for (int j = 0; j < FJ; j++) {
                    MxType<El>::mma(acc[i][j], a[of][i], b[of][j]);
                    between(i * FJ + j);
                }
            if constexpr (SUM)
                if (sum_on) {
#pragma unroll
                    for (int j = 0; j < FJ; j++) {
                        El e[16 / sizeof(El)];
                        __builtin_memcpy(e, &b[of][j], 16);
#pragma unroll
                        for (int q = 0; q < (int)(16 / sizeof(El)); q++) sums[j] += (float)e[q];
                    }
                }
        };
        lp.init(P, K, t);
        lq.init(Q, K, t);
        const int64_t slabs = (K + KS - 1) / KS;
        ahead(0, 0);
        if constexpr (DMA) ahead(1, 1);
#pragma unroll
        for (int i = 0; i < FI; i++)
#pragma unroll
            for (int j = 0; j < FJ; j++)
#pragma unroll
                for (int e = 0; e < 16; e++) acc[i][j][e] = 0;
#pragma unroll
        for (int j = 0; j < FJ; j++) sums[j] = 0.0f;
        settle(0, 0);
        if constexpr (DMA) tile_barrier(); else lds_barrier();
        if constexpr (!DMA) ahead(1, 1);
        fetch(0, 0, 0);
        for (int64_t s = 0; s < slabs; s++) {
            const int cur = s & 1, nxt = cur ^ 1;
#pragma unroll
            for (int ks = 0; ks + 1 < KSTEPS; ks++) {
                fetch(cur, ks + 1, (ks + 1) & 1);
                __builtin_amdgcn_sched_barrier(0);
                multiply(ks & 1, [](int) {});
                __builtin_amdgcn_sched_barrier(0);
            }
            // (behind the last slab all this goes on with zeros, which nobody uses: one path for the accumulators)
            settle(s + 1, nxt);
            if constexpr (DMA) tile_barrier(); else lds_barrier();   // (loads into registers stay on their way)
            fetch(nxt, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (DMA) {
                // the new slab's loads go out between the products, whose pipe they leave alone
                const lds_bytes to = lds + cur * STAGE;
                const auto sp = lp.slab((s + 2) * KS);
                const auto sq = lq.slab((s + 2) * KS);
                multiply((KSTEPS - 1) & 1, [&](int m) __attribute__((always_inline)) {
#pragma unroll
                    for (int i = 0; i < EACH; i++)
                        if (i * (FI * FJ) / EACH == m) {
                            if (i < lp.PER) lp.dma(sp, i < lp.PER ? i : 0, to, wave);
                            else lq.dma(sq, i < lp.PER ? 0 : i - lp.PER, to + TI * SLAB, wave);
                        }
                    __builtin_amdgcn_sched_barrier(0);
                });
            } else {
                ahead(s + 2, cur);
                __builtin_amdgcn_sched_barrier(0);
                multiply((KSTEPS - 1) & 1, [](int) {});
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        tile_barrier();
#endif
    }

    // Writes a finished tile.  The accumulators' order has four adjacent i per lane and another j in every lane.  In passes of COLS
    // columns per row of waves, the waves put their parts side by side into LDS (f32; chunk c of column j at c ^ (j & 15): no two
    // lanes on one bank) and take whole columns out of it, so that a store is one run of TI outputs.  Its length matters where
    // columns do not begin on lines of 128 bytes (2,000 f32 scores a frame), because every run that a line's border cuts costs a
    // line more: 131,072 x 2,000 f32 with next to nothing to multiply take 305 us in runs of 128 bytes and 214 us in runs of 1 KB.
    // Two areas in turn: one barrier a pass.
    //   held.j[FJ]: what column 32 c + (l & 31) of lane l's wave needs (lane_j); held.i[V]: what the lane's outputs need, those from
    //   lane_i on.  pre(v, j, r): four sums on their way into LDS; post(v, i, j, r): outputs, j() = the column's held.j; out: a
    //   TileOut.
    template <class O> static __device__ __forceinline__ int lane_i() { return (threadIdx.x & 63) % (TI / RUN<O>) * RUN<O>; }
    static __device__ __forceinline__ int lane_j(int c) { return (threadIdx.x >> 6) / WI * FJ * 32 + c * 32 + (threadIdx.x & 31); }

    template <class O, class Held, class Pre, class Post, class Put>
    static __device__ __forceinline__ void write_out(unsigned char *smem, const acc_t (&acc)[FI][FJ], const Held &held, Pre &&pre, Post &&post, Put &&out) {
        constexpr int V = RUN<O>, ROW = TI * 4, COLS = 2 * WJ * 32 * ROW <= LDS ? 32 : 16, LPR = TI / V, RPI = 64 / LPR, EACH = COLS / WI;
        static_assert(2 * WJ * COLS * ROW <= LDS && LPR <= 64 && EACH % RPI == 0 && EACH >= 1, "tile shape");
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int wi = wave % WI, wj = wave / WI, h = lane >> 5, j = lane & 31;
#pragma unroll
        for (int pass = 0; pass < FJ * 32 / COLS; pass++) {
            const int c = pass * COLS / 32, from = pass * COLS % 32;
            unsigned char *st = smem + ((pass & 1) * WJ + wj) * (COLS * ROW);
            if (COLS == 32 || (j >= from && j < from + COLS)) {
#pragma unroll
                for (int f = 0; f < FI; f++)
#pragma unroll
                    for (int b = 0; b < 4; b++) {
                        const acc_t &x = acc[f][c];
                        const float v[4] = {(float)x[4 * b], (float)x[4 * b + 1], (float)x[4 * b + 2], (float)x[4 * b + 3]};
                        f32x4_t r;
                        pre(v, held.j[c], r);
                        *reinterpret_cast<f32x4_t *>(st + (j - from) * ROW + (((wi * FI + f) * 8 + b * 2 + h) ^ (j & 15)) * 16) = r;
                    }
            }
            if constexpr (WI > 1) lds_barrier(); else __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int q = 0; q < EACH / RPI; q++) {
                const int first = wi * EACH + q * RPI, col = first + lane / LPR;
                float v[V], r[V];
#pragma unroll
                for (int e = 0; e < V / 4; e++) {
                    const f32x4_t x = *reinterpret_cast<const f32x4_t *>(st + col * ROW + ((lane % LPR * (V / 4) + e) ^ ((from + col) & 15)) * 16);
#pragma unroll
                    for (int d = 0; d < 4; d++) v[4 * e + d] = x[d];
                }
                post(v, held.i, [&]() { return from_lane(held.j[c], from + col); }, r);
                out(wj * FJ * 32 + c * 32 + from + first, srx_pack<O, V>(r));
            }
        }
    }
};

// An output matrix, i adjacent: the tile that begins at (i = 0, j = 0) = base and of which ni x nj exist; TI / RUN lanes to a column.
// Whole tiles go out without a look at each run's place, and every address is a scalar and the lane's 32-bit offset.
// STREAM: past the caches, which the operands need (131,072 x 1,024 -> 2,048 f32 in 8 bits: 418 us through them, 366 us past them).
template <class O, int TI, bool STREAM = true>
struct TileOut {
    static constexpr int V = RUN<O>, LPR = TI / V;
    O *base;
    int64_t ld;
    int ni, nj;   // of the lane: outputs from its first i on, columns from its own on
    bool whole;
    unsigned lane;
    __device__ __forceinline__ TileOut(O *b, int64_t ld_, int ni_, int nj_, bool whole_) : base(b), ld(ld_), whole(whole_) {
        const int l = threadIdx.x & 63;
        lane = (unsigned)(l / LPR * ld * (int64_t)sizeof(O)) + l % LPR * 16;
        ni = ni_ - l % LPR * V;
        nj = nj_ - l / LPR;
    }
    // (a run is stored whole whatever its alignment)
    __device__ __forceinline__ void operator()(int j, const typename SrxVec<O, V>::type &r) const {
        typedef int any_four __attribute__((ext_vector_type(4), aligned(2)));
        char *p = reinterpret_cast<char *>(base + (int64_t)j * ld);
        if (whole || (j < nj && ni >= V)) {
            if constexpr (STREAM) __builtin_nontemporal_store(__builtin_bit_cast(any_four, r), reinterpret_cast<any_four *>(p + lane));
            else __builtin_memcpy(p + lane, &r, 16);
        } else if (j < nj && ni > 0) {
#pragma unroll
            for (int e = 0; e < V; e++)
                if (e < ni) reinterpret_cast<O *>(p + lane)[e] = r[e];
        }
    }
};

// A tile of 32 x 32 for few rows, where the other operand is read once and nothing else costs: THIN_WAVES waves take the slabs in
// turn, straight from memory into fragments (a wave's four k-steps use whole lines), two slabs in flight each, and add their
// parts through LDS.  Any alignment and size, rows layout for both operands.  emit(i, j, v): four adjacent i.
static constexpr int THIN_WAVES = 8, THIN_LDS = THIN_WAVES * 32 * 32 * 4;

template <class El>
struct ThinOperand {
    static constexpr int Z = sizeof(El), EPC = 16 / Z, KS = SLAB / Z;
    const El *row;
    bool live;
    int64_t K;
    __device__ __forceinline__ void init(const TileOperand &o, int64_t K_, int lane) {
        live = (lane & 31) < o.n;
        row = reinterpret_cast<const El *>(o.base) + (int64_t)(lane & 31) * o.ld + (lane >> 5) * EPC;
        K = K_ - (lane >> 5) * EPC;   // elements from `row` on
    }
    __device__ __forceinline__ void load(int64_t slab, i32x4_t (&v)[KSTEPS]) const {
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ks++) {
            const int64_t k = slab * KS + ks * 2 * EPC, have = live ? K - k : 0;
            i32x4_t r = {0, 0, 0, 0};
            if (have >= EPC) __builtin_memcpy(&r, row + k, 16);
            else if (have > 0) {
                El e[EPC];
#pragma unroll
                for (int q = 0; q < EPC; q++) e[q] = q < have ? row[k + q] : (El)0;
                __builtin_memcpy(&r, e, 16);
            }
            v[ks] = r;
        }
    }
};

template <class El, class Emit>
__device__ __forceinline__ void thin_product(unsigned char *smem, const TileOperand &P, const TileOperand &Q, int64_t K, Emit &&emit) {
    typedef typename MxType<El>::acc acc_t;
    typedef decltype(acc_t{}[0] + acc_t{}[0]) val;
    typedef val val4 __attribute__((ext_vector_type(4)));
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    ThinOperand<El> p, q;
    p.init(P, K, lane);
    q.init(Q, K, lane);
    acc_t acc;
#pragma unroll
    for (int e = 0; e < 16; e++) acc[e] = 0;
    const int64_t slabs = (K + p.KS - 1) / p.KS;
    i32x4_t a[2][KSTEPS], b[2][KSTEPS];
    p.load(wave, a[0]);
    q.load(wave, b[0]);
    for (int64_t s = wave; s < slabs; s += 2 * THIN_WAVES) {
#pragma unroll
        for (int u = 0; u < 2; u++) {   // (slabs past the end are zeros)
            p.load(s + (u + 1) * THIN_WAVES, a[u ^ 1]);
            q.load(s + (u + 1) * THIN_WAVES, b[u ^ 1]);
#pragma unroll
            for (int ks = 0; ks < KSTEPS; ks++) MxType<El>::mma(acc, a[u][ks], b[u][ks]);
        }
    }
    val4 *st = reinterpret_cast<val4 *>(smem);   // [wave][j][8 chunks of i, turned by j]
    const int h = lane >> 5, j = lane & 31;
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const val4 v = {acc[4 * c], acc[4 * c + 1], acc[4 * c + 2], acc[4 * c + 3]};
        st[(wave * 32 + j) * 8 + ((2 * c + h) ^ (j & 7))] = v;
    }
    __syncthreads();
    if (t < 256) {
        const int oj = t >> 3, c = t & 7;
        typedef std::conditional_t<std::is_same<val, int>::value, unsigned, val> part;   // (whole numbers: a sum past the range wraps)
        part v[4];
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = (part)st[oj * 8 + (c ^ (oj & 7))][e];
#pragma unroll
        for (int w = 1; w < THIN_WAVES; w++) {
            const val4 more = st[(w * 32 + oj) * 8 + (c ^ (oj & 7))];
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] += (part)more[e];
        }
        const float f[4] = {(float)(val)v[0], (float)(val)v[1], (float)(val)v[2], (float)(val)v[3]};
        emit(c * 4, oj, f);
    }
}

// v to p[0 .. 4), the first `n` of them
template <class O>
__device__ __forceinline__ void store_four(O *p, const float (&v)[4], int64_t n) {
    const typename SrxVec<O, 4>::type r = srx_pack<O, 4>(v);
    if (n >= 4) __builtin_memcpy(p, &r, 4 * sizeof(O));
    else
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (e < n) p[e] = r[e];
}

// The tile (i, j) of workgroup b.  Workgroups go to the eight XCDs in turn, and each XCD has an L2 of its own: an XCD gets a run
// of neighbouring tiles, and the run goes through bands of TILE_BAND tiles of j, j first, so that the 32 tiles that its CUs hold at
// a time are about 4 x 8 and read 12 operand slabs between them (in rows of i: 2 x 16 and 18).  ni * nj < 2^31 / TILE_BAND.
static constexpr unsigned TILE_BAND = 8;
__device__ __forceinline__ void tile_of(int64_t b, int64_t ni, int64_t nj, int64_t &i, int64_t &j) {
    // (32 bits: a 64-bit division is a hundred instructions, and this stands between a workgroup's tiles)
    const unsigned n = (unsigned)(ni * nj), q = n / 8, r = n % 8, x = (unsigned)b % 8;
    const unsigned item = x * q + (x < r ? x : r) + (unsigned)b / 8, row = TILE_BAND * (unsigned)ni;
    const unsigned band = item / row, in = item - band * row, left = (unsigned)nj - band * TILE_BAND;
    const unsigned h = left < TILE_BAND ? left : TILE_BAND, ti = in / h;
    i = ti;
    j = band * TILE_BAND + (in - ti * h);
}

// Tile of 256 x 256 on 8 waves or of 128 x 128 on 4?  A CU holds one of the former or two of the latter.  A round of the small
// ones costs 0.63 of a round of the large (8 groups, 65,536 rows, 1,024 x 1,024 bf16: 20.8 us and 33 us; 165 us against 187 us in
// all); few tiles are better spread over the chip as small ones.  Fitted at that reduction of 16 slabs only: where the slabs are few
// (429 8-bit elements: 4) a tile's stores weigh more than the rule knows.
static inline bool tile_large(int64_t large, int64_t small, int64_t cus) {
    return ceil_div64(large, cus) * 100 <= ceil_div64(small, 2 * cus) * 63;
}
// Can an operand's memory go straight into LDS (TileLoader::dma)?
static inline bool tile_dma(const void *base, int64_t ld, int64_t extent, int z) {
    const int64_t epc = 16 / z;
    return srx_aligned(base, 16) && ld % epc == 0 && extent % epc == 0 && ld * z < (1 << 22);
}
