// Gated linear recurrence along the frames of every utterance of a ragged batch, and its backward pass.
//
//   SRX_SCAN_VALUE    h_t = a_t h_(t-1) + x_t              a_t = gate_t
//   SRX_SCAN_SIGMOID  h_t = a_t h_(t-1) + (1 - a_t) x_t    a_t = 1 / (1 + exp(-gate_t))
//
// per channel, h_(-1) = h0.  Backward, with lambda_t = dh_t + a_(t+1) lambda_(t+1) (dh_last behind the last frame):
//   dx_t = lambda_t [(1 - a_t)],  dgate_t = lambda_t h_(t-1)  [lambda_t (h_(t-1) - x_t) a_t (1 - a_t)],  dh0 = a_0 lambda_0.
//
// HBM-bound: three elements move per (frame, channel) forward, five backward.  One lane owns V channels (4 bytes of a row)
// of one segment and walks its frames SB at a time, the next SB rows' loads in flight while the current ones are worked on;
// state and gradient are f32 throughout, every output is rounded once.
//
// Measured (a large copy moves 5.0 TB/s): 499,674 frames x 512 bf16 in 1,000 utterances, SIGMOID: forward 370 us, 1,600 MB with the
// states, 4.3 TB/s; backward 615 us, 2,630 MB, 4.3 TB/s.  One recording of 120,000 x 1,024 f16, VALUE, cut: forward 80 + 18 + 145 us,
// backward 79 + 18 + 238.  1,000 x 39 f32 channels, cut: 30 + 10 + 43 us; 25 of a wave's 64 lanes idle and rows of 156 bytes.
//
// A segment is a whole utterance where the utterances are many and alike; otherwise every utterance is cut into pieces of L
// frames: (1) k_scan_agg reduces each piece to (A, B) with state_out = A state_in + B, (2) k_scan_carry runs the pieces of an
// utterance through that, (3) the main kernel starts every piece from its carry.  Piece (u, j) has the number
// off[u] / L + u + j, a closed form that needs no table: off[u+1] / L + 1 - off[u] / L pieces are at least the
// ceil(frames / L) that utterance u needs.
//
// The backward pass needs h_(t-1).  The forward pass leaves the f32 state in front of every SB-th frame (4 / SB bytes per
// element) and the backward pass recomputes the SB states in between: fewer bytes than reading h back (SIGMOID: 3 reads in
// place of 4) and the gradient of a 16-bit layer is not taken at rounded states.
#include "srx_dtype.h"

static constexpr int SB = SRX_SCAN_STATE_EVERY;   // frames per register block and per stored state

struct ScanArgs {
    const void *gate, *x, *dh;       // [frames][ld]
    int64_t ld_gate, ld_x, ld_dh;
    void *h, *dgate, *dx;
    int64_t ld_h, ld_dgate, ld_dx;
    const float *s_in;               // [n_utt][D] h0 / dh_last, or null
    float *s_out;                    // [n_utt][D] h_last / dh0, or null
    float *states;                   // [total / SB + n_utt][D] or null
    float *A, *B;                    // [pieces][D]: reductions, then (in B) carries
    const int64_t *off;
    int64_t total, pieces;
    int n_utt, D;
    int64_t L;                       // frames per piece; 0: a segment is an utterance
};

__device__ __forceinline__ int64_t clamp64(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : v > hi ? hi : v; }

// utterance u's frames, kept inside [0, total) whatever the table holds
__device__ __forceinline__ void utt_range(const ScanArgs &p, int u, int64_t &lo, int64_t &hi) {
    lo = clamp64(p.off[u], 0, p.total);
    hi = clamp64(p.off[u + 1], lo, p.total);
}

// piece number -> (utterance, first frame, end, frames of the utterance in front of it); an empty range where the number is
// one of the spare ones
struct Seg {
    __device__ __forceinline__ bool spare() const { return first > stop || (first == stop && first != base); }
    int u;
    int64_t first, end, base, stop;   // frames of the piece; of its utterance
};
__device__ __forceinline__ Seg seg_of(const ScanArgs &p, int64_t s) {
    Seg g;
    if (p.L == 0) {
        g.u = (int)s;
        utt_range(p, g.u, g.base, g.stop);
        g.first = g.base;
        g.end = g.stop;
        return g;
    }
    int lo = 0, hi = p.n_utt;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (clamp64(p.off[mid], 0, p.total) / p.L + mid <= s) lo = mid; else hi = mid;
    }
    g.u = lo;
    utt_range(p, lo, g.base, g.stop);
    const int64_t j = s - (g.base / p.L + lo);
    g.first = j < 0 ? g.stop + 1 : g.base + j * p.L;   // in front of the first utterance: spare
    g.end = g.first + p.L < g.stop ? g.first + p.L : g.stop;
    return g;
}

template <class T, int MODE>
__device__ __forceinline__ void gate_of(float g, float &a, float &na) {
    if constexpr (MODE == SRX_SCAN_VALUE) {
        a = g;
        na = 1.0f;
    } else {
        // a = 1 / (1 + e), 1 - a = e a with e = exp(-g): both without cancellation.  The exponent is held at 115 (where a is
        // 2^-115 and 1 - a is 1) so that e stays finite; a NaN passes.  16-bit types: the hardware's exp2 and reciprocal (a few
        // 1e-7 relative, 1/1000 of the output's rounding); f32: the accurate functions.
        if constexpr (sizeof(T) == 4) {
            const float e = expf(g < -80.0f ? 80.0f : -g);
            a = 1.0f / (1.0f + e);
            na = e * a;
        } else {
            const float t = -1.44269504088896340736f * g, e = __builtin_amdgcn_exp2f(t > 115.0f ? 115.0f : t);
            a = __builtin_amdgcn_rcpf(1.0f + e);
            na = e * a;
        }
    }
}

// Which (segment, channels) a lane owns.  UNI: a wave works on one segment (its frame counters live in scalar registers);
// otherwise lanes are dealt out over (segment, channel) in turn, so that few channels still fill a wave.
template <int V, bool UNI>
__device__ __forceinline__ bool lane_item(const ScanArgs &p, int64_t nseg, int64_t &seg, int &ch) {
    const int dv = (p.D + V - 1) / V;
    if constexpr (UNI) {
        const int tiles = (dv + 63) / 64;
        const int64_t wave = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        seg = wave / tiles;
        const int tile = (int)(wave - seg * tiles);
        ch = (tile * 64 + (int)(threadIdx.x & 63)) * V;
        return seg < nseg && ch < p.D;
    } else {
        const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
        seg = id / dv;
        ch = (int)(id - seg * dv) * V;
        return seg < nseg;
    }
}

template <class T, int V>
struct Rows { typename SrxVec<T, V>::type r[SB]; };

// NT: rows that are whole 128-byte lines pass the caches by, since nothing is read twice while it would still be there (the map of
// pieces at 2,048 x 1,024 bf16 115 -> 81 us, k_scan_back at 1,024 utterances x 512 bf16 649 -> 626); rows that share lines with their
// neighbours need the caches (39 f32 channels: 43 -> 61 us without).
template <class vec, bool NT>
__device__ __forceinline__ vec fetch(const char *p) {
    if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const vec *>(p));
    else return *reinterpret_cast<const vec *>(p);
}

// SB rows from `row` on (rows behind end - 1 repeat it: in bounds, their values are not used).  The row's address is uniform where
// the wave works on one segment, the lane adds its 32-bit offset: one scalar add per row
template <class T, int V, bool NT>
__device__ __forceinline__ void load_rows(Rows<T, V> &d, const void *p, int64_t ld, int64_t row, int64_t end, unsigned ch) {
    typedef typename SrxVec<T, V>::type vec;
    const char *base = reinterpret_cast<const char *>(p) + row * ld * (int64_t)sizeof(T);
    const int64_t step = ld * (int64_t)sizeof(T);
    const unsigned lane = ch * (unsigned)sizeof(T);
    if (row + SB <= end) {
#pragma unroll
        for (int i = 0; i < SB; i++) {
            d.r[i] = fetch<vec, NT>(base + lane);
            base += step;
        }
    } else {
#pragma unroll
        for (int i = 0; i < SB; i++) {
            d.r[i] = fetch<vec, NT>(base + lane);
            if (row + i + 1 < end) base += step;
        }
    }
}

template <class T, int V, bool NT>
__device__ __forceinline__ void store_row(char *row, unsigned ch, const float (&f)[V]) {
    typedef typename SrxVec<T, V>::type vec;
    vec *at = reinterpret_cast<vec *>(row + ch * (unsigned)sizeof(T));
    if constexpr (NT) __builtin_nontemporal_store(srx_pack<T, V>(f), at);
    else *at = srx_pack<T, V>(f);
}
template <class T>
__device__ __forceinline__ char *row_at(void *p, int64_t ld, int64_t row) { return reinterpret_cast<char *>(p) + row * ld * (int64_t)sizeof(T); }

// ---- forward, main pass
template <class T, int MODE, int V, bool UNI, bool NT>
__global__ __launch_bounds__(256) void k_scan(ScanArgs p) {
    int64_t s;
    int ch;
    if (!lane_item<V, UNI>(p, p.L ? p.pieces : p.n_utt, s, ch)) return;
    const Seg g = seg_of(p, s);
    if (g.spare()) return;
    float st[V];
#pragma unroll
    for (int v = 0; v < V; v++) {
        const float *c = p.L ? p.B + s * p.D : p.s_in ? p.s_in + (int64_t)g.u * p.D : nullptr;
        st[v] = c ? c[ch + v] : 0.0f;
    }
    if (g.first < g.end) {
        Rows<T, V> ga, xa;
        load_rows<T, V, NT>(ga, p.gate, p.ld_gate, g.first, g.end, ch);
        load_rows<T, V, NT>(xa, p.x, p.ld_x, g.first, g.end, ch);
        float *keep = p.states ? p.states + (g.base / SB + g.u + (g.first - g.base) / SB) * p.D + ch : nullptr;
        for (int64_t row = g.first; row < g.end; row += SB) {
            Rows<T, V> gn = ga, xn = xa;
            if (row + SB < g.end) {
                load_rows<T, V, NT>(gn, p.gate, p.ld_gate, row + SB, g.end, ch);
                load_rows<T, V, NT>(xn, p.x, p.ld_x, row + SB, g.end, ch);
            }
            if (keep) {
#pragma unroll
                for (int v = 0; v < V; v++) keep[v] = st[v];
                keep += p.D;
            }
            const bool full = row + SB <= g.end;
            char *out = row_at<T>(p.h, p.ld_h, row);
#pragma unroll
            for (int i = 0; i < SB; i++) {
                float a[V], b[V];
#pragma unroll
                for (int v = 0; v < V; v++) {
                    float na;
                    gate_of<T, MODE>(srx_elem<T, V>(ga.r[i], v), a[v], na);
                    const float xv = srx_elem<T, V>(xa.r[i], v);
                    b[v] = MODE == SRX_SCAN_VALUE ? xv : na * xv;
                }
                if (full || row + i < g.end) {
#pragma unroll
                    for (int v = 0; v < V; v++) st[v] = __builtin_fmaf(a[v], st[v], b[v]);
                    store_row<T, V, NT>(out, ch, st);
                    out += p.ld_h * (int64_t)sizeof(T);
                }
            }
            ga = gn;
            xa = xn;
        }
    }
    if (p.s_out && g.end == g.stop) {
#pragma unroll
        for (int v = 0; v < V; v++) p.s_out[(int64_t)g.u * p.D + ch + v] = st[v];
    }
}

// ---- backward, main pass
template <class T, int MODE, int V, bool UNI, bool NT>
__global__ __launch_bounds__(256) void k_scan_back(ScanArgs p) {
    int64_t s;
    int ch;
    if (!lane_item<V, UNI>(p, p.L ? p.pieces : p.n_utt, s, ch)) return;
    const Seg g = seg_of(p, s);
    if (g.spare()) return;
    float c[V];   // a_(t+1) lambda_(t+1)
#pragma unroll
    for (int v = 0; v < V; v++) {
        const float *q = p.L ? p.B + s * p.D : p.s_in ? p.s_in + (int64_t)g.u * p.D : nullptr;
        c[v] = q ? q[ch + v] : 0.0f;
    }
    if (g.first < g.end) {
        int64_t row = g.first + (g.end - g.first - 1) / SB * SB;
        const float *keep = p.states + (g.base / SB + g.u + (row - g.base) / SB) * p.D + ch;
        Rows<T, V> ga, xa, da;
        float sa[V];
        load_rows<T, V, NT>(ga, p.gate, p.ld_gate, row, g.end, ch);
        load_rows<T, V, NT>(xa, p.x, p.ld_x, row, g.end, ch);
        load_rows<T, V, NT>(da, p.dh, p.ld_dh, row, g.end, ch);
#pragma unroll
        for (int v = 0; v < V; v++) sa[v] = keep[v];
        for (; row >= g.first; row -= SB) {
            Rows<T, V> gn = ga, xn = xa, dn = da;
            float sn[V];
#pragma unroll
            for (int v = 0; v < V; v++) sn[v] = sa[v];
            if (row > g.first) {
                load_rows<T, V, NT>(gn, p.gate, p.ld_gate, row - SB, g.end, ch);
                load_rows<T, V, NT>(xn, p.x, p.ld_x, row - SB, g.end, ch);
                load_rows<T, V, NT>(dn, p.dh, p.ld_dh, row - SB, g.end, ch);
                keep -= p.D;
#pragma unroll
                for (int v = 0; v < V; v++) sn[v] = keep[v];
            }
            const bool full = row + SB <= g.end;
            float av[SB][V], nav[SB][V], prev[SB][V];
#pragma unroll
            for (int i = 0; i < SB; i++) {
#pragma unroll
                for (int v = 0; v < V; v++) {
                    gate_of<T, MODE>(srx_elem<T, V>(ga.r[i], v), av[i][v], nav[i][v]);
                    prev[i][v] = sa[v];
                    const float xv = srx_elem<T, V>(xa.r[i], v);
                    sa[v] = __builtin_fmaf(av[i][v], sa[v], MODE == SRX_SCAN_VALUE ? xv : nav[i][v] * xv);
                }
            }
            char *odx = row_at<T>(p.dx, p.ld_dx, row), *odg = row_at<T>(p.dgate, p.ld_dgate, row);
#pragma unroll
            for (int i = SB - 1; i >= 0; i--) {
                if (full || row + i < g.end) {
                    float dx[V], dg[V];
#pragma unroll
                    for (int v = 0; v < V; v++) {
                        const float lam = srx_elem<T, V>(da.r[i], v) + c[v];
                        if constexpr (MODE == SRX_SCAN_VALUE) {
                            dx[v] = lam;
                            dg[v] = lam * prev[i][v];
                        } else {
                            dx[v] = lam * nav[i][v];
                            dg[v] = dx[v] * av[i][v] * (prev[i][v] - srx_elem<T, V>(xa.r[i], v));
                        }
                        c[v] = av[i][v] * lam;
                    }
                    store_row<T, V, NT>(odx + i * (p.ld_dx * (int64_t)sizeof(T)), ch, dx);
                    store_row<T, V, NT>(odg + i * (p.ld_dgate * (int64_t)sizeof(T)), ch, dg);
                }
            }
            ga = gn;
            xa = xn;
            da = dn;
#pragma unroll
            for (int v = 0; v < V; v++) sa[v] = sn[v];
        }
    }
    if (p.s_out && g.first == g.base) {
#pragma unroll
        for (int v = 0; v < V; v++) p.s_out[(int64_t)g.u * p.D + ch + v] = c[v];
    }
}

// Products of gates.  Gates above 1 (VALUE only) can overflow a piece's product: a gate of exactly zero still ends it, and a
// state of exactly zero still stays zero through it.  Gates below 1 let it underflow: it is then left at +-GONE, which a finite
// state does not pass and an infinite one does, with its sign, as it passes the gates one by one; exactly zero is a product
// that holds a gate of zero (and no infinity passes: NaN).
static constexpr float GONE = 0x1p-149f;
template <int MODE>
struct Gates {
    float product = 1.0f, least = 1.0f;
    __device__ __forceinline__ void take(float a) {
        product *= a;
        if (MODE == SRX_SCAN_VALUE) least = __builtin_elementwise_minimum(least, fabsf(a));   // (a sigmoid is never zero)
    }
    __device__ __forceinline__ float all() const { return least == 0.0f ? 0.0f : fabsf(product) < GONE ? __builtin_copysignf(GONE, product) : product; }
};
// A s + B; one comparison on the way of s, since this is what a walk over pieces waits for
__device__ __forceinline__ float carry(float A, float B, float s) {
    constexpr int ZERO = 0x060, FINITE = 0x1f8;   // classes: -0, +0; these, denormal and normal ones
    const bool none = __builtin_amdgcn_classf(s, fabsf(A) <= GONE ? FINITE : ZERO);
    return none ? B : __builtin_fmaf(A, s, B);
}

// ---- a piece as one affine map of the state that enters it (BACK: from its far end)
template <class T, int MODE, int V, bool UNI, bool NT, bool BACK>
__global__ __launch_bounds__(256) void k_scan_agg(ScanArgs p) {
    int64_t s;
    int ch;
    if (!lane_item<V, UNI>(p, p.pieces, s, ch)) return;
    const Seg g = seg_of(p, s);
    if (g.first >= g.end) return;
    if (BACK ? g.first == g.base : g.end == g.stop) return;   // nothing follows it
    Gates<MODE> A[V];
    float B[V];
#pragma unroll
    for (int v = 0; v < V; v++) B[v] = 0.0f;
    const void *second = BACK ? p.dh : p.x;
    const int64_t ld2 = BACK ? p.ld_dh : p.ld_x;
    const int64_t nblk = (g.end - g.first + SB - 1) / SB;
    auto blk_row = [&](int64_t b) { return g.first + (BACK ? nblk - 1 - b : b) * SB; };
    Rows<T, V> ga, xa;
    load_rows<T, V, NT>(ga, p.gate, p.ld_gate, blk_row(0), g.end, ch);
    load_rows<T, V, NT>(xa, second, ld2, blk_row(0), g.end, ch);
    for (int64_t b = 0; b < nblk; b++) {
        Rows<T, V> gn = ga, xn = xa;
        if (b + 1 < nblk) {
            load_rows<T, V, NT>(gn, p.gate, p.ld_gate, blk_row(b + 1), g.end, ch);
            load_rows<T, V, NT>(xn, second, ld2, blk_row(b + 1), g.end, ch);
        }
        const int64_t row = blk_row(b);
        const bool full = row + SB <= g.end;
#pragma unroll
        for (int k = 0; k < SB; k++) {
            const int i = BACK ? SB - 1 - k : k;
            float a[V], b[V];
#pragma unroll
            for (int v = 0; v < V; v++) {
                float na;
                gate_of<T, MODE>(srx_elem<T, V>(ga.r[i], v), a[v], na);
                const float xv = srx_elem<T, V>(xa.r[i], v);
                b[v] = BACK || MODE == SRX_SCAN_VALUE ? xv : na * xv;
            }
            if (full || row + i < g.end) {
#pragma unroll
                for (int v = 0; v < V; v++) {
                    B[v] = BACK ? a[v] * (b[v] + B[v]) : __builtin_fmaf(a[v], B[v], b[v]);
                    A[v].take(a[v]);
                }
            }
        }
        ga = gn;
        xa = xn;
    }
#pragma unroll
    for (int v = 0; v < V; v++) {
        p.A[s * p.D + ch + v] = A[v].all();
        p.B[s * p.D + ch + v] = B[v];
    }
}

// ---- the state that enters each piece, left in B.  One workgroup: 64 channels of one utterance, its pieces in CW runs of
// consecutive ones; each wave reduces its run, the runs' maps are chained through LDS, and each wave walks its run again.  Bound by
// the latency of that walk: 375 pieces of 1,024 channels (3 MB) 18 us.
static constexpr int CW = 16;

template <bool BACK>
__global__ __launch_bounds__(64 * CW) void k_scan_carry(ScanArgs p) {
    __shared__ float la[CW][64], lb[CW][64];
    const int u = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int ch = blockIdx.y * 64 + lane;
    int64_t lo, hi;
    utt_range(p, u, lo, hi);
    const int64_t s0 = lo / p.L + u, m = (hi - lo + p.L - 1) / p.L;   // its pieces: s0 .. s0 + m - 1
    const bool on = ch < p.D;
    const int64_t per = (m + CW - 1) / CW, k0 = w * per, k1 = k0 + per < m ? k0 + per : m;
    auto at = [&](int64_t k) { return (s0 + (BACK ? m - 1 - k : k)) * p.D + ch; };
    Gates<SRX_SCAN_VALUE> A;
    float B = 0.0f;
    if (on)
        for (int64_t k = k0; k < k1 && k < m - 1; k++) {   // the last piece's map is never needed (and not there)
            const float a = p.A[at(k)], b = p.B[at(k)];
            B = carry(a, b, B);
            A.take(a);
        }
    la[w][lane] = A.all();
    lb[w][lane] = B;
    __syncthreads();
    if (!on) return;
    float st = p.s_in ? p.s_in[(int64_t)u * p.D + ch] : 0.0f;
    for (int i = 0; i < w; i++) st = carry(la[i][lane], lb[i][lane], st);
    if (m == 0 && w == 0) p.B[s0 * p.D + ch] = st;   // an empty utterance passes its state on
    for (int64_t k = k0; k < k1; k++) {
        float a = 0.0f, b = 0.0f;
        if (k < m - 1) { a = p.A[at(k)]; b = p.B[at(k)]; }
        p.B[at(k)] = st;
        st = carry(a, b, st);
    }
}

// ------------------------------------------------------------------------------------------------ host side
struct ScanPlan {
    int64_t L = 0, pieces = 0;   // L == 0: a segment is an utterance
};

// Cut or not.  SCAN_WAVES waves of 64 lanes with 4 bytes each keep the loads in flight that HBM needs; L gives about so many
// pieces.  Whole utterances win while the longest is no longer than SCAN_WHOLE such pieces (one read of the inputs instead of
// two), pieces win beyond (few or long utterances leave the chip empty).  Where little work leaves L to the latency of its frames, short
// pieces win until the walk over an utterance's pieces takes longer: forward and backward of 14,630 x 2 sigmoid f32 in 7 utterances
// 116 us in pieces of 64 frames, 82 of 32, 68 of 16; 20,000 x 1 in one utterance 138, 103, 122.  SCAN_PIECES to an utterance at most.
static constexpr int64_t SCAN_MAX_FRAMES = 1ll << 40;
static constexpr int SCAN_MAX_DIM = 1 << 20;
static constexpr int64_t SCAN_WAVES = 6144;
static constexpr int64_t SCAN_WHOLE = 3, SCAN_PIECES = 640;

static ScanPlan scan_plan(int n_utt, int64_t total, int64_t max_frames, int D) {
    ScanPlan pl;
    if (max_frames <= 0 || max_frames > total) max_frames = total;
    const int64_t tiles = ceil_div64(D, 64);
    int64_t L = ceil_div64(ceil_div64(total * tiles, SCAN_WAVES), SB) * SB;
    const int64_t least = ceil_div64(ceil_div64(max_frames, SCAN_PIECES), SB) * SB;
    if (L < least) L = least;
    if (L < SB) L = SB;
    if (max_frames <= SCAN_WHOLE * L) return pl;
    pl.L = L;
    pl.pieces = total / L + n_utt;
    return pl;
}

extern "C" int64_t srx_gated_scan_scratch_bytes(const srx_ctx *ctx, int n_utt, int64_t total_frames, int64_t max_frames, int D) {
    if (!ctx || n_utt < 0 || total_frames < 0 || max_frames < 0 || D < 1 || total_frames > SCAN_MAX_FRAMES || D > SCAN_MAX_DIM) return -1;
    return 2 * scan_plan(n_utt, total_frames, max_frames, D).pieces * D * (int64_t)sizeof(float);
}

extern "C" int64_t srx_gated_scan_states_len(const srx_ctx *ctx, int n_utt, int64_t total_frames, int D) {
    if (!ctx || n_utt < 0 || total_frames < 0 || D < 1 || total_frames > SCAN_MAX_FRAMES || D > SCAN_MAX_DIM) return -1;
    return (total_frames / SB + n_utt) * D;
}

template <class T, int MODE, int V, bool UNI, bool NT>
static void scan_launch(srx_ctx *ctx, const ScanArgs &p, bool back) {
    const int64_t nseg = p.L ? p.pieces : p.n_utt;
    const int dv = (p.D + V - 1) / V;
    const int64_t blocks = UNI ? ceil_div64(nseg * ((dv + 63) / 64), 4) : ceil_div64(nseg * dv, 256);
    const dim3 g((unsigned)blocks), b(256), gc((unsigned)p.n_utt, (unsigned)((p.D + 63) / 64));
    if (p.L) {
        {
            SrxProf prof_(ctx, "k_scan_agg");
            if (back) hipLaunchKernelGGL((k_scan_agg<T, MODE, V, UNI, NT, true>), g, b, 0, ctx->stream, p);
            else hipLaunchKernelGGL((k_scan_agg<T, MODE, V, UNI, NT, false>), g, b, 0, ctx->stream, p);
        }
        SrxProf prof_(ctx, "k_scan_carry");
        if (back) hipLaunchKernelGGL((k_scan_carry<true>), gc, dim3(64 * CW), 0, ctx->stream, p);
        else hipLaunchKernelGGL((k_scan_carry<false>), gc, dim3(64 * CW), 0, ctx->stream, p);
    }
    SrxProf prof_(ctx, back ? "k_scan_back" : "k_scan");
    if (back) hipLaunchKernelGGL((k_scan_back<T, MODE, V, UNI, NT>), g, b, 0, ctx->stream, p);
    else hipLaunchKernelGGL((k_scan<T, MODE, V, UNI, NT>), g, b, 0, ctx->stream, p);
}

template <class T, int MODE>
static void scan_pick(srx_ctx *ctx, const ScanArgs &p, bool back, bool wide, bool lines) {
    // 4 bytes per lane and row where the rows allow it; few channels: lanes dealt out over several segments (a wave of one
    // segment would leave more than half of its lanes idle)
    constexpr int V = sizeof(T) == 2 ? 2 : 1;
    if (V == 1 || wide) {
        if (p.D <= 32 * V) scan_launch<T, MODE, V, false, false>(ctx, p, back);
        else if (lines) scan_launch<T, MODE, V, true, true>(ctx, p, back);
        else scan_launch<T, MODE, V, true, false>(ctx, p, back);
        return;
    }
    if (p.D > 32) scan_launch<T, MODE, 1, true, false>(ctx, p, back); else scan_launch<T, MODE, 1, false, false>(ctx, p, back);
}

static int scan_run(srx_ctx *ctx, const char *name, int mode, int dtype, ScanArgs &p, int64_t max_frames, void *scratch, int64_t scratch_bytes,
                    bool back) {
    const ScanPlan pl = scan_plan(p.n_utt, p.total, max_frames, p.D);
    p.L = pl.L;
    p.pieces = pl.pieces;
    const int64_t need = 2 * pl.pieces * p.D * (int64_t)sizeof(float);
    if (need) {
        SRX_REQUIRE(ctx, scratch && scratch_bytes >= need, "%s: scratch of %lld bytes, %lld needed (srx_gated_scan_scratch_bytes)", name,
                    (long long)(scratch ? scratch_bytes : 0), (long long)need);
        SRX_REQUIRE(ctx, srx_aligned(scratch, 4), "%s: scratch is not 4-byte aligned", name);
        p.A = reinterpret_cast<float *>(scratch);
        p.B = p.A + pl.pieces * p.D;
    }
    const int64_t waves = (pl.L ? pl.pieces : p.n_utt) * ceil_div64(p.D, 64);
    SRX_REQUIRE(ctx, srx_grid_fits(ceil_div64(waves, 4), 256) && (!pl.L || srx_grid_fits(p.n_utt, 64 * CW)), "%s: too many utterances and channels", name);
    // `lines`: every row starts on a 128-byte line
    bool wide = p.D % 2 == 0, lines = true;
    const size_t z = srx_dtype_size(dtype);
    auto row = [&](const void *q, int64_t ld) {
        wide = wide && srx_aligned(q, 4) && ld % 2 == 0;
        lines = lines && srx_aligned(q, 128) && ld * z % 128 == 0;
    };
    row(p.gate, p.ld_gate);
    row(p.x, p.ld_x);
    if (back) {
        row(p.dh, p.ld_dh);
        row(p.dgate, p.ld_dgate);
        row(p.dx, p.ld_dx);
    } else row(p.h, p.ld_h);
    const bool sg = mode == SRX_SCAN_SIGMOID;
    if (dtype == SRX_F32) { if (sg) scan_pick<float, SRX_SCAN_SIGMOID>(ctx, p, back, wide, lines); else scan_pick<float, SRX_SCAN_VALUE>(ctx, p, back, wide, lines); }
    else if (dtype == SRX_F16) { if (sg) scan_pick<srx_f16, SRX_SCAN_SIGMOID>(ctx, p, back, wide, lines); else scan_pick<srx_f16, SRX_SCAN_VALUE>(ctx, p, back, wide, lines); }
    else { if (sg) scan_pick<srx_bf16, SRX_SCAN_SIGMOID>(ctx, p, back, wide, lines); else scan_pick<srx_bf16, SRX_SCAN_VALUE>(ctx, p, back, wide, lines); }
    SRX_LAUNCH_CHECK(ctx);
    return SRX_OK;
}

static int scan_check(srx_ctx *ctx, const char *name, int mode, int dtype, int n_utt, int64_t total, int64_t max_frames, int D) {
    SRX_REQUIRE(ctx, mode == SRX_SCAN_VALUE || mode == SRX_SCAN_SIGMOID, "%s: mode %d", name, mode);
    SRX_REQUIRE(ctx, srx_dtype_size(dtype) != 0, "%s: element type %d", name, dtype);
    SRX_REQUIRE(ctx, n_utt >= 0 && total >= 0 && max_frames >= 0 && D >= 1, "%s: bad size", name);
    SRX_REQUIRE(ctx, total <= SCAN_MAX_FRAMES && D <= SCAN_MAX_DIM, "%s: %lld frames of %d channels (at most %lld of %d)", name, (long long)total, D,
                (long long)SCAN_MAX_FRAMES, SCAN_MAX_DIM);
    return SRX_OK;
}

extern "C" int srx_gated_scan_dev(srx_ctx *ctx, int mode, int dtype, const void *gate_dev, int64_t ld_gate, const void *x_dev, int64_t ld_x,
                                  const float *h0_dev, const int64_t *frame_off_dev, int n_utt, int64_t total_frames, int64_t max_frames, int D,
                                  void *h_dev, int64_t ld_h, float *h_last_dev, float *states_dev, void *scratch_dev, int64_t scratch_bytes) {
    SRX_ENTER(ctx, "srx_gated_scan_dev");
    const char *name = "srx_gated_scan_dev";
    int rc = scan_check(ctx, name, mode, dtype, n_utt, total_frames, max_frames, D);
    if (rc != SRX_OK) return rc;
    if (n_utt == 0) return SRX_OK;
    SRX_REQUIRE(ctx, frame_off_dev && (total_frames == 0 || (gate_dev && x_dev && h_dev)), "%s: null argument", name);
    SRX_REQUIRE(ctx, ld_gate >= D && ld_x >= D && ld_h >= D, "%s: a row stride below %d channels", name, D);
    const size_t z = srx_dtype_size(dtype);
    SRX_REQUIRE(ctx, srx_aligned(gate_dev, z) && srx_aligned(x_dev, z) && srx_aligned(h_dev, z) && srx_aligned(h0_dev, 4) && srx_aligned(h_last_dev, 4) && srx_aligned(states_dev, 4) &&
                         srx_aligned(frame_off_dev, 8),
                "%s: misaligned buffer", name);
    ScanArgs p{};
    p.gate = gate_dev; p.ld_gate = ld_gate;
    p.x = x_dev; p.ld_x = ld_x;
    p.h = h_dev; p.ld_h = ld_h;
    p.s_in = h0_dev; p.s_out = h_last_dev; p.states = states_dev;
    p.off = frame_off_dev; p.total = total_frames; p.n_utt = n_utt; p.D = D;
    return scan_run(ctx, name, mode, dtype, p, max_frames, scratch_dev, scratch_bytes, false);
}

extern "C" int srx_gated_scan_backward_dev(srx_ctx *ctx, int mode, int dtype, const void *gate_dev, int64_t ld_gate, const void *x_dev, int64_t ld_x,
                                           const float *states_dev, const void *dh_dev, int64_t ld_dh, const float *dh_last_dev,
                                           const int64_t *frame_off_dev, int n_utt, int64_t total_frames, int64_t max_frames, int D,
                                           void *dgate_dev, int64_t ld_dgate, void *dx_dev, int64_t ld_dx, float *dh0_dev, void *scratch_dev,
                                           int64_t scratch_bytes) {
    SRX_ENTER(ctx, "srx_gated_scan_backward_dev");
    const char *name = "srx_gated_scan_backward_dev";
    int rc = scan_check(ctx, name, mode, dtype, n_utt, total_frames, max_frames, D);
    if (rc != SRX_OK) return rc;
    if (n_utt == 0) return SRX_OK;
    SRX_REQUIRE(ctx, frame_off_dev && (total_frames == 0 || (gate_dev && x_dev && states_dev && dh_dev && dgate_dev && dx_dev)), "%s: null argument", name);
    SRX_REQUIRE(ctx, ld_gate >= D && ld_x >= D && ld_dh >= D && ld_dgate >= D && ld_dx >= D, "%s: a row stride below %d channels", name, D);
    const size_t z = srx_dtype_size(dtype);
    SRX_REQUIRE(ctx, srx_aligned(gate_dev, z) && srx_aligned(x_dev, z) && srx_aligned(dh_dev, z) && srx_aligned(dgate_dev, z) && srx_aligned(dx_dev, z) &&
                         srx_aligned(states_dev, 4) && srx_aligned(dh_last_dev, 4) && srx_aligned(dh0_dev, 4) && srx_aligned(frame_off_dev, 8),
                "%s: misaligned buffer", name);
    ScanArgs p{};
    p.gate = gate_dev; p.ld_gate = ld_gate;
    p.x = x_dev; p.ld_x = ld_x;
    p.dh = dh_dev; p.ld_dh = ld_dh;
    p.dgate = dgate_dev; p.ld_dgate = ld_dgate;
    p.dx = dx_dev; p.ld_dx = ld_dx;
    p.s_in = dh_last_dev; p.s_out = dh0_dev; p.states = const_cast<float *>(states_dev);
    p.off = frame_off_dev; p.total = total_frames; p.n_utt = n_utt; p.D = D;
    return scan_run(ctx, name, mode, dtype, p, max_frames, scratch_dev, scratch_bytes, true);
}
