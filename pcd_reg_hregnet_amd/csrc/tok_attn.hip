// tok_attn.hip -- attention over token sequences: forward, and the backward pass that
// recomputes the probabilities from the stored logarithm of their sums; a learned relative
// position bias by buckets and its gradient are part of both.
//
//   s_ij = scale q_i . k_j + bias[bucket(j - i - start)]     (masked: -inf)
//   p_ij = exp(s_ij - lse_i),  o_i = sum_j p_ij v_j
//   D_i  = do_i . o_i,  ds_ij = p_ij (do_i . v_j - D_i)
//   dv_j = sum_i p_ij do_i,  dk_j = scale sum_i ds_ij q_i,  dq_i = scale sum_j ds_ij k_j
//   dbias[b] = sum of ds_ij over all pairs in bucket b
//
// All products run on v_mfma_f32_32x32x16_bf16: bf16 operands as they are, f32 operands as
// three exact bf16 pieces (six products).  Scores are made transposed (keys x queries) where
// the next product sums over keys, and straight (queries x keys) where it sums over queries:
// the result registers are then already the next product's operand.  Scores, sums and
// accumulators are f32; p and ds are rounded to bf16 for bf16 tensors (off by at most 2^-8 of
// each, as the tensors themselves are; to 16 bits where that costs nothing or few keys average too little
// of it: attn_split, few_keys, prob_pieces), and cut into three exact pieces for f32 tensors.

#include <float.h>

#include "tokens.h"

namespace {

using namespace hreg_tok;

constexpr float LOG2E = 1.4426950408889634f;
constexpr int NT = 256;          // threads a workgroup
constexpr int ROWS = 128;        // rows a workgroup owns: 32 a wave
constexpr int CUS = 256;
constexpr int FEW_KEYS = 64;
constexpr int MAX_BINS = 2049;   // offsets -max_distance .. max_distance with max_distance <= 1024

// DW: a call's width rounded up to 32, 48, 64, 96 or 128 columns, which scores are summed over and
// results are kept for (in blocks of 32); a tile's rows in LDS step by a power of two.  (2 x 4096 x 16
// heads x 96 bf16, forward and backward: 1101 us with 96, 1230 with 128; 2 x 2048 x 8 x 40 f32: 408
// with 48, 444 with 64.)
constexpr int pitch(int dw) { return dw <= 32 ? 32 : dw <= 64 ? 64 : 128; }
constexpr int blocks(int dw) { return (dw + 31) / 32; }

// Rows of a tile that goes through LDS, and the waves a SIMD that the registers are cut to.  Two
// waves a SIMD hide each other's waits (2 x 4096 x 16 heads x 128 bf16, us: forward 387 with two, 572
// with one; key gradients and the rest of the backward pass 964 and 1120) as long as little spills:
// f32 backward at 128 columns keeps 400 registers (620 us with one wave, 1770 with two), f32 key
// gradients at 64 columns and bf16 ones at 128 with a bias keep 300 (214 / 260, 451 / 531).  64 rows
// halve the barriers of 32, but at 128 columns the key gradients have no registers for them (746 us
// with 32, 1939 with 64).  There the fragments' addresses are made again at every tile too (TIGHT:
// 34 spilled registers become 4, 722 -> 660 us; elsewhere it only costs instructions).
template <class T, int DW>
struct Shape {
    static constexpr bool F32 = Elem<T>::NP > 1;
    static constexpr int FWD_KEYS = F32 && DW > 32 ? 32 : 64, BWD_ROWS = F32 && DW > 32 ? 32 : DW > 64 ? 32 : 64;
    static constexpr int Q_KEYS = F32 && DW > 32 ? 32 : 64;
    static constexpr int FWD_WAVES = F32 && DW > 64 ? 1 : 2, Q_WAVES = FWD_WAVES;
    static constexpr int KV_WAVES = F32 && DW > 32 ? 1 : 2, KV_BIAS_WAVES = DW > (F32 ? 32 : 64) ? 1 : 2;
    static constexpr bool TIGHT = !F32 && DW > 64;
    static constexpr int SPLIT_WAVES = F32 && DW > 64 ? 1 : 2;
    // waves that share 32 rows in a small call (8 x 512 keys x 4 heads x 32 f32: 126 -> 78 us with 4;
    // 2 x 700 x 8 x 64 f32: 146 -> 99 with 2, 137 with 4, whose tiles leave one workgroup a CU)
    static constexpr int SHARE = F32 && DW > 64 ? 1 : DW > 32 ? 2 : 4;
};

struct Buckets {
    int n, far, both, exact, nthresh;
    int thresh[HREG_TOK_MAX_THRESH];
};

struct Args {
    const void *q, *k, *v, *out_r, *dout;
    void *out, *rest, *dq, *dk, *dv, *dbias;
    float *lse, *delta, *bins, *part, *sums;
    const int *q_len, *k_len;
    int *own;  // [B][H][tiles][waves]: whether the wave has a row with a 1 / sum of its own (bf16 with a bias)
    const uint8_t *key_mask;
    const void *bias;
    int64_t qs[3], ks[3], vs[3], os[3], dos[3], mask_sb;
    int B, Nq, Nk, H, Hk, D, causal, align_end, bias_f32, splits, groups, share_kv, tile_rows, group_tables, split_bytes;
    float scale;
    Buckets bk;
};

// the bucket of offset o = key position - query position: one for each offset up to `exact`,
// then steps of the logarithm, whose first offsets are bk.thresh
__device__ __forceinline__ int bucket_of(const Buckets &bk, int o) {
    const int n = bk.both ? (o < 0 ? -o : o) : (o < 0 ? -o : 0);
    int b = n;
    if (n >= bk.exact) {
        b = bk.exact;
        for (int t = 0; t < bk.nthresh; ++t) b += n >= bk.thresh[t];
    }
    return b + (bk.both && o > 0 ? bk.n / 2 : 0);
}

// a bucket's bias in units of log2.  A finite one stays finite: the type's lowest value leaves a key visible
// (a row that sees only such keys shares itself out among them), -infinity alone hides it.
__device__ __forceinline__ float bias_at(const Args &a, int b, int h) {
    const size_t at = (size_t)b * a.H + h;
    const float v = a.bias_f32 ? static_cast<const float *>(a.bias)[at] : (float)static_cast<const __bf16 *>(a.bias)[at];
    return fabsf(v) < INFINITY ? fminf(fmaxf(v * LOG2E, -FLT_MAX), FLT_MAX) : v;
}

// This workgroup's batch entry, head and tile.  Workgroups go round the 8 XCDs: each XCD takes whole
// heads, so that tiles that read the same keys share an L2, and walks them tile by tile over its
// heads, so that the long tiles of a causal call (callers number them first) all start early.
struct Where { int b, h, tile; };
__device__ __forceinline__ Where where(int batch, int heads, int tiles) {
    const int all = batch * heads;
    int head, tile;
    if (all % 8 == 0) {
        const int k = blockIdx.x >> 3, mine = all >> 3;
        head = (blockIdx.x & 7) * mine + k % mine;
        tile = k / mine;
    } else {
        const int n = xcd_block(blockIdx.x, gridDim.x);
        head = n / tiles;
        tile = n % tiles;
    }
    return {head / heads, head % heads, tile};
}

struct Span { int nq, nk, start; };  // valid rows, valid keys, position of query 0
__device__ __forceinline__ Span span_of(const Args &a, int b) {
    Span s;
    s.nq = a.q_len ? min(max(a.q_len[b], 0), a.Nq) : a.Nq;
    s.nk = a.k_len ? min(max(a.k_len[b], 0), a.Nk) : a.Nk;
    s.start = a.align_end ? s.nk - s.nq : 0;
    return s;
}

// Two [R][DP] tiles (keys and values, or queries and output gradients) on their way from global
// memory into LDS while the ones before are used: issue() starts, land() waits and makes them whole.
// bf16 goes straight into LDS (16 bytes a lane, two buffers, one barrier a tile); f32 goes through
// registers, where it is cut into its pieces (one buffer, two barriers).  Rows at or beyond `valid`,
// rows whose mask is 0 and columns at or beyond D are zero, whatever memory holds there; they are
// never read.
template <class T, int DP, int R>
struct Tiles {
    static constexpr int CPR = DP / 8, N = R * CPR / NT, NP = Elem<T>::NP, PLANE = R * DP, TILE = NP * PLANE;
    static constexpr bool DIRECT = NP == 1;
    static constexpr size_t BYTES = (size_t)(DIRECT ? 2 : 1) * 2 * TILE * 2;
    static_assert(R * CPR % NT == 0, "tile");
    uint16_t *lds;
    Chunk<T> cx[DIRECT ? 1 : N], cy[DIRECT ? 1 : N];
    int buf;  // the buffer that is used

    __device__ __forceinline__ const uint16_t *x() const { return lds + buf * 2 * TILE; }
    __device__ __forceinline__ const uint16_t *y() const { return x() + TILE; }

    __device__ __forceinline__ void init(uint16_t *at, int D) {
        lds = at;
        buf = DIRECT ? 1 : 0;
        if (DIRECT && D < DP) {  // the columns that no load writes
            for (int e = threadIdx.x; e < 4 * TILE / 8; e += NT) reinterpret_cast<u32x4_m *>(at)[e] = u32x4{0, 0, 0, 0};
            __syncthreads();
        }
    }
    __device__ __forceinline__ void issue(const T *px, int64_t ldx, const T *py, int64_t ldy, int row0, int valid, int D,
                                          const uint8_t *mask) {
        const bool whole = D == DP && row0 + R <= valid && !mask;  // (uniform)
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int id = threadIdx.x + u * NT, tr = id / CPR, r = row0 + tr;
            const int d = (DIRECT ? (id % CPR) ^ swz<DP>(tr) : id % CPR) * 8;
            const bool ok = whole || (r < valid && d < D && (!mask || mask[r]));
            if constexpr (DIRECT) {
                const uint16_t *to = lds + (buf ^ 1) * 2 * TILE + (u * NT + (threadIdx.x & ~63)) * 8;
                if (whole || ok) {
                    global_to_lds(px + (int64_t)r * ldx + d, to);
                    global_to_lds(py + (int64_t)r * ldy + d, to + TILE);
                }
            } else if (ok) {
                cx[u].load(px + (int64_t)r * ldx + d);
                cy[u].load(py + (int64_t)r * ldy + d);
            } else {
                cx[u].zero();
                cy[u].zero();
            }
        }
    }
    __device__ __forceinline__ void land(int row0, int valid, const uint8_t *mask) {
        if constexpr (DIRECT) {
            buf ^= 1;
            __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's rows are there
            __syncthreads();                     // every wave's are, and the other buffer is free
            if (mask || row0 + R > valid) {
                uint16_t *to = lds + buf * 2 * TILE;
#pragma unroll
                for (int u = 0; u < N; ++u) {
                    const int id = threadIdx.x + u * NT, r = row0 + id / CPR;
                    if (r >= valid || (mask && !mask[r])) {
                        *reinterpret_cast<u32x4_m *>(to + id * 8) = u32x4{0, 0, 0, 0};
                        *reinterpret_cast<u32x4_m *>(to + TILE + id * 8) = u32x4{0, 0, 0, 0};
                    }
                }
                __syncthreads();
            }
        } else {
            __syncthreads();
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const int id = threadIdx.x + u * NT, at = tile_at<DP>(id / CPR, id % CPR);
                bf16x8 p[NP];
                cx[u].pieces(p);
#pragma unroll
                for (int s = 0; s < NP; ++s) *reinterpret_cast<u32x4_m *>(lds + s * PLANE + at) = __builtin_bit_cast(u32x4, p[s]);
                cy[u].pieces(p);
#pragma unroll
                for (int s = 0; s < NP; ++s)
                    *reinterpret_cast<u32x4_m *>(lds + TILE + s * PLANE + at) = __builtin_bit_cast(u32x4, p[s]);
            }
            __syncthreads();
        }
    }
};

// one row's pieces as an operand with the row in lane & 31, straight from global memory
template <class T, int DW>
__device__ __forceinline__ void load_row(const T *row, bool ok, int D, int lane,
                                         bf16x8 (&f)[DW / 16][Elem<T>::NP], bool negate = false) {
#pragma unroll
    for (int c = 0; c < DW / 16; ++c) {
        const int d = 16 * c + 8 * (lane >> 5);
        Chunk<T> x;
        if (ok && d < D) x.load(row + d);
        else x.zero();
        if (negate) x.negate();
        x.pieces(f[c]);
    }
}

// What the backward pass makes a row's probabilities from.  bf16: p = exp2(s - log2 of the sum).
// f32: p = exp2(s - m) / sum with the forward pass's own m and 1 / sum, because the logarithm of a
// sum near 2^10 is rounded by 2^-21 and that error would be common to a row: it does not cancel in
// the bias gradient's sums (6 times their error).  bf16 with a bias has them too in rows with |m| >= LARGE
// (the others 1 for 1 / sum): m + log2(sum) is rounded by 2^-24 of m, and with a bias of -1e9 or the type's
// lowest value on all that a row sees nothing of the sum is left.  A row without keys: p = exp2(s - inf) = 0.
constexpr float LARGE = 4096.f;
struct RowSum { float ref, inv; };
template <class T>
__device__ __forceinline__ void save_sum(const Args &a, size_t row, bool any, float m, float l, float inv) {
    const bool sum = Elem<T>::NP == 1 && !(a.bias && fabsf(m) >= LARGE);  // log2 of the sum, NaN among them
    a.lse[row] = !any ? INFINITY : sum ? m + __builtin_amdgcn_logf(l) : m;
    if (Elem<T>::NP > 1 || a.bias) a.lse[(size_t)a.B * a.H * a.Nq + row] = sum || !any ? 1.f : inv;
}
template <class T, bool BIAS>
__device__ __forceinline__ RowSum row_sum_of(const Args &a, size_t row, bool ok) {
    RowSum r{INFINITY, 1.f};
    if (!ok) return r;
    r.ref = a.lse[row];
    if constexpr (Elem<T>::NP > 1 || BIAS) r.inv = a.lse[(size_t)a.B * a.H * a.Nq + row];
    return r;
}
template <bool OWN>
__device__ __forceinline__ float prob(float x, float inv) {  // x = s - ref
    const float p = __builtin_amdgcn_exp2f(x);
    return OWN ? p * inv : p;
}

// ---------------------------------------------------------------------- forward --

// One head's bias over the offsets -far - PAD .. far + PAD, in units of log2, in LDS.  A 32 x 32
// tile of scores touches 63 offsets: if all lie beyond far it takes one value, else its offsets are
// inside the table without clamping (lane and register steps are constant: paired LDS reads).
constexpr int PAD = 64;
__device__ __forceinline__ int table_size(int far) { return 2 * (far + PAD) + 1; }
__device__ __forceinline__ void fill_table(const Args &a, float *tab, int h) {
    const int far = a.bk.far;
    for (int o = threadIdx.x; o < table_size(far); o += NT)
        tab[o] = bias_at(a, bucket_of(a.bk, min(max(o - far - PAD, -far), far)), h);
}

// Scores of 32 keys (rows) against the wave's 32 queries (columns) in units of log2: s = s * scale2 +
// bias.  base = first key - first query's position, kpos = first key - this lane's query's.
__device__ __forceinline__ void add_bias(f32x16 &s, float scale2, const float *tab, int far, int base, int kpos, int half) {
    if (base - 31 >= far || base + 31 <= -far) {
        const float b = tab[base < 0 ? 0 : 2 * (far + PAD)];
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], scale2, b);
    } else {
        const float *t = tab + (kpos + 4 * half + far + PAD);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], scale2, t[8 * (r >> 2) + (r & 3)]);
    }
}

// LDS of a kernel whose KW waves share rows: its tiles, then MATS joined matrices of the sharing
// waves in the same place
template <class T, int DP, int R, int KW, int MATS>
constexpr size_t area() {
    constexpr size_t tiles = Tiles<T, DP, R>::BYTES, join = (size_t)(4 / KW) * (KW - 1) * MATS * 32 * (DP + 4) * 4;
    return tiles > join ? tiles : join;
}

// Which of 32 keys the lane's query sees, bit 8 (r >> 2) + (r & 3) for register r of its half.  kpos =
// position of the first key - the query's; seen: bit k = key k exists and is not masked
__device__ __forceinline__ uint32_t visible(const Args &a, int kpos, uint32_t seen, int half) {
    if (a.causal) {  // the keys up to the query's own position
        const int n = min(max(1 - kpos, 0), 32);
        seen &= n == 32 ? ~0u : (1u << n) - 1;
    }
    return seen >> (4 * half);
}
// registers whose bit is 0 become v (only on the edge tiles, hence the empty asm: without it the
// compiler makes the selections everywhere)
__device__ __forceinline__ void keep_only(f32x16 &s, uint32_t bits, float v) {
    asm volatile("");
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = bits >> (8 * (r >> 2) + (r & 3)) & 1 ? s[r] : v;
}
__device__ __forceinline__ uint32_t seen_keys(int krow, int nk, const uint8_t *mask) {
    if (!mask) return krow + 32 <= nk ? ~0u : krow >= nk ? 0u : (1u << (nk - krow)) - 1;
    const int k = krow + (threadIdx.x & 31);
    return (uint32_t)__ballot(k < nk && mask[min(k, nk - 1)]);
}

// acc += (32 rows of a tile)^T x, x in the lane's two fragments of 16 rows.  f32: each 32 rows' sum is
// made on its own and then added, rounded to nearest: the matrix cores round down each time they add to
// a result (4 x 517 keys x 40: out and its gradients 4.5e-7 to 4.9e-7 off otherwise, 2.6e-7 to 3.1e-7
// with this and the row sums made by tiles).
template <int DP, int ND, int NP, int NB>
__device__ __forceinline__ void add_rows(f32x16 (&acc)[ND], const uint16_t *tile, int plane, int row, const Lane<DP> &at,
                                         const bf16x8 (&x)[2][NB]) {
    if constexpr (NP == 1) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                bf16x8 f[NP];
                col_frag<DP>(tile, plane, row + 16 * c, 32 * d, at, f);
                mma(acc[d], f, x[c]);
            }
    } else {
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            f32x16 part = zero16();
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                bf16x8 f[NP];
                col_frag<DP>(tile, plane, row + 16 * c, 32 * d, at, f);
                mma(part, f, x[c]);
            }
            acc[d] += part;
        }
    }
}

// Whether the workgroup's first query sees at most FEW_KEYS keys (the same in every wave), of which
// `first` exist for it.  Where a bias gradient is to come, bf16 rows take 16 bits of p there: few keys
// average little of p's rounding to 8 away, and its error in out, through D = do . o, is common to a row's
// ds (3 x 237 queries x 32 heads x 72: 9 keys 3.1e-3 -> 1.6e-3 off, of which 1.6e-3 is its own rounding, 60
// keys 2.3e-3 -> 1.6e-3; 120 keys are at 1.9e-3 without).  It is asked of the keys that are seen, not of those
// that the tensors have room for, so that padding does not change it.
__device__ __forceinline__ bool few_keys(int first, const uint8_t *mask, int lane) {
    if (first <= FEW_KEYS) return true;
    if (!mask) return false;
    int n = 0;
    for (int k0 = 0; k0 < first && n <= FEW_KEYS; k0 += 256)
#pragma unroll
        for (int u = 0; u < 256; u += 64) {
            const int k = k0 + u + lane;
            n += __popcll(__ballot(k < first && mask[min(k, first - 1)]));
        }
    return n <= FEW_KEYS;
}

// one row's result: sums over its keys, written as out (and what training keeps)
template <class T>
__device__ __forceinline__ void finish_row(const Args &a, int b, int i, int h, int col, const f32x4 &o, float m, float l) {
    const bool any = l != 0.f;  // (a NaN sum stays NaN)
    const float inv = any ? 1.f / l : 0.f;
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = any ? o[e] * inv : 0.f;
    store4(static_cast<T *>(a.out) + b * a.os[0] + (int64_t)i * a.os[1] + h * a.os[2] + col, x[0], x[1], x[2], x[3]);
    if constexpr (Elem<T>::NP == 1) {
        if (a.rest)
            store4(static_cast<T *>(a.rest) + (((int64_t)b * a.Nq + i) * a.H + h) * a.D + col, x[0] - (float)(T)x[0],
                   x[1] - (float)(T)x[1], x[2] - (float)(T)x[2], x[3] - (float)(T)x[3]);
    }
    if (a.lse && col == 0) save_sum<T>(a, ((size_t)b * a.H + h) * a.Nq + i, any, m, l, inv);
}

// 128 rows of one head, 32 a wave: the columns of its scores are its queries.  One pass over the keys
// with the running maximum and sum; a row's rescaling is skipped while no row of the wave finds a
// larger score.  bf16 at 64 columns is bound by the exponentials and sums (four vector instructions
// and a quarter-rate exponential a score against 16 cycles of matrix product), at 128 columns by both
// and by the waits between them; f32 by its six products.  2 x 4096 x 16 heads: 128 columns 302 us
// (910 TFLOP/s), 64 columns 183 us (750); f32 2 x 2048 x 8 x 64: 116 us (148).
template <class T, int DW, int KT, bool BIAS, int PP>
__device__ __forceinline__ void fwd_rows(const Args &a) {
    constexpr int NP = Elem<T>::NP, DP = pitch(DW), ND = blocks(DW), MT = KT / 32, PLANE = KT * DP;
    extern __shared__ __attribute__((aligned(16))) uint16_t lds[];
    typedef Tiles<T, DP, KT> KV;
    float *tab = reinterpret_cast<float *>(reinterpret_cast<char *>(lds) + KV::BYTES);
    const int tiles = (a.Nq + ROWS - 1) / ROWS;
    const Where w = where(a.B, a.H, tiles);
    const Span sp = span_of(a, w.b);
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x >> 6;
    const int q0 = (tiles - 1 - w.tile) * ROWS, i = q0 + 32 * wave + (lane & 31);
    const int hk = w.h / (a.H / a.Hk);
    const T *K = static_cast<const T *>(a.k) + w.b * a.ks[0] + hk * a.ks[2];
    const T *V = static_cast<const T *>(a.v) + w.b * a.vs[0] + hk * a.vs[2];
    const uint8_t *mask = a.key_mask ? a.key_mask + w.b * a.mask_sb : nullptr;
    if constexpr (BIAS) fill_table(a, tab, w.h);

    // without a bias scores stay as the products give them and their running maximum with them
    // (q takes a negative scale's sign): one fused multiply-add before each exponential
    bf16x8 qf[DW / 16][NP];
    load_row<T, DW>(static_cast<const T *>(a.q) + w.b * a.qs[0] + (int64_t)i * a.qs[1] + w.h * a.qs[2], i < sp.nq, a.D,
                    lane, qf, a.scale < 0.f);
    const float scale2 = fmaxf(fabsf(a.scale) * LOG2E, 1e-37f), unit = BIAS ? 1.f : scale2;
    f32x16 acc[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] = zero16();
    float m = -INFINITY, l = 0.f;

    // keys that some row of the workgroup sees
    const int last = min(q0 + ROWS, sp.nq) - 1;
    const int kend = last < q0 ? 0 : a.causal ? min(sp.nk, max(last + sp.start + 1, 0)) : sp.nk;
    KV kv;
    kv.init(lds, a.D);
    Lane<DP> at(lane);
    if (kend > 0) kv.issue(K, a.ks[1], V, a.vs[1], 0, sp.nk, a.D, mask);
    for (int j0 = 0; j0 < kend; j0 += KT) {
        kv.land(j0, sp.nk, mask);
        const uint16_t *kt = kv.x(), *vt = kv.y();
        if (j0 + KT < kend) kv.issue(K, a.ks[1], V, a.vs[1], j0 + KT, sp.nk, a.D, mask);
        const int qw = q0 + 32 * wave + sp.start;  // position of the wave's first query
        if (a.causal && j0 > qw + 32 - 1) continue;
        const bool edge = mask || j0 + KT > sp.nk || (a.causal && j0 + KT - 1 > qw);
        f32x16 s[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) s[t] = zero16();
#pragma unroll
        for (int c = 0; c < DW / 16; ++c)
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                bf16x8 kf[NP];
                row_frag<DP>(kt, PLANE, 32 * t, c, at, kf);
                mma(s[t], kf, qf[c]);
            }
        if constexpr (NP == 1) interleave<MT * DW / 16, 1, 2>();
        const int kpos = j0 - (i + sp.start);
        float top = m;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            if constexpr (BIAS) add_bias(s[t], scale2, tab, a.bk.far, j0 + 32 * t - qw, kpos + 32 * t, half);
            if (edge) keep_only(s[t], visible(a, kpos + 32 * t, seen_keys(j0 + 32 * t, sp.nk, mask), half), -INFINITY);
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, s[t][r]);
        }
        top = fmaxf(top, __shfl_xor(top, 32));
        const float ref = top == -INFINITY ? 0.f : top * unit;  // a row without a key so far keeps sums of 0
        if (__any(top != m)) {
            const float shrink = __builtin_amdgcn_exp2f(__builtin_fmaf(m, unit, -ref));
            l *= shrink;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[d][r] *= shrink;
            m = top;
        }
        float sum = 0.f;  // (a tile's on its own first: adding thousands of keys one by one rounds as often)
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[t][r] = __builtin_amdgcn_exp2f(BIAS ? s[t][r] - ref : __builtin_fmaf(s[t][r], unit, -ref));
                sum += s[t][r];
            }
        l += sum;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            bf16x8 pf[2][PP];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float p[8];
#pragma unroll
                for (int r = 0; r < 8; ++r) p[r] = s[t][8 * c + r];
                to_pieces<PP>(p, pf[c]);
            }
            add_rows<DP, ND, NP>(acc, vt, PLANE, 32 * t, at, pf);
        }
        if constexpr (NP == 1) interleave<MT * 2 * ND, 2, 4>();
    }
    l += __shfl_xor(l, 32);
    if (i >= a.Nq) return;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int col = 32 * d + 2 * r + 4 * half;
            if (col < a.D)
                finish_row<T>(a, w.b, i, w.h, col, f32x4{acc[d][r], acc[d][r + 1], acc[d][r + 2], acc[d][r + 3]}, m * unit,
                              i < sp.nq ? l : 0.f);
        }
}

// PP is chosen here, by the keys that the workgroup sees
template <class T, int DW, int KT, bool BIAS>
__global__ __launch_bounds__(NT, (Shape<T, DW>::FWD_WAVES)) void attn_fwd(Args a) {
    constexpr int NP = Elem<T>::NP;
    if constexpr (BIAS && NP == 1) {
        const int tiles = (a.Nq + ROWS - 1) / ROWS;
        const Where w = where(a.B, a.H, tiles);
        const Span sp = span_of(a, w.b);
        const int seen = a.causal ? min(sp.nk, (tiles - 1 - w.tile) * ROWS + sp.start + 1) : sp.nk;  // by its first query
        if (a.rest && few_keys(seen, a.key_mask ? a.key_mask + w.b * a.mask_sb : nullptr, threadIdx.x & 63)) {
            fwd_rows<T, DW, KT, BIAS, 2>(a);
            return;
        }
    }
    fwd_rows<T, DW, KT, BIAS, NP>(a);
}

// ------------------------------------------------------- forward, keys split --

// Few rows, many keys: a workgroup takes 32 rows of one key head (row r is token r / G, head r % G
// of the group, so a token's G heads share every key that is read) and one run of the keys; its
// four waves take 32 keys each in turn and join in LDS, the runs join in attn_join.  Each wave stages
// its own keys, then its own values, in its own LDS, without a barrier; the next tile is on its way
// in registers.  Bound by the bytes of the cache: 8 x up to 32768 keys x 8 key heads x 128 bf16, 805 MB:
// 153 us (5.3 TB/s; a large copy reaches 4.7).  So bf16 keeps 16 bits of p: its second product is 1 % (2 x
// 16384 keys x 64 heads on 8: 36.7 -> 37.0 us), and out is as near as its own rounding (error 2.2e-3 -> 1.7e-3).
template <class T, int DP>
struct WaveStage {
    static constexpr int CPR = DP / 8, N = 32 * CPR / 64, NP = Elem<T>::NP, PLANE = 32 * DP;
    Chunk<T> c[N];
    __device__ __forceinline__ void load(const T *base, int64_t ld, int row0, int valid, int D, const uint8_t *mask, int lane) {
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int id = lane + u * 64, r = row0 + id / CPR, d = id % CPR * 8;
            if (r < valid && d < D && (!mask || mask[r])) c[u].load(base + (int64_t)r * ld + d);
            else c[u].zero();
        }
    }
    __device__ __forceinline__ void store(uint16_t *t, int lane) const {
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int id = lane + u * 64;
            bf16x8 p[NP];
            c[u].pieces(p);
#pragma unroll
            for (int s = 0; s < NP; ++s)
                *reinterpret_cast<u32x4_m *>(t + s * PLANE + tile_at<DP>(id / CPR, id % CPR)) = __builtin_bit_cast(u32x4, p[s]);
        }
    }
};

template <class T, int DW, bool BIAS>
__global__ __launch_bounds__(NT, (Shape<T, DW>::SPLIT_WAVES)) void attn_split(Args a) {
    constexpr int NP = Elem<T>::NP, PP = NP == 1 ? 2 : NP, DP = pitch(DW), ND = blocks(DW), PLANE = 32 * DP;
    constexpr int OLD = DP + 4;  // a joined row's step in LDS
    extern __shared__ __attribute__((aligned(16))) uint16_t lds[];
    __shared__ float ml[4][2][32];
    const int G = a.H / a.Hk, R = a.Nq * G, tiles = (R + 31) / 32;
    const Where w = where(a.B, a.Hk, tiles * a.splits);  // the splits of a tile are neighbours of its keys' others
    const int split = w.tile % a.splits, tile = w.tile / a.splits;
    const Span sp = span_of(a, w.b);
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x >> 6;
    const int r = tile * 32 + (lane & 31), i = r / G, h = w.h * G + r % G;
    const bool there = r < R && i < sp.nq;
    const T *K = static_cast<const T *>(a.k) + w.b * a.ks[0] + w.h * a.ks[2];
    const T *V = static_cast<const T *>(a.v) + w.b * a.vs[0] + w.h * a.vs[2];
    const uint8_t *mask = a.key_mask ? a.key_mask + w.b * a.mask_sb : nullptr;
    uint16_t *buf = lds + wave * NP * PLANE;
    // the bias of the group's heads: their tables in LDS, or (many heads) bucket by bucket from memory
    float left = 0.f, right = 0.f;  // beyond the far offsets
    const float *tab = nullptr;
    if constexpr (BIAS) {
        const int W = table_size(a.bk.far), hb = r < R ? h : w.h * G;
        if (a.group_tables) {
            float *at = reinterpret_cast<float *>(reinterpret_cast<char *>(lds) + a.split_bytes);
            for (int g = 0; g < G; ++g) fill_table(a, at + g * W, w.h * G + g);
            tab = at + (hb - w.h * G) * W + a.bk.far + PAD;
        }
        left = bias_at(a, bucket_of(a.bk, -a.bk.far), hb);
        right = bias_at(a, bucket_of(a.bk, a.bk.far), hb);
        __syncthreads();
    }
    bf16x8 qf[DW / 16][NP];
    load_row<T, DW>(static_cast<const T *>(a.q) + w.b * a.qs[0] + (int64_t)i * a.qs[1] + h * a.qs[2], there, a.D, lane, qf);
    const float scale2 = a.scale * LOG2E;
    f32x16 acc[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] = zero16();
    float m = -INFINITY, l = 0.f;

    // keys that some row of the tile sees, in `splits` runs of whole 128
    const int first_pos = tile * 32 / G + sp.start, last_i = min((tile * 32 + 31) / G, sp.nq - 1);
    const int kend = tile * 32 / G >= sp.nq ? 0 : a.causal ? min(sp.nk, max(last_i + sp.start + 1, 0)) : sp.nk;
    const int run = ((kend + a.splits - 1) / a.splits + 127) / 128 * 128;
    const int j_end = min(kend, (split + 1) * run);
    int j0 = split * run + 32 * wave;
    const Lane<DP> at(lane);
    WaveStage<T, DP> sk, sv;
    if (j0 < j_end) {
        sk.load(K, a.ks[1], j0, sp.nk, a.D, mask, lane);
        sv.load(V, a.vs[1], j0, sp.nk, a.D, mask, lane);
    }
    for (; j0 < j_end; j0 += 128) {
        sk.store(buf, lane);
        if (j0 + 128 < j_end) sk.load(K, a.ks[1], j0 + 128, sp.nk, a.D, mask, lane);
        wave_sync();
        f32x16 s = zero16();
#pragma unroll
        for (int c = 0; c < DW / 16; ++c) {
            bf16x8 kf[NP];
            row_frag<DP>(buf, PLANE, 0, c, at, kf);
            mma(s, kf, qf[c]);
        }
        const int kpos = j0 - (i + sp.start);
        const bool edge = mask || j0 + 32 > sp.nk || (a.causal && j0 + 31 > first_pos);
        const bool near = BIAS && __any(kpos + 31 > -a.bk.far && kpos < a.bk.far);
        float top = m;
        if (!near) {
            const float bias = kpos < 0 ? left : right;
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = BIAS ? __builtin_fmaf(s[e], scale2, bias) : s[e] * scale2;
        } else if (a.group_tables) {
            const float *t = tab + min(max(kpos, -a.bk.far - PAD), a.bk.far + PAD - 31) + 4 * half;
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = __builtin_fmaf(s[e], scale2, t[8 * (e >> 2) + (e & 3)]);
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int o = min(max(kpos + 8 * (e >> 2) + 4 * half + (e & 3), -a.bk.far), a.bk.far);
                s[e] = __builtin_fmaf(s[e], scale2, bias_at(a, bucket_of(a.bk, o), r < R ? h : w.h * G));
            }
        }
        if (edge) keep_only(s, visible(a, kpos, seen_keys(j0, sp.nk, mask), half), -INFINITY);
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, s[e]);
        top = fmaxf(top, __shfl_xor(top, 32));
        const float ref = top == -INFINITY ? 0.f : top;
        if (__any(top != m)) {
            const float shrink = __builtin_amdgcn_exp2f(m - ref);
            l *= shrink;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[d][e] *= shrink;
            m = top;
        }
        wave_sync();  // the keys are read
        sv.store(buf, lane);
        if (j0 + 128 < j_end) sv.load(V, a.vs[1], j0 + 128, sp.nk, a.D, mask, lane);
        wave_sync();
        float sum = 0.f;
        bf16x8 pf[2][PP];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                p[e] = __builtin_amdgcn_exp2f(s[8 * c + e] - ref);
                sum += p[e];
            }
            to_pieces<PP>(p, pf[c]);
        }
        l += sum;
        add_rows<DP, ND, NP>(acc, buf, PLANE, 0, at, pf);
        wave_sync();  // the values are read
    }

    // join the waves: every one scales its sums to the common maximum, four rows' parts are added
    l += __shfl_xor(l, 32);
    if (!there) m = -INFINITY, l = 0.f;
    if (half == 0) ml[wave][0][lane] = m, ml[wave][1][lane] = l;
    __syncthreads();
    float *part = reinterpret_cast<float *>(lds);  // [wave][32][OLD]
    {
        const int q = lane & 31;
        const float all = fmaxf(fmaxf(ml[0][0][q], ml[1][0][q]), fmaxf(ml[2][0][q], ml[3][0][q]));
        const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - all);
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                *reinterpret_cast<f32x4_m *>(part + (wave * 32 + q) * OLD + 32 * d + 2 * e + 4 * half) =
                    f32x4{acc[d][e] * f, acc[d][e + 1] * f, acc[d][e + 2] * f, acc[d][e + 3] * f};
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 32 * DP / 4; e += NT) {
        const int q = e / (DP / 4), col = e % (DP / 4) * 4, rr = tile * 32 + q;
        if (rr >= R || col >= a.D) continue;
        const float all = fmaxf(fmaxf(ml[0][0][q], ml[1][0][q]), fmaxf(ml[2][0][q], ml[3][0][q]));
        f32x4 o{0.f, 0.f, 0.f, 0.f};
        float sum = 0.f;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            o += *reinterpret_cast<const f32x4_m *>(part + (v * 32 + q) * OLD + col);
            // (no maximum: the sum is 0 where the wave's keys are none, NaN where its scores all are)
            sum += ml[v][0][q] == -INFINITY ? ml[v][1][q] : ml[v][1][q] * __builtin_amdgcn_exp2f(ml[v][0][q] - all);
        }
        if (a.splits == 1) {
            finish_row<T>(a, w.b, rr / G, w.h * G + rr % G, col, o, all, sum);
        } else {
            const size_t at = (((size_t)w.b * a.Hk + w.h) * R + rr) * a.splits + split;
            *reinterpret_cast<f32x4_m *>(a.part + at * a.D + col) = o;
            if (col == 0) a.sums[2 * at] = all, a.sums[2 * at + 1] = sum;
        }
    }
}

// out of the runs' partial results: 32 lanes a row, runs in order
template <class T>
__global__ __launch_bounds__(NT) void attn_join(Args a) {
    const int G = a.H / a.Hk, R = a.Nq * G, lane = threadIdx.x % 32, col = lane * 4;
    const int64_t row = (int64_t)blockIdx.x * (NT / 32) + threadIdx.x / 32;
    if (row >= (int64_t)a.B * a.Hk * R) return;
    const float *sums = a.sums + 2 * row * a.splits, *part = a.part + row * a.splits * a.D + min(col, a.D - 4);
    float all = -INFINITY;
    for (int s = lane; s < a.splits; s += 32) all = fmaxf(all, sums[2 * s]);
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) all = fmaxf(all, __shfl_xor(all, k));
    f32x4 o{0.f, 0.f, 0.f, 0.f};
    float sum = 0.f;
    for (int s0 = 0; s0 < a.splits; s0 += 32) {
        float f = 0.f, l = 0.f;  // lane s: run s0 + s
        if (s0 + lane < a.splits) {
            const float m = sums[2 * (s0 + lane)];
            l = sums[2 * (s0 + lane) + 1];  // (no maximum: 0, or NaN where all scores are)
            f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - all);
            if (m != -INFINITY) l *= f;
        }
        const int n = min(a.splits - s0, 32);
#pragma unroll 4
        for (int s = 0; s < n; ++s) {
            o += *reinterpret_cast<const f32x4_m *>(part + (int64_t)(s0 + s) * a.D) * __shfl(f, (threadIdx.x & 32) + s);
            sum += __shfl(l, (threadIdx.x & 32) + s);
        }
    }
    const int r = row % R, hk = row / R % a.Hk, b = row / R / a.Hk;
    if (col < a.D) finish_row<T>(a, b, r / G, hk * G + r % G, col, o, all, sum);
}

// ---------------------------------------------------------------------- backward --

// D_i = do_i . o_i of the lane's row, half of it each in lanes l and l + 32.  o and what it lost in
// rounding (bf16): that error would be common to a row's ds.
template <class T, int DW>
__device__ __forceinline__ float row_dot(const Args &a, int b, int h, int i, bool ok, int lane) {
    const T *x = static_cast<const T *>(a.dout) + b * a.dos[0] + (int64_t)i * a.dos[1] + h * a.dos[2];
    const T *y = static_cast<const T *>(a.out_r) + b * a.os[0] + (int64_t)i * a.os[1] + h * a.os[2];
    const T *z = static_cast<const T *>(a.rest) + (((int64_t)b * a.Nq + i) * a.H + h) * a.D;
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < DW / 16; ++c) {
        const int d = 16 * c + 8 * (lane >> 5);
        if (!ok || d >= a.D) continue;
        Chunk<T> u, v;
        u.load(x + d);
        v.load(y + d);
        s += u.dot(v);
        if (a.rest) {
            v.load(z + d);
            s += u.dot(v);
        }
    }
    return s + __shfl_xor(s, 32);
}

// the same for a call that wants no query gradients: delta[b][h][i], 32 rows a wave
template <class T, int DW>
__global__ __launch_bounds__(NT) void attn_delta(Args a) {
    const int64_t rows = (int64_t)a.B * a.H * a.Nq, row = (int64_t)blockIdx.x * (NT / 2) + threadIdx.x / 64 * 32 + threadIdx.x % 32;
    const bool in = row < rows;
    const int i = in ? row % a.Nq : 0, h = in ? row / a.Nq % a.H : 0, b = in ? row / a.Nq / a.H : 0;
    const float s = row_dot<T, DW>(a, b, h, i, in && i < span_of(a, b).nq, threadIdx.x & 63);
    if (in && threadIdx.x % 64 < 32) a.delta[row] = s;
}

// The pieces that p and ds go into their products in.  A bf16 call that is too small to fill the card
// keeps 16 bits of them instead of 8: its products are not what it waits for, and few values
// average less of the rounding away (gradients 1.05 instead of 1.45 times as far from the exact ones
// as their own rounding).
template <class T, int KW>
constexpr int prob_pieces() { return Elem<T>::NP == 1 && KW > 1 ? 2 : Elem<T>::NP; }

// dk, dv of 128 keys: every wave keeps 32 keys and walks all rows of all heads that share them, so
// the sums over a group need no second pass and have one order.  Where that leaves too few
// workgroups each walks one of a.groups parts of the group, and sum_group adds the parts' f32 results.
// KW waves share 32 keys, each taking every KW-th 32 rows (a small call has few keys to give a wave
// of its own): their sums join in LDS, in wave order.  Scores are straight (rows are queries), so p
// and ds are operands of the second products as they stand.  Bound by the matrix products and the
// waits for their operands: 256 registers leave no room to read far ahead.  2 x 4096 x 16 heads x 128
// bf16: 580 us (950 TFLOP/s); 64 columns 320 us (860); f32 2 x 2048 x 8 x 64: 215 us (160).
// OWN: probabilities are multiplied by the rows' 1 / sum.
template <class T, int DW, int QT, int KW, bool BIAS, bool OWN>
__device__ __forceinline__ void bwd_kv_rows(const Args &a) {
    constexpr int NP = Elem<T>::NP, PP = prob_pieces<T, KW>(), DP = pitch(DW), ND = blocks(DW), PLANE = QT * DP, ROWS = 128 / KW;
    static_assert(QT % (32 * KW) == 0, "tile");
    extern __shared__ __attribute__((aligned(16))) uint16_t lds[];
    typedef Tiles<T, DP, QT> QD;
    float *lt = reinterpret_cast<float *>(reinterpret_cast<char *>(lds) + area<T, DP, QT, KW, 2>()), *et = lt + QT, *it = et + QT, *tab = lt + 6 * QT;
    const Where w0 = where(a.B, a.Hk * a.groups, (a.Nk + ROWS - 1) / ROWS);
    const Where w{w0.b, w0.h / a.groups, w0.tile};
    const Span sp = span_of(a, w.b);
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x >> 6;
    const int share = wave % KW, k0 = w.tile * ROWS + 32 * (wave / KW), j = k0 + (lane & 31);
    const uint8_t *mask = a.key_mask ? a.key_mask + w.b * a.mask_sb : nullptr;
    const bool ok = j < sp.nk && (!mask || mask[j]);
    bf16x8 kf[DW / 16][NP], vf[DW / 16][NP];
    load_row<T, DW>(static_cast<const T *>(a.k) + w.b * a.ks[0] + (int64_t)j * a.ks[1] + w.h * a.ks[2], ok, a.D, lane, kf);
    load_row<T, DW>(static_cast<const T *>(a.v) + w.b * a.vs[0] + (int64_t)j * a.vs[1] + w.h * a.vs[2], ok, a.D, lane, vf);
    f32x16 dk[ND], dv[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) dk[d] = dv[d] = zero16();
    const float scale2 = a.scale * LOG2E;
    const int first = a.causal ? max(w.tile * ROWS - sp.start, 0) : 0;  // rows before see no key of the tile
    const int G = a.H / a.Hk;
    QD qd;
    qd.init(lds, a.D);
    Lane<DP> at(lane);
    const int g0 = w0.h % a.groups * (G / a.groups);
    if (w.tile * ROWS < sp.nk)
        for (int g = g0; g < g0 + G / a.groups; ++g) {
            const int h = w.h * G + g;
            const T *Q = static_cast<const T *>(a.q) + w.b * a.qs[0] + h * a.qs[2];
            const T *dO = static_cast<const T *>(a.dout) + w.b * a.dos[0] + h * a.dos[2];
            const size_t row0 = ((size_t)w.b * a.H + h) * a.Nq;
            __syncthreads();  // the last head's table and rows are read
            if constexpr (BIAS) fill_table(a, tab, h);
            if (first < sp.nq) qd.issue(Q, a.qs[1], dO, a.dos[1], first, sp.nq, a.D, nullptr);
            // the rows' sums and dots go through registers into one of two buffers, a tile ahead: a
            // load that is waited for at each tile costs as much as the tile
            RowSum rs{INFINITY, 1.f};
            float dot = 0.f;
            const bool mine = threadIdx.x < QT;
            if (mine && first < sp.nq) {
                const int i = first + threadIdx.x;
                rs = row_sum_of<T, BIAS>(a, row0 + i, i < sp.nq);
                lt[threadIdx.x] = -rs.ref;
                it[threadIdx.x] = rs.inv;
                et[threadIdx.x] = i < sp.nq ? a.delta[row0 + i] : 0.f;
            }
            for (int i0 = first, now = 0; i0 < sp.nq; i0 += QT, now ^= 3 * QT) {
                qd.land(i0, sp.nq, nullptr);
                const uint16_t *qt = qd.x(), *dt = qd.y();
                if constexpr (Shape<T, DW>::TIGHT) at.opaque();
                if (i0 + QT < sp.nq) {
                    qd.issue(Q, a.qs[1], dO, a.dos[1], i0 + QT, sp.nq, a.D, nullptr);
                    const int i = i0 + QT + threadIdx.x;
                    rs = row_sum_of<T, BIAS>(a, row0 + i, mine && i < sp.nq);
                    dot = mine && i < sp.nq ? a.delta[row0 + i] : 0.f;
                }
#pragma unroll
                for (int u = 0; u < QT / 32 / KW; ++u) {
                    const int t = u * KW + share;
                    const int p0 = i0 + 32 * t + sp.start;  // position of the first query
                    if (i0 + 32 * t >= sp.nq || (a.causal && p0 + 31 < k0)) continue;
                    const bool edge = a.causal && p0 < k0 + 31;
                    const bool near = BIAS && !(k0 - p0 - 31 >= a.bk.far || k0 - p0 + 31 <= -a.bk.far);
                    const float b = BIAS ? tab[k0 < p0 ? 0 : 2 * (a.bk.far + PAD)] : 0.f;
                    f32x16 s = zero16(), dp = zero16();
#pragma unroll
                    for (int c = 0; c < DW / 16; ++c) {
                        bf16x8 f[NP];
                        row_frag<DP>(qt, PLANE, 32 * t, c, at, f);
                        mma(s, f, kf[c]);
                        row_frag<DP>(dt, PLANE, 32 * t, c, at, f);
                        mma(dp, f, vf[c]);
                    }
#pragma unroll
                    for (int r0 = 0; r0 < 16; r0 += 4) {  // four rows' sums and dots at once
                        const int row = now + 32 * t + 2 * r0 + 4 * half;
                        const f32x4 ref = *reinterpret_cast<const f32x4_m *>(lt + row), dot4 = *reinterpret_cast<const f32x4_m *>(et + row);
                        f32x4 inv{1.f, 1.f, 1.f, 1.f};
                        if constexpr (OWN) inv = *reinterpret_cast<const f32x4_m *>(it + row);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int r = r0 + e;
                            float x;
                            if constexpr (BIAS) {
                                const float w = near ? tab[j - p0 + a.bk.far + PAD - (2 * r0 + 4 * half + e)] : b;
                                x = __builtin_fmaf(s[r], scale2, w) + ref[e];
                            } else {
                                x = __builtin_fmaf(s[r], scale2, ref[e]);
                            }
                            s[r] = prob<OWN>(x, inv[e]);
                            dp[r] = s[r] * (dp[r] - dot4[e]);
                        }
                    }
                    if (edge) {  // rows from the key's own position on
                        const int n = j - p0;
                        const uint32_t bits = (n <= 0 ? ~0u : n >= 32 ? 0u : ~0u << n) >> (4 * half);
                        keep_only(s, bits, 0.f);
                        keep_only(dp, bits, 0.f);
                    }
                    bf16x8 pf[2][PP], sf[2][PP];
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float p[8], ds[8];
#pragma unroll
                        for (int r = 0; r < 8; ++r) p[r] = s[8 * c + r], ds[r] = dp[8 * c + r];
                        to_pieces<PP>(p, pf[c]);
                        to_pieces<PP>(ds, sf[c]);
                        if constexpr (NP == 1) {
#pragma unroll
                            for (int d = 0; d < ND; ++d) {
                                bf16x8 f[NP];
                                col_frag<DP>(dt, PLANE, 32 * t + 16 * c, 32 * d, at, f);
                                mma(dv[d], f, pf[c]);
                                col_frag<DP>(qt, PLANE, 32 * t + 16 * c, 32 * d, at, f);
                                mma(dk[d], f, sf[c]);
                            }
                        }
                    }
                    if constexpr (NP > 1) {
                        add_rows<DP, ND, NP>(dv, dt, PLANE, 32 * t, at, pf);
                        add_rows<DP, ND, NP>(dk, qt, PLANE, 32 * t, at, sf);
                    }
                }
                if (mine) {
                    const int next = now ^ (3 * QT);
                    lt[next + threadIdx.x] = -rs.ref;
                    it[next + threadIdx.x] = rs.inv;
                    et[next + threadIdx.x] = dot;
                }
            }
        }
    if constexpr (KW > 1) {
        constexpr int LD = DP + 4;
        float *buf = reinterpret_cast<float *>(lds) + (wave / KW) * (KW - 1) * 2 * 32 * LD + (lane & 31) * LD + 4 * half;
        __syncthreads();
#pragma unroll
        for (int v = 1; v < KW; ++v)
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    float *at = buf + (v - 1) * 2 * 32 * LD + 32 * d + 2 * r;
                    if (share == v) {
                        store4(at, dk[d][r], dk[d][r + 1], dk[d][r + 2], dk[d][r + 3]);
                        store4(at + 32 * LD, dv[d][r], dv[d][r + 1], dv[d][r + 2], dv[d][r + 3]);
                    }
                }
        __syncthreads();
        if (share) return;
#pragma unroll
        for (int v = 1; v < KW; ++v)
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const float *at = buf + (v - 1) * 2 * 32 * LD + 32 * d + 2 * r;
                    const f32x4 x = *reinterpret_cast<const f32x4_m *>(at), y = *reinterpret_cast<const f32x4_m *>(at + 32 * LD);
#pragma unroll
                    for (int e = 0; e < 4; ++e) dk[d][r + e] += x[e], dv[d][r + e] += y[e];
                }
    }
    if (j < a.Nk) {
        const float f = a.scale;
        if (a.groups > 1) {
            const int64_t at = ((((int64_t)w.b * a.Nk + j) * a.Hk + w.h) * a.groups + w0.h % a.groups) * a.D;
            float *ok_ = a.part + at, *ov = a.sums + at;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const int col = 32 * d + 2 * r + 4 * half;
                    if (col >= a.D) continue;
                    store4(ok_ + col, ok ? dk[d][r] * f : 0.f, ok ? dk[d][r + 1] * f : 0.f, ok ? dk[d][r + 2] * f : 0.f,
                           ok ? dk[d][r + 3] * f : 0.f);
                    store4(ov + col, ok ? dv[d][r] : 0.f, ok ? dv[d][r + 1] : 0.f, ok ? dv[d][r + 2] : 0.f,
                           ok ? dv[d][r + 3] : 0.f);
                }
            return;
        }
        const int64_t at = (((int64_t)w.b * a.Nk + j) * a.Hk + w.h) * a.D;
        T *ok_ = static_cast<T *>(a.dk) + at, *ov = static_cast<T *>(a.dv) + at;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int col = 32 * d + 2 * r + 4 * half;
                if (col >= a.D) continue;
                store4(ok_ + col, ok ? dk[d][r] * f : 0.f, ok ? dk[d][r + 1] * f : 0.f, ok ? dk[d][r + 2] * f : 0.f,
                       ok ? dk[d][r + 3] * f : 0.f);
                store4(ov + col, ok ? dv[d][r] : 0.f, ok ? dv[d][r + 1] : 0.f, ok ? dv[d][r + 2] : 0.f,
                       ok ? dv[d][r + 3] : 0.f);
            }
    }
}

// bf16 with a bias: multiplied only where a row asks for it, which the query gradients' waves have noted (2 x
// 2048 x 16 heads x 128, forward and backward: 348 us with the multiplication, 333 with the notes)
template <class T, int DW, int QT, int KW, bool BIAS>
__global__ __launch_bounds__(NT, (KW > 1 ? 1 : BIAS ? Shape<T, DW>::KV_BIAS_WAVES : Shape<T, DW>::KV_WAVES)) void attn_bwd_kv(Args a) {
    constexpr bool F32 = Elem<T>::NP > 1;
    if constexpr (!F32 && BIAS) {
        const Where w = where(a.B, a.Hk * a.groups, (a.Nk + 128 / KW - 1) / (128 / KW));
        const int64_t n = (int64_t)(a.H / a.Hk / a.groups) * ((a.Nq + a.tile_rows - 1) / a.tile_rows) * 4;  // its heads are neighbours
        const int *own = a.own + ((int64_t)w.b * a.Hk * a.groups + w.h) * n;
        int any = !a.own;  // (a call without query gradients has no notes)
        if (a.own)
            for (int64_t i = threadIdx.x & 63; i < n; i += 64) any |= own[i];
        if (__any(any)) {  // (the same in every wave)
            bwd_kv_rows<T, DW, QT, KW, BIAS, true>(a);
            return;
        }
    }
    bwd_kv_rows<T, DW, QT, KW, BIAS, F32>(a);
}

// dk and dv of a group from its parts, in order
template <class T>
__global__ __launch_bounds__(NT) void sum_group(Args a) {
    const int G = a.groups, C = a.D / 4;
    const int64_t e = (int64_t)blockIdx.x * NT + threadIdx.x, row = e / C;
    if (row >= (int64_t)a.B * a.Nk * a.Hk) return;
    const int col = e % C * 4;
    const float *from = (blockIdx.y ? a.sums : a.part) + row * G * a.D + col;
    f32x4 s = *reinterpret_cast<const f32x4_m *>(from);
    for (int g = 1; g < G; ++g) s += *reinterpret_cast<const f32x4_m *>(from + (int64_t)g * a.D);
    store4(static_cast<T *>(blockIdx.y ? a.dv : a.dk) + row * a.D + col, s[0], s[1], s[2], s[3]);
}

// The bias gradient of one wave: sums of ds over the diagonals of its 32 x 32 tiles.  Offset
// o = base - t with t = (query - key) mod 32 (add) or that + 32 (carry): every value moves to
// lane t of its half, two sums a lane.  The carry of a tile is the add of the next one, so each
// diagonal goes once to the wave's bins (twice where the wave's tiles do not follow each other);
// beyond the far offsets one sum a lane is kept.  No atomics: every sum has one order.
struct Diagonals {
    float carry = 0.f, left = 0.f, right = 0.f;
    int base = 0;
    __device__ __forceinline__ void flush(float v, int at, float *bins, int far, int lane) {
        v += __shfl_xor(v, 32);
        const int o = at - (lane & 31);
        if (lane < 32) {
            if (o <= -far) left += v;
            else if (o >= far) right += v;
            else bins[o + far] += v;
        }
    }
    // ds of keys base_key .. +31 (rows) and the wave's queries; b = first key - first query position
    __device__ __forceinline__ void tile(const f32x16 &ds, int b, float *bins, int far, int lane) {
        const int t = lane & 31, half = lane >> 5;
        if (base != b) flush(carry, base, bins, far, lane), carry = 0.f;  // (uniform)
        float a = carry;
        carry = 0.f;
        if (b - 31 >= far || b + 31 <= -far) {
            flush(a, b, bins, far, lane);
            float s = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) s += ds[r];
            if (b < 0) left += s;
            else right += s;
        } else {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int kr = 8 * (r >> 2) + 4 * half + (r & 3);
                const float x = __shfl(ds[r], ((t + kr) & 31) | (lane & 32));
                if (t + kr < 32) a += x;
                else carry += x;
            }
            flush(a, b, bins, far, lane);
        }
        base = b + 32;
    }
    __device__ __forceinline__ void end(float *bins, int far, int lane) {
        flush(carry, base, bins, far, lane);
        left = wave_sum_f32(left);
        right = wave_sum_f32(right);
        if (lane == 0) {
            bins[0] += left;
            bins[2 * far] += right;
        }
    }
};

// dq of 128 / KW rows (KW waves share 32, each taking every KW-th 32 keys), and the bias gradient's
// sums over their diagonals.  2 x 4096 x 16 heads x 128 bf16: 435 us (950 TFLOP/s); 64 columns 257 us
// (800); f32 2 x 2048 x 8 x 64: 164 us (157).
template <class T, int DW, int KT, int KW, bool BIAS>
__global__ __launch_bounds__(NT, (KW == 1 ? Shape<T, DW>::Q_WAVES : 1)) void attn_bwd_q(Args a) {
    constexpr int NP = Elem<T>::NP, PP = prob_pieces<T, KW>(), DP = pitch(DW), ND = blocks(DW), PLANE = KT * DP, ROWS = 128 / KW;
    static_assert(KT % (32 * KW) == 0, "tile");
    extern __shared__ __attribute__((aligned(16))) uint16_t lds[];
    typedef Tiles<T, DP, KT> KV;
    const int W = 2 * a.bk.far + 1;
    float *tab = reinterpret_cast<float *>(reinterpret_cast<char *>(lds) + area<T, DP, KT, KW, 1>());
    const int tiles = (a.Nq + ROWS - 1) / ROWS;
    const Where w = where(a.B, a.H, tiles);
    const Span sp = span_of(a, w.b);
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x >> 6;
    const int tile = tiles - 1 - w.tile, q0 = tile * ROWS, share = wave % KW, i = q0 + 32 * (wave / KW) + (lane & 31);
    const int hk = w.h / (a.H / a.Hk);
    const T *K = static_cast<const T *>(a.k) + w.b * a.ks[0] + hk * a.ks[2];
    const T *V = static_cast<const T *>(a.v) + w.b * a.vs[0] + hk * a.vs[2];
    const uint8_t *mask = a.key_mask ? a.key_mask + w.b * a.mask_sb : nullptr;
    float *all_bins = tab + table_size(a.bk.far), *bins = all_bins + wave * W;
    if constexpr (BIAS) {
        fill_table(a, tab, w.h);
        for (int o = threadIdx.x; o < 4 * W; o += NT) all_bins[o] = 0.f;
    }
    bf16x8 qf[DW / 16][NP], df[DW / 16][NP];
    load_row<T, DW>(static_cast<const T *>(a.q) + w.b * a.qs[0] + (int64_t)i * a.qs[1] + w.h * a.qs[2], i < sp.nq, a.D,
                    lane, qf);
    // The matrix cores round sums down, not to nearest: do . v comes out about 1e-8 of its size too
    // low, which a single ds does not feel but a bias gradient's sum over 10^6 of them does (f32: 9
    // times the error of one rounded to nearest).  Odd queries take -do, and their error the other way.
    const bool odd = NP > 1 && (lane & 1);
    load_row<T, DW>(static_cast<const T *>(a.dout) + w.b * a.dos[0] + (int64_t)i * a.dos[1] + w.h * a.dos[2], i < sp.nq,
                    a.D, lane, df, odd);
    const float sign = odd ? -1.f : 1.f;
    const size_t row = ((size_t)w.b * a.H + w.h) * a.Nq + i;
    const RowSum rs = row_sum_of<T, BIAS>(a, row, i < sp.nq);
    const float delta = row_dot<T, DW>(a, w.b, w.h, i, i < sp.nq, lane);
    if (half == 0 && share == 0 && i < a.Nq) a.delta[row] = delta;  // (the key gradients read it)
    if constexpr (BIAS && NP == 1) {
        const bool own = __any(rs.inv != 1.f);
        if (lane == 0) a.own[(((int64_t)w.b * a.H + w.h) * tiles + tile) * 4 + wave] = own;
    }
    const float scale2 = a.scale * LOG2E, delta_inv = delta * rs.inv;
    f32x16 acc[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] = zero16();
    Diagonals dg;
    const int last = min(q0 + ROWS, sp.nq) - 1;
    const int kend = last < q0 ? 0 : a.causal ? min(sp.nk, max(last + sp.start + 1, 0)) : sp.nk;
    KV kv;
    kv.init(lds, a.D);
    Lane<DP> at(lane);
    if (kend > 0) kv.issue(K, a.ks[1], V, a.vs[1], 0, sp.nk, a.D, mask);
    for (int j0 = 0; j0 < kend; j0 += KT) {
        kv.land(j0, sp.nk, mask);
        const uint16_t *kt = kv.x(), *vt = kv.y();
        if constexpr (Shape<T, DW>::TIGHT) at.opaque();
        if (j0 + KT < kend) kv.issue(K, a.ks[1], V, a.vs[1], j0 + KT, sp.nk, a.D, mask);
        const int qw = q0 + 32 * (wave / KW) + sp.start;
#pragma unroll
        for (int u = 0; u < KT / 32 / KW; ++u) {
            const int t = u * KW + share, j = j0 + 32 * t;
            if (j >= kend || (a.causal && j > qw + 31)) continue;
            const bool edge = mask || j + 32 > sp.nk || (a.causal && j + 31 > qw);
            f32x16 s = zero16(), dp = zero16();
#pragma unroll
            for (int c = 0; c < DW / 16; ++c) {
                bf16x8 f[NP];
                row_frag<DP>(kt, PLANE, 32 * t, c, at, f);
                mma(s, f, qf[c]);
                row_frag<DP>(vt, PLANE, 32 * t, c, at, f);
                mma(dp, f, df[c]);
            }
            if constexpr (BIAS) add_bias(s, scale2, tab, a.bk.far, j - qw, j - (i + sp.start), half);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float x = BIAS ? s[r] - rs.ref : __builtin_fmaf(s[r], scale2, -rs.ref);
                if constexpr (NP > 1) s[r] = prob<true>(x, rs.inv) * __builtin_fmaf(dp[r], sign, -delta);
                else s[r] = prob<false>(x, 1.f) * __builtin_fmaf(dp[r], rs.inv, -delta_inv);
            }
            if (edge) keep_only(s, visible(a, j - (i + sp.start), seen_keys(j, sp.nk, mask), half), 0.f);
            if (BIAS && a.dbias) dg.tile(s, j - qw, bins, a.bk.far, lane);
            bf16x8 sf[2][PP];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float x[8];
#pragma unroll
                for (int r = 0; r < 8; ++r) x[r] = s[8 * c + r];
                to_pieces<PP>(x, sf[c]);
            }
            add_rows<DP, ND, NP>(acc, kt, PLANE, 32 * t, at, sf);
        }
    }
    if constexpr (KW > 1) {
        constexpr int LD = DP + 4;
        float *buf = reinterpret_cast<float *>(lds) + (wave / KW) * (KW - 1) * 32 * LD + (lane & 31) * LD + 4 * half;
        __syncthreads();
#pragma unroll
        for (int v = 1; v < KW; ++v)
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int r = 0; r < 16; r += 4)
                    if (share == v)
                        store4(buf + (v - 1) * 32 * LD + 32 * d + 2 * r, acc[d][r], acc[d][r + 1], acc[d][r + 2], acc[d][r + 3]);
        __syncthreads();
#pragma unroll
        for (int v = 1; v < KW; ++v)
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const f32x4 x = *reinterpret_cast<const f32x4_m *>(buf + (v - 1) * 32 * LD + 32 * d + 2 * r);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[d][r + e] += x[e];
                }
    }
    if (i < a.Nq && a.dq && share == 0) {
        T *o = static_cast<T *>(a.dq) + (((int64_t)w.b * a.Nq + i) * a.H + w.h) * a.D;
        const float f = a.scale;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int col = 32 * d + 2 * r + 4 * half;
                if (col < a.D) store4(o + col, acc[d][r] * f, acc[d][r + 1] * f, acc[d][r + 2] * f, acc[d][r + 3] * f);
            }
    }
    if (BIAS && a.dbias) {
        if (kend == 0) __syncthreads();  // the bins were cleared by other waves
        dg.end(bins, a.bk.far, lane);
        __syncthreads();
        float *to = a.bins + (((size_t)w.h * a.B + w.b) * tiles + tile) * W;
        for (int o = threadIdx.x; o < W; o += NT)
            to[o] = ((all_bins[o] + all_bins[W + o]) + all_bins[2 * W + o]) + all_bins[3 * W + o];
    }
}

// dbias[bucket][h] from the workgroups' diagonal sums: a workgroup sums one bucket's offsets (a run:
// buckets go by distance and side) over batch and tiles, in 64 bits and in one order.
template <class T>
__global__ __launch_bounds__(NT) void bias_reduce(Args a) {
    __shared__ double sum[NT];
    __shared__ int from, to;
    const int h = blockIdx.x, n = blockIdx.y, far = a.bk.far, W = 2 * far + 1, tiles = (a.Nq + a.tile_rows - 1) / a.tile_rows;
    if (threadIdx.x == 0) from = W, to = 0;
    __syncthreads();
    for (int o = threadIdx.x; o < W; o += NT)
        if (bucket_of(a.bk, o - far) == n) atomicMin(&from, o), atomicMax(&to, o + 1);
    __syncthreads();
    const int lo = from, w = to - lo, parts = a.B * tiles;  // (no offset: w <= 0)
    const float *in = a.bins + (size_t)h * parts * W + lo;
    double s = 0.;
    if (w == 1) {  // (most buckets)
#pragma unroll 4
        for (int p = threadIdx.x; p < parts; p += NT) s += in[(size_t)p * W];
    } else if (w > 1) {
        for (int p0 = 0; p0 < parts; p0 += 1 << 16) {  // (so that the flat index keeps 32 bits)
            const uint32_t all = (uint32_t)min(parts - p0, 1 << 16) * w;
#pragma unroll 4
            for (uint32_t e = threadIdx.x; e < all; e += NT) {
                const uint32_t p = e / (uint32_t)w;
                s += in[(size_t)(p0 + p) * W + (e - p * w)];
            }
        }
    }
    sum[threadIdx.x] = s;
    __syncthreads();
    for (int k = NT / 2; k > 0; k >>= 1) {
        if (threadIdx.x < k) sum[threadIdx.x] += sum[threadIdx.x + k];
        __syncthreads();
    }
    if (threadIdx.x == 0) static_cast<T *>(a.dbias)[(size_t)n * a.H + h] = (T)(float)sum[0];
}

// ------------------------------------------------------------------- C interface --

constexpr int64_t MAX_GRID = ((int64_t)1 << 32) / NT - 1;
int row_tiles(int n) { return (n + ROWS - 1) / ROWS; }

// rows of (batch, tokens, heads) in 16-byte steps; a dimension of one is never stepped over
bool rows_ok(const void *p, const int64_t s[3], int esize, int b, int n, int h) {
    const int64_t e = 16 / esize;
    return p && reinterpret_cast<uintptr_t>(p) % 16 == 0 && (b == 1 || s[0] % e == 0) && (n == 1 || s[1] % e == 0) &&
           (h == 1 || s[2] % e == 0);
}

// the argument checks shared by both directions; fills the kernels' arguments
int take(const hreg_tok_attn_t *p, Args &a) {
    if (!p || (p->dtype != HREG_TOK_F32 && p->dtype != HREG_TOK_BF16)) return HREG_ERR_INVALID;
    if (p->B < 0 || p->Nq < 0 || p->Nk < 0 || p->H < 1 || p->Hk < 1 || p->H % p->Hk) return HREG_ERR_INVALID;
    if (p->D < 8 || p->D > 128 || p->D % 8) return HREG_ERR_UNSUPPORTED;
    // (a launch has fewer than 2^32 threads)
    if ((int64_t)p->B * p->H * row_tiles(p->Nq) > MAX_GRID || (int64_t)p->B * p->H * row_tiles(p->Nk) > MAX_GRID ||
        (int64_t)p->B * p->H > MAX_GRID || (int64_t)p->Nq * (p->H / p->Hk) > (1 << 30) ||
        p->Nq > (1 << 30) || p->Nk > (1 << 30))
        return HREG_ERR_UNSUPPORTED;
    const int es = p->dtype == HREG_TOK_F32 ? 4 : 2;
    const bool empty = p->B == 0 || p->Nq == 0;
    if (!empty && (!rows_ok(p->q, p->qs, es, p->B, p->Nq, p->H) || !rows_ok(p->out, p->os, es, p->B, p->Nq, p->H) ||
                   reinterpret_cast<uintptr_t>(p->out_rest) % 16)) return HREG_ERR_INVALID;
    if (p->B > 0 && p->Nk > 0 && (!rows_ok(p->k, p->ks, es, p->B, p->Nk, p->Hk) || !rows_ok(p->v, p->vs, es, p->B, p->Nk, p->Hk))) return HREG_ERR_INVALID;
    a = Args{};
    a.q = p->q; a.k = p->k; a.v = p->v; a.out = p->out; a.out_r = p->out; a.dout = p->dout;
    a.rest = p->dtype == HREG_TOK_BF16 ? p->out_rest : nullptr;
    a.dq = p->dq; a.dk = p->dk; a.dv = p->dv; a.dbias = p->dbias;
    a.lse = p->lse; a.q_len = p->q_len; a.k_len = p->k_len; a.key_mask = p->key_mask; a.bias = p->bias;
    for (int i = 0; i < 3; ++i) {
        a.qs[i] = p->qs[i]; a.ks[i] = p->ks[i]; a.vs[i] = p->vs[i]; a.os[i] = p->os[i]; a.dos[i] = p->dos[i];
    }
    a.mask_sb = p->mask_sb;
    a.B = p->B; a.Nq = p->Nq; a.Nk = p->Nk; a.H = p->H; a.Hk = p->Hk; a.D = p->D;
    a.causal = p->causal != 0; a.align_end = p->align_end != 0; a.scale = p->scale;
    if (p->bias) {
        if (p->bias_dtype != HREG_TOK_F32 && p->bias_dtype != HREG_TOK_BF16) return HREG_ERR_INVALID;
        const int side = p->both ? p->num_buckets / 2 : p->num_buckets, exact = side / 2;
        if (p->num_buckets < 2 || (p->both && (p->num_buckets % 2 || side < 2)) || p->max_distance <= exact)
            return HREG_ERR_INVALID;
        if (p->num_buckets > HREG_TOK_MAX_BUCKETS || p->max_distance > (MAX_BINS - 1) / 2) return HREG_ERR_UNSUPPORTED;
        if (p->nthresh != side - exact - 1 || p->nthresh > HREG_TOK_MAX_THRESH) return HREG_ERR_INVALID;
        a.bias_f32 = p->bias_dtype == HREG_TOK_F32;
        a.bk.n = p->num_buckets; a.bk.far = p->max_distance; a.bk.both = p->both != 0; a.bk.exact = exact;
        a.bk.nthresh = p->nthresh;
        for (int t = 0; t < p->nthresh; ++t) a.bk.thresh[t] = p->thresh[t];
    }
    return HREG_OK;
}

// launches F<T, DW, tile, BIAS> with its dynamic LDS (above the 64 KB default where needed)
template <class K>
int launch(K *kernel, int grid, size_t lds, void *stream, const Args &a) {
    if (lds > 65536 &&
        hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess)
        return HREG_ERR_LAUNCH;
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(NT), lds, as_stream(stream), a);
    HREG_CHECK_LAUNCH();
    return HREG_OK;
}

template <class T, int DW, bool BIAS>
int fwd(const Args &a, void *stream) {
    if (a.splits) {
        const int R = a.Nq * (a.H / a.Hk);
        constexpr int DP = pitch(DW);
        const size_t tile = (size_t)4 * Elem<T>::NP * 32 * DP * 2, join = (size_t)4 * 32 * (DP + 4) * 4;
        Args b = a;
        b.split_bytes = tile > join ? tile : join;
        const size_t tables = BIAS ? (size_t)(a.H / a.Hk) * (2 * (a.bk.far + PAD) + 1) * 4 : 0;
        b.group_tables = tables <= 32768;
        const int rc = launch(attn_split<T, DW, BIAS>, a.B * a.Hk * ((R + 31) / 32) * a.splits,
                              b.split_bytes + (b.group_tables ? tables : 0), stream, b);
        if (rc != HREG_OK || a.splits == 1) return rc;
        const int64_t rows = (int64_t)a.B * a.H * a.Nq;
        hipLaunchKernelGGL(attn_join<T>, dim3((rows + NT / 32 - 1) / (NT / 32)), dim3(NT), 0, as_stream(stream), a);
        HREG_CHECK_LAUNCH();
        return HREG_OK;
    }
    constexpr int KT = Shape<T, DW>::FWD_KEYS;
    const size_t lds = Tiles<T, pitch(DW), KT>::BYTES + (BIAS ? (2 * (a.bk.far + PAD) + 1) * 4 : 0);
    return launch(attn_fwd<T, DW, KT, BIAS>, a.B * a.H * row_tiles(a.Nq), lds, stream, a);
}

template <class T, int DW, int KW, bool BIAS>
int bwd_kv(const Args &a, void *stream) {
    constexpr int QT = KW > 1 ? 32 * KW : Shape<T, DW>::BWD_ROWS;
    const size_t lds = area<T, pitch(DW), QT, KW, 2>() + (6 * QT + (BIAS ? 2 * (a.bk.far + PAD) + 1 : 0)) * 4;
    return launch(attn_bwd_kv<T, DW, QT, KW, BIAS>, a.B * a.Hk * a.groups * ((a.Nk + 128 / KW - 1) / (128 / KW)), lds, stream, a);
}
template <class T, int DW, int KW, bool BIAS>
int bwd_q(const Args &a, void *stream) {
    constexpr int KT = KW > 1 ? 32 * KW : Shape<T, DW>::Q_KEYS;
    const size_t W = 2 * a.bk.far + 1, lds = area<T, pitch(DW), KT, KW, 1>() + (BIAS ? W + 2 * PAD + 4 * W : 0) * 4;
    return launch(attn_bwd_q<T, DW, KT, KW, BIAS>, a.B * a.H * ((a.Nq + a.tile_rows - 1) / a.tile_rows), lds, stream, a);
}

template <class T, int DW, bool BIAS>
int bwd(const Args &a, void *stream) {
    constexpr int SHARE = Shape<T, DW>::SHARE;
    int rc = HREG_OK;
    // the query gradients' kernel first: it leaves the rows' dots for the key gradients
    if (a.Nq > 0 && (a.dq || a.dbias)) {
        rc = a.tile_rows < ROWS ? bwd_q<T, DW, SHARE, BIAS>(a, stream) : bwd_q<T, DW, 1, BIAS>(a, stream);
    } else if (a.Nq > 0) {
        const int64_t rows = (int64_t)a.B * a.H * a.Nq;
        hipLaunchKernelGGL((attn_delta<T, DW>), dim3((rows + NT / 2 - 1) / (NT / 2)), dim3(NT), 0, as_stream(stream), a);
        HREG_CHECK_LAUNCH();
    }
    if (rc == HREG_OK && a.Nk > 0 && a.dk) {
        rc = a.share_kv ? bwd_kv<T, DW, SHARE, BIAS>(a, stream) : bwd_kv<T, DW, 1, BIAS>(a, stream);
        if (rc == HREG_OK && a.groups > 1) {
            const int64_t n = (int64_t)a.B * a.Nk * a.Hk * (a.D / 4);
            hipLaunchKernelGGL(sum_group<T>, dim3((n + NT - 1) / NT, 2), dim3(NT), 0, as_stream(stream), a);
            HREG_CHECK_LAUNCH();
        }
    }
    return rc;
}

template <class T, bool BIAS, bool BACK>
int by_width(const Args &a, void *stream) {
    if constexpr (BACK) {
        if (a.D <= 32) return bwd<T, 32, BIAS>(a, stream);
        if (a.D <= 48) return bwd<T, 48, BIAS>(a, stream);
        if (a.D <= 64) return bwd<T, 64, BIAS>(a, stream);
        if (a.D <= 96) return bwd<T, 96, BIAS>(a, stream);
        return bwd<T, 128, BIAS>(a, stream);
    } else {
        if (a.D <= 32) return fwd<T, 32, BIAS>(a, stream);
        if (a.D <= 48) return fwd<T, 48, BIAS>(a, stream);
        if (a.D <= 64) return fwd<T, 64, BIAS>(a, stream);
        if (a.D <= 96) return fwd<T, 96, BIAS>(a, stream);
        return fwd<T, 128, BIAS>(a, stream);
    }
}

template <bool BACK>
int by_type(const hreg_tok_attn_t *p, const Args &a, void *stream) {
    if (p->dtype == HREG_TOK_F32)
        return a.bias ? by_width<float, true, BACK>(a, stream) : by_width<float, false, BACK>(a, stream);
    return a.bias ? by_width<__bf16, true, BACK>(a, stream) : by_width<__bf16, false, BACK>(a, stream);
}

// 0: the row kernel; else the number of runs of the split kernel: where all rows of a key head fit
// one of its tiles, or few row tiles face many keys.  (us, row / split kernel: 1 token x 32768 keys
// 1110 / 160; 2 x 700 x 8 heads x 128 bf16 29 / 37; 4 x 517 x 8 x 40 f32 with a bias 39 / 47.)  Two
// workgroups a CU are enough: 4 tokens x 8191 keys take 34 us with 512, 45 with 1024.
int split_of(const hreg_tok_attn_t *p) {
    const int64_t R = (int64_t)p->Nq * (p->H / p->Hk), tiles = (int64_t)p->B * p->Hk * ((R + 31) / 32);
    const int64_t rows = (int64_t)p->B * p->H * row_tiles(p->Nq);
    if (tiles == 0 || (R > 32 && (rows >= CUS || p->Nk <= 16 * rows))) return 0;
    int64_t s = (2 * CUS + tiles - 1) / tiles, most = (p->Nk + 255) / 256;
    s = s < most ? s : most;
    return s < 1 ? 1 : s > 256 ? 256 : (int)s;
}
size_t part_floats(const hreg_tok_attn_t *p, int splits) {  // results, then maxima and sums
    return splits > 1 ? (size_t)p->B * p->H * p->Nq * splits : 0;
}

// How the backward pass is divided.  groups: parts of a group's heads that the key gradients are
// split over, as few as give four workgroups a CU (2 x 4096 keys x 4 of 16 heads x 128 bf16: one long
// workgroup a CU otherwise, 1600 -> 938 us); share_kv, tile_rows: whether waves share rows, and the query rows of a workgroup.  Sharing pays
// while fewer than 160 workgroups are there without it (96: 146 -> 99 us; 160: 141 -> 176).
struct BwdPlan { int groups, share_kv, tile_rows; };
template <class T>
int share_of(int D) {
    return D <= 32 ? Shape<T, 32>::SHARE : D <= 64 ? Shape<T, 64>::SHARE : Shape<T, 128>::SHARE;
}
BwdPlan bwd_plan(const hreg_tok_attn_t *p) {
    const int G = p->H / p->Hk, share = p->dtype == HREG_TOK_F32 ? share_of<float>(p->D) : share_of<__bf16>(p->D);
    const int64_t keys = (int64_t)p->B * p->Hk * row_tiles(p->Nk), rows = (int64_t)p->B * p->H * row_tiles(p->Nq);
    BwdPlan q;
    q.groups = 1;
    if (p->dk)
        while (q.groups < G && (G % q.groups || keys * q.groups < 4 * CUS)) ++q.groups;
    q.share_kv = share > 1 && keys * q.groups < 160;
    q.tile_rows = rows < 160 ? ROWS / share : ROWS;
    return q;
}
size_t group_floats(const hreg_tok_attn_t *p) {
    const int groups = bwd_plan(p).groups;
    return groups > 1 ? (size_t)p->B * p->Nk * p->Hk * groups * p->D : 0;
}
size_t bins_bytes(const hreg_tok_attn_t *p) {
    if (!p->bias) return 0;
    const size_t rows = bwd_plan(p).tile_rows, tiles = (p->Nq + rows - 1) / rows;
    return ((size_t)p->B * p->H * tiles * (2 * (size_t)p->max_distance + 1) * 4 + 255) / 256 * 256;
}
size_t own_bytes(const hreg_tok_attn_t *p) {
    if (!p->bias || p->dtype != HREG_TOK_BF16) return 0;
    const size_t rows = bwd_plan(p).tile_rows;
    return ((size_t)p->B * p->H * ((p->Nq + rows - 1) / rows) * 16 + 255) / 256 * 256;
}
size_t delta_bytes(const hreg_tok_attn_t *p) { return ((size_t)p->B * p->H * p->Nq * 4 + 255) / 256 * 256; }

}  // namespace

extern "C" {

size_t hreg_tok_attn_ws_bytes(const hreg_tok_attn_t *p, int backward) {
    if (!p || p->B < 0 || p->Nq < 0 || p->Nk < 0 || p->H < 1 || p->Hk < 1 || p->H % p->Hk || p->D < 1) return 0;
    if (!backward) return part_floats(p, split_of(p)) * (p->D + 2) * 4;
    return delta_bytes(p) + bins_bytes(p) + own_bytes(p) + 2 * group_floats(p) * 4;
}

int hreg_tok_attn_fwd(const hreg_tok_attn_t *p, void *stream) {
    Args a;
    const int rc = take(p, a);
    if (rc != HREG_OK) return rc;
    if (a.B == 0 || a.Nq == 0) return HREG_OK;
    const size_t need = hreg_tok_attn_ws_bytes(p, 0);
    if (p->ws_bytes < need || (need && (!p->ws || reinterpret_cast<uintptr_t>(p->ws) % 256))) return HREG_ERR_INVALID;
    a.splits = split_of(p);
    a.part = static_cast<float *>(p->ws);
    a.sums = a.part + part_floats(p, a.splits) * p->D;
    return by_type<false>(p, a, stream);
}

int hreg_tok_attn_bwd(const hreg_tok_attn_t *p, void *stream) {
    Args a;
    const int rc = take(p, a);
    if (rc != HREG_OK) return rc;
    if (!a.bias) a.dbias = nullptr;
    if (a.B > 0 && a.Nq > 0 && (!rows_ok(p->dout, p->dos, p->dtype == HREG_TOK_F32 ? 4 : 2, p->B, p->Nq, p->H) || !p->lse)) return HREG_ERR_INVALID;
    for (const void *g : {p->dq, p->dk, p->dv})
        if (reinterpret_cast<uintptr_t>(g) % 16) return HREG_ERR_INVALID;
    if (!p->dk != !p->dv) return HREG_ERR_INVALID;
    const size_t need = hreg_tok_attn_ws_bytes(p, 1);
    if (p->ws_bytes < need || (need && (!p->ws || reinterpret_cast<uintptr_t>(p->ws) % 256))) return HREG_ERR_INVALID;
    const BwdPlan plan = bwd_plan(p);
    a.tile_rows = plan.tile_rows;
    a.share_kv = plan.share_kv;
    a.delta = static_cast<float *>(p->ws);
    a.bins = reinterpret_cast<float *>(static_cast<char *>(p->ws) + delta_bytes(p));
    a.groups = plan.groups;
    char *const own = static_cast<char *>(p->ws) + delta_bytes(p) + bins_bytes(p);
    if (a.dq || a.dbias) a.own = reinterpret_cast<int *>(own);  // (else the kernel that writes it does not run)
    a.part = reinterpret_cast<float *>(own + own_bytes(p));
    a.sums = a.part + group_floats(p);
    if (a.B > 0) {
        const int rc2 = by_type<true>(p, a, stream);
        if (rc2 != HREG_OK) return rc2;
    }
    if (a.dbias) {  // an empty batch too: the gradient is zero
        if (a.bias_f32) hipLaunchKernelGGL(bias_reduce<float>, dim3(a.H, a.bk.n), dim3(NT), 0, as_stream(stream), a);
        else hipLaunchKernelGGL(bias_reduce<__bf16>, dim3(a.H, a.bk.n), dim3(NT), 0, as_stream(stream), a);
        HREG_CHECK_LAUNCH();
    }
    return HREG_OK;
}

}  // extern "C"
