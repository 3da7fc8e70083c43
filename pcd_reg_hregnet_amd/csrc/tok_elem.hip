// tok_elem.hip -- dropout from a counter-based generator, and the gated residual with the norm
// behind one block and the norm before the next, forward and backward.
//
// The generator is Philox4x32-10 (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3",
// 2011): a counter's four output words are the random bits of eight consecutive elements, 16 each,
// so the mask is made again wherever it is needed and never stored.

#include "tokens.h"

namespace {

using namespace hreg_tok;

constexpr int NT = 256;

// A launch has fewer than 2^32 threads a dimension: many workgroups go into two
__device__ __forceinline__ int64_t block_number() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }
dim3 grid_of(int64_t blocks) {
    const int64_t x = blocks < (1 << 21) ? blocks : 1 << 21;
    return dim3((uint32_t)x, (uint32_t)((blocks + x - 1) / x));
}

struct Rng {
    uint64_t seed;
    const uint64_t *dev;
    uint32_t site, step;
    float keep;  // 1 / (1 - step / 65536)
};

__device__ __forceinline__ uint64_t rng_seed(const Rng &g) { return g.dev ? *g.dev : g.seed; }

// the output words of one counter (group of eight elements)
__device__ __forceinline__ u32x4 philox(uint64_t group, uint32_t site, uint64_t seed) {
    uint32_t c0 = (uint32_t)group, c1 = (uint32_t)(group >> 32), c2 = site, c3 = 0;
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return u32x4{c0, c1, c2, c3};
}

// the 16 bits of elements first .. first + 7, two a word; EIGHT: first is a multiple of eight
template <bool EIGHT>
__device__ __forceinline__ u32x4 bits_of(uint64_t first, uint32_t site, uint64_t seed) {
    const u32x4 a = philox(first >> 3, site, seed);
    const int off = first & 7;
    if (EIGHT || off == 0) return a;
    const u32x4 b = philox((first >> 3) + 1, site, seed);
    uint32_t w[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = off & 4 ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = off & 2 ? w[i + 1] : w[i];
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = off & 1 ? (w[i] >> 16) | (w[i + 1] << 16) : w[i];
    return r;
}

// 1 / (1 - p) or 0 for eight elements
template <bool EIGHT>
__device__ __forceinline__ void mask_of(const Rng &g, uint64_t first, uint64_t seed, float (&m)[8]) {
    const u32x4 w = bits_of<EIGHT>(first, g.site, seed);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m[2 * i] = (w[i] & 0xffffu) >= g.step ? g.keep : 0.f;
        m[2 * i + 1] = (w[i] >> 16) >= g.step ? g.keep : 0.f;
    }
}

__device__ __forceinline__ void unpack(const u32x4 &w, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = bf16_lo(w[i]), v[2 * i + 1] = bf16_hi(w[i]);
}

// eight consecutive elements, n of them there (the others 0); VEC: 16-byte aligned and all there
template <bool VEC>
__device__ __forceinline__ void load8(const __bf16 *p, int n, float (&v)[8]) {
    if constexpr (VEC) {
        unpack(*reinterpret_cast<const u32x4_m *>(p), v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? (float)p[i] : 0.f;
    }
}
template <bool VEC>
__device__ __forceinline__ void load8(const float *p, int n, float (&v)[8]) {
    if constexpr (VEC) {
        const f32x4 a = *reinterpret_cast<const f32x4_m *>(p), b = *reinterpret_cast<const f32x4_m *>(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : 0.f;
    }
}
template <bool VEC, class T>
__device__ __forceinline__ void store8(T *p, int n, const float (&v)[8]) {
    if constexpr (VEC) {
        if constexpr (sizeof(T) == 2) {
            *reinterpret_cast<u32x4_m *>(p) = u32x4{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]),
                                                    pack_bf16(v[6], v[7])};
        } else {
            store4(p, v[0], v[1], v[2], v[3]);
            store4(p + 4, v[4], v[5], v[6], v[7]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = (T)v[i];
    }
}

// ------------------------------------------------------------------------ dropout --

// Eight elements a thread from one counter (16 bits an element: p to 2^-16, and half the generator's
// multiplications of 32).  8 x 4096 x 2048 bf16: 45 us (6.0 TB/s, part of it the last-level cache's).

template <class T, bool VEC>
__global__ __launch_bounds__(NT) void dropout_kernel(const T *__restrict__ x, T *__restrict__ y, int64_t n, Rng g) {
    const int64_t at = (block_number() * NT + threadIdx.x) * 8;
    if (at >= n) return;
    float v[8], m[8];
    const int have = (int)min((int64_t)8, n - at);
    if (VEC && have == 8) load8<true>(x + at, 8, v);
    else load8<false>(x + at, have, v);
    mask_of<true>(g, at, rng_seed(g), m);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = m[i] != 0.f ? v[i] * m[i] : 0.f;  // a dropped NaN is gone
    if (VEC && have == 8) store8<true>(y + at, 8, v);
    else store8<false>(y + at, have, v);
}

// ----------------------------------------------------- gated residual and its norms --

struct Block {
    const void *x, *f, *gate, *post_w, *post_b, *pre_w, *pre_b, *dy, *dh;
    void *y, *h, *dx, *df, *dgate;
    float *stats, *part, *gpart;  // part [parts][4][C]; gpart [gate rows][splits][C]
    int R, C, gate_rows, post, pre, param_f32, splits, want;  // want: bit k: column sum k
    float scale, eps;
    Rng rng;
};

// A row has TPR threads of eight elements each: 16, 32 or 64 of a wave (the workgroup's 256 threads
// then hold several rows), or a workgroup of TPR.  A row's waits are hidden by the other rows of its
// CU, so the fewer registers and the more rows the better (rows of 4096 bf16, backward: 369 us with
// 16 elements a thread and two waves a SIMD).
template <int TPR> constexpr int threads() { return TPR > 64 ? TPR : NT; }

// How a thread's elements are reached.  WHOLE: every thread of a row has eight, 16-byte aligned, and
// the call has it all (both norms, both gradients in, the rows' gradients out): nothing is
// asked per thread and little per call.  ALIGNED: eight or none.  SINGLE: one by one, any alignment.
// (67 million elements bf16, a gate for each row, us: rows of 4096 with both norms 122 forward and 232 backward,
// without the norm behind the block, so ALIGNED, 116 and 375; of 4088 with both 124 and 405, 768: 146 and 340,
// 5120: 164 and 361.  ALIGNED takes 137 registers at 512 threads a row, which leaves three waves a SIMD.)
enum { SINGLE, ALIGNED, WHOLE };

// sum over the TPR threads of a row, in every one of them
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float *lds) {
    v = row_sum16(v);
    if constexpr (TPR >= 32) v = fadd_rn(v, __shfl_xor(v, 16));
    if constexpr (TPR >= 64) v = fadd_rn(v, __shfl_xor(v, 32));
    if constexpr (TPR > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = lds[0];
#pragma unroll
        for (int w = 1; w < TPR / 64; ++w) v = fadd_rn(v, lds[w]);
    }
    return v;
}

// the thread's eight elements of a row, of which n > 0 are there; 0 beyond
template <int MODE, class T>
__device__ __forceinline__ void get8(const void *p, int64_t at, int n, float (&v)[8]) {
    if (MODE == WHOLE || n > 0) {
        load8<(MODE >= ALIGNED)>(static_cast<const T *>(p) + at, n, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.f;
    }
}

// a parameter's elements c .. c + 7, of which n are there; `other` where there is no such parameter
// and in a thread behind the row's end (n <= 0), which must not read there
template <int MODE>
__device__ __forceinline__ void param8(const void *p, int f32, int c, int n, float other, float (&v)[8]) {
    if (!p || (MODE != WHOLE && n <= 0)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = other;
    } else if (f32) load8<(MODE >= ALIGNED)>(static_cast<const float *>(p) + c, n, v);
    else load8<(MODE >= ALIGNED)>(static_cast<const __bf16 *>(p) + c, n, v);
}

// mean and 1 / deviation of a row held in registers (two passes: the mean, then the squares
// around it)
template <int TPR>
__device__ __forceinline__ void row_stats(const float (&v)[8], int kind, float inv_c, int n, float eps, float &mu, float &rs,
                                          float *lds) {
    mu = 0.f;
    if (kind == 2) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += v[i];
        mu = row_sum<TPR>(s, lds) * inv_c;
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float d = i < n ? v[i] - mu : 0.f;
        s = __builtin_fmaf(d, d, s);
    }
    rs = 1.f / sqrtf(row_sum<TPR>(s, lds) * inv_c + eps);
}

// Every input is read once and stays in registers through both norms.  Bound by its bytes: rows of
// 4096 bf16 (16384 of them, a gate for each) 115 us (5.8 TB/s).
template <class T, int TPR, int MODE>
__global__ __launch_bounds__(threads<TPR>()) void block_fwd(Block a) {
    __shared__ float lds[16];
    constexpr bool VEC = MODE >= ALIGNED, USUAL = MODE == WHOLE;
    const int r = (int)block_number() * (threads<TPR>() / TPR) + threadIdx.x / TPR, C = a.C, c = threadIdx.x % TPR * 8;
    const int n = USUAL ? 8 : C - c;
    if (r >= a.R) return;  // (a workgroup of one row leaves as a whole)
    const int64_t at = (int64_t)r * C + c;
    const float inv_c = 1.f / (float)C;
    float y[8], mu = 0.f, rs = 1.f, mu2 = 0.f, rs2 = 1.f;
    get8<MODE, T>(a.x, at, n, y);
    if (USUAL || a.f) {
        float u[8], w[8], b[8];
        get8<MODE, T>(a.f, at, n, u);
        if (USUAL || a.post) {
            row_stats<TPR>(u, a.post, inv_c, n, a.eps, mu, rs, lds);
            param8<MODE>(a.post_w, a.param_f32, c, n, 1.f, w);
            param8<MODE>(a.post_b, a.param_f32, c, n, 0.f, b);
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] = __builtin_fmaf((u[i] - mu) * rs, w[i], b[i]);
        }
        if (a.rng.step) {
            mask_of<VEC>(a.rng, at, rng_seed(a.rng), w);
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] = w[i] != 0.f ? u[i] * w[i] : 0.f;
        }
        if (a.gate) {
            get8<MODE, T>(a.gate, (int64_t)(r / a.gate_rows) * C + c, n, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] *= w[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = i < n ? __builtin_fmaf(a.scale, u[i], y[i]) : 0.f;
        if (n > 0) store8<VEC>(static_cast<T *>(a.y) + at, n, y);
    }
    if (USUAL || a.pre) {
        float w[8], b[8];
        row_stats<TPR>(y, a.pre, inv_c, n, a.eps, mu2, rs2, lds);
        param8<MODE>(a.pre_w, a.param_f32, c, n, 1.f, w);
        param8<MODE>(a.pre_b, a.param_f32, c, n, 0.f, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = __builtin_fmaf((y[i] - mu2) * rs2, w[i], b[i]);
        if (n > 0) store8<VEC>(static_cast<T *>(a.h) + at, n, w);
    }
    if (a.stats && c == 0) *reinterpret_cast<f32x4_m *>(a.stats + 4 * (int64_t)r) = f32x4{mu, rs, mu2, rs2};
}

// Column sums of the backward pass, in this order: the norms' weights and, where they are wanted
// (FULL), their biases and a gate that several rows share.
enum { S_POST_W, S_PRE_W, S_POST_B, S_PRE_B, S_GATE };
template <bool FULL> constexpr int sums() { return FULL ? 5 : 2; }

// One row's gradients; column sums stay in registers.  The statistics are the forward pass's,
// everything else is computed again.  Bound by its bytes (f, y, dy, dh and the gate read, dx, df and
// the gate's gradient written) and, with dropout, nearly as much by its instructions: the same rows
// 225 us (4.8 TB/s).
template <class T, int TPR, int MODE, bool FULL>
__device__ __forceinline__ void back_row(const Block &a, int r, int c, uint64_t seed, bool direct_gate, float inv_c, float *lds,
                                         float (&sum)[sums<FULL>()][8]) {
    constexpr bool VEC = MODE >= ALIGNED, USUAL = MODE == WHOLE;
    const int C = a.C, n = USUAL ? 8 : C - c;
    const int64_t at = (int64_t)r * C + c;
    const f32x4 st = *reinterpret_cast<const f32x4_m *>(a.stats + 4 * (int64_t)r);
    float dx[8], x[8], g[8], f[8], q[8], w[8], b[8];
    // all of the row's reads first
    const bool pre = USUAL || (a.pre && a.dh);
    get8<MODE, T>(a.dy, at, USUAL || a.dy ? n : 0, dx);
    get8<MODE, T>(a.dh, at, pre ? n : 0, g);
    get8<MODE, T>(a.y, at, pre ? n : 0, x);
    get8<MODE, T>(a.f, at, USUAL || a.f ? n : 0, f);
    if (a.gate) get8<MODE, T>(a.gate, (int64_t)(r / a.gate_rows) * C + c, n, q);
    if (pre) {
        float s1 = 0.f, s2 = 0.f;
        param8<MODE>(a.pre_w, a.param_f32, c, n, 1.f, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = i < n ? (x[i] - st[2]) * st[3] : 0.f;
            sum[S_PRE_W][i] = __builtin_fmaf(g[i], x[i], sum[S_PRE_W][i]);
            if constexpr (FULL) sum[S_PRE_B][i] += g[i];
            g[i] = i < n ? g[i] * w[i] : 0.f;
            s1 = __builtin_fmaf(g[i], x[i], s1);
            s2 += g[i];
        }
        s1 = row_sum<TPR>(s1, lds) * inv_c;
        s2 = a.pre == 2 ? row_sum<TPR>(s2, lds) * inv_c : 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) dx[i] = __builtin_fmaf(st[3], __builtin_fmaf(-x[i], s1, g[i] - s2), dx[i]);
    }
    if (n > 0 && (USUAL || a.dx)) store8<VEC>(static_cast<T *>(a.dx) + at, n, dx);
    if (!USUAL && !a.f) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = i < n ? dx[i] * a.scale : 0.f;
    if (a.rng.step) {
        mask_of<VEC>(a.rng, at, seed, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = w[i] != 0.f ? g[i] * w[i] : 0.f;
    }
    const bool post = USUAL || a.post;
    if (post) {
        param8<MODE>(a.post_w, a.param_f32, c, n, 1.f, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = i < n ? (f[i] - st[0]) * st[1] : 0.f;
    }
    if (a.gate) {
        float dg[8];
        if (post) {
            param8<MODE>(a.post_b, a.param_f32, c, n, 0.f, b);
#pragma unroll
            for (int i = 0; i < 8; ++i) dg[i] = g[i] * __builtin_fmaf(f[i], w[i], b[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) dg[i] = g[i] * f[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] *= q[i];
        if (direct_gate) {
            if (n > 0 && a.dgate) store8<VEC>(static_cast<T *>(a.dgate) + at, n, dg);
        } else if constexpr (FULL) {
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[S_GATE][i] += dg[i];
        }
    }
    if (post) {
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            sum[S_POST_W][i] = __builtin_fmaf(g[i], f[i], sum[S_POST_W][i]);
            if constexpr (FULL) sum[S_POST_B][i] += g[i];
            g[i] = i < n ? g[i] * w[i] : 0.f;
            s1 = __builtin_fmaf(g[i], f[i], s1);
            s2 += g[i];
        }
        s1 = row_sum<TPR>(s1, lds) * inv_c;
        s2 = a.post == 2 ? row_sum<TPR>(s2, lds) * inv_c : 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = st[1] * __builtin_fmaf(-f[i], s1, g[i] - s2);
    }
    if (n > 0 && (USUAL || a.df)) store8<VEC>(static_cast<T *>(a.df) + at, n, g);
}

// One column sum of the workgroup's rows in flight, in their order, to out[C] (f32)
template <int TPR>
__device__ __forceinline__ void write_sum(float (&v)[8], float *out, int C, int c, float *lds) {
    constexpr int SLOTS = threads<TPR>() / TPR;
    if constexpr (SLOTS > 1) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) lds[threadIdx.x * 8 + i] = v[i];
        __syncthreads();
        for (int e = threadIdx.x; e < TPR * 8; e += NT) {
            float s = 0.f;
            for (int t = 0; t < SLOTS; ++t) s += lds[t * TPR * 8 + e];
            if (e < C) out[e] = s;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < C) out[c + i] = v[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
}

// grid (splits, groups in flight).  A gate row's rows (all rows without a gate) are cut into
// `splits` runs; the gate's column sum ends with each run, the parameters' run on.  With a gate
// for each row the workgroups share all rows and write its gradient directly.
template <class T, int TPR, int MODE, bool FULL>
__global__ __launch_bounds__(threads<TPR>()) void block_bwd(Block a) {
    constexpr int SLOTS = threads<TPR>() / TPR, NSUM = sums<FULL>();
    __shared__ float lds[SLOTS > 1 ? NT * 8 : 16];
    const int c = threadIdx.x % TPR * 8, slot = threadIdx.x / TPR;
    const uint64_t seed = a.rng.step ? rng_seed(a.rng) : 0;
    const float inv_c = 1.f / (float)a.C;
    float sum[NSUM][8];
#pragma unroll
    for (int s = 0; s < NSUM; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[s][i] = 0.f;
    const bool direct = a.gate && a.gate_rows == 1;
    const int len = direct || !a.gate ? a.R : a.gate_rows, groups = a.R / len;
    for (int g = blockIdx.y; g < groups; g += gridDim.y) {
        const int run = (len + a.splits - 1) / a.splits;
        const int first = min((int)blockIdx.x * run, len), last = min(first + run, len);
        for (int r = first + slot; r < last; r += SLOTS)
            back_row<T, TPR, MODE, FULL>(a, g * len + r, c, seed, direct, inv_c, lds, sum);
        if constexpr (FULL)
            if (a.gpart) write_sum<TPR>(sum[S_GATE], a.gpart + ((int64_t)g * a.splits + blockIdx.x) * a.C, a.C, c, lds);
    }
    const int64_t part = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
#pragma unroll
    for (int s = 0; s < (FULL ? S_GATE : NSUM); ++s)
        if (a.want >> s & 1) write_sum<TPR>(sum[s], a.part + (part * 4 + s) * a.C, a.C, c, lds);
}

// out[s][c] = sum over n of in[s * stride_s + n * stride_n + c], eight lanes a column, one order
struct Reduce {
    const float *in;
    void *out[4];
    int64_t stride_s, stride_n, out_stride;
    int n, C, f32;
};
__global__ __launch_bounds__(NT) void sum_parts(Reduce a) {
    __shared__ float lds[NT];
    const int c = blockIdx.x * 32 + threadIdx.x % 32, lane = threadIdx.x / 32, s = blockIdx.y;
    void *out = a.out_stride ? a.out[0] : a.out[s];
    float v = 0.f;
    if (c < a.C && out)
#pragma unroll 8
        for (int n = lane; n < a.n; n += 8) v += a.in[s * a.stride_s + n * a.stride_n + c];
    lds[threadIdx.x] = v;
    __syncthreads();
    if (lane == 0 && c < a.C && out) {
        for (int t = 1; t < 8; ++t) v += lds[t * 32 + threadIdx.x];
        const int64_t at = s * a.out_stride + c;
        if (a.f32) static_cast<float *>(out)[at] = v;
        else static_cast<__bf16 *>(out)[at] = (__bf16)v;
    }
}

// ------------------------------------------------------------------- C interface --

Rng make_rng(uint32_t step, uint64_t seed, const uint64_t *dev, uint32_t site) {
    return {seed, dev, site, step, 65536.f / (65536.f - (float)step)};
}

bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// threads of a row
int row_threads(int C) { return C <= 128 ? 16 : C <= 256 ? 32 : C <= 512 ? 64 : C <= 1024 ? 128 : C <= 2048 ? 256 : C <= 4096 ? 512 : 1024; }

// whether the backward pass sums more columns than the norms' weights
bool full_sums(const hreg_tok_block_t *p) { return (p->gate && p->gate_rows > 1 && p->dgate) || p->dpost_b || p->dpre_b; }

// How the backward pass divides its rows: splits of a gate row's rows, gate rows in flight.  As many
// workgroups as the registers let run (12 or 16 waves a CU; rows of 4096 bf16, us: 240 with 16, 274
// with 12, 247 with 24; rows of 1024 with biases 142 with 12, 178 with 16), but four rows a thread
// at least: each workgroup's column sums are written and read once more.
struct Plan { int splits, flight, groups; };
Plan plan_of(const hreg_tok_block_t *p) {
    const int len = p->gate && p->gate_rows > 1 ? p->gate_rows : p->R, tpr = row_threads(p->C);
    const int waves = tpr > 64 ? tpr / 64 : 4, slots = tpr > 64 ? 1 : NT / tpr, most = 256 * (full_sums(p) ? 12 : 16) / waves;
    Plan q;
    q.groups = len ? p->R / len : 0;
    q.flight = q.groups < most ? (q.groups > 0 ? q.groups : 1) : most;
    q.splits = most / q.flight;
    const int rows = (len + 4 * slots - 1) / (4 * slots);
    if (q.splits > rows) q.splits = rows;
    if (q.splits < 1) q.splits = 1;
    return q;
}

size_t part_bytes(const hreg_tok_block_t *p, const Plan &q) {
    return ((size_t)q.splits * q.flight * 4 * p->C * 4 + 255) / 256 * 256;
}

int take(const hreg_tok_block_t *p, Block &a) {
    if (!p || (p->dtype != HREG_TOK_F32 && p->dtype != HREG_TOK_BF16) ||
        (p->param_dtype != HREG_TOK_F32 && p->param_dtype != HREG_TOK_BF16))
        return HREG_ERR_INVALID;
    if (p->R < 0 || p->C < 1 || p->post < 0 || p->post > 2 || p->pre < 0 || p->pre > 2 || p->step > 65535) return HREG_ERR_INVALID;
    if (p->C > 8192 || p->R > (1 << 30)) return HREG_ERR_UNSUPPORTED;
    if (p->gate && (p->gate_rows < 1 || p->R % p->gate_rows || (p->R > 0 && !p->f))) return HREG_ERR_INVALID;
    a = Block{};
    a.x = p->x; a.f = p->f; a.gate = p->gate; a.post_w = p->post_w; a.post_b = p->post_b; a.pre_w = p->pre_w;
    a.pre_b = p->pre_b; a.dy = p->dy; a.dh = p->dh; a.y = p->y; a.h = p->h; a.dx = p->dx; a.df = p->df; a.dgate = p->dgate;
    a.stats = p->stats; a.R = p->R; a.C = p->C; a.gate_rows = p->gate ? p->gate_rows : 1;
    a.post = p->f ? p->post : 0; a.pre = p->pre; a.param_f32 = p->param_dtype == HREG_TOK_F32;
    a.scale = p->scale; a.eps = p->eps;
    a.rng = make_rng(p->f ? p->step : 0, p->seed, p->seed_dev, p->site);
    return HREG_OK;
}

template <bool BACK, class T, int TPR, int MODE>
int go(const Block &a, const Plan &q, void *stream) {
    const dim3 block(threads<TPR>());
    if constexpr (BACK) {
        const bool full = MODE == SINGLE || a.gpart || a.want >> S_POST_B;
        if constexpr (MODE != SINGLE) {
            if (!full) hipLaunchKernelGGL((block_bwd<T, TPR, MODE, false>), dim3(q.splits, q.flight), block, 0, as_stream(stream), a);
        }
        if (full) hipLaunchKernelGGL((block_bwd<T, TPR, MODE, true>), dim3(q.splits, q.flight), block, 0, as_stream(stream), a);
    } else {
        constexpr int SLOTS = threads<TPR>() / TPR;
        hipLaunchKernelGGL((block_fwd<T, TPR, MODE>), grid_of((a.R + SLOTS - 1) / SLOTS), block, 0, as_stream(stream), a);
    }
    HREG_CHECK_LAUNCH();
    return HREG_OK;
}

template <bool BACK, class T, int TPR>
int by_mode(const Block &a, int mode, const Plan &q, void *stream) {
    return mode == WHOLE     ? go<BACK, T, TPR, WHOLE>(a, q, stream)
           : mode == ALIGNED ? go<BACK, T, TPR, ALIGNED>(a, q, stream)
                             : go<BACK, T, TPR, SINGLE>(a, q, stream);
}

template <bool BACK, class T>
int by_width(const Block &a, int mode, const Plan &q, void *stream) {
    switch (row_threads(a.C)) {
        case 16: return by_mode<BACK, T, 16>(a, mode, q, stream);
        case 32: return by_mode<BACK, T, 32>(a, mode, q, stream);
        case 64: return by_mode<BACK, T, 64>(a, mode, q, stream);
        case 128: return by_mode<BACK, T, 128>(a, mode, q, stream);
        case 256: return by_mode<BACK, T, 256>(a, mode, q, stream);
        case 512: return by_mode<BACK, T, 512>(a, mode, q, stream);
        default: return by_mode<BACK, T, 1024>(a, mode, q, stream);
    }
}

template <bool BACK>
int by_type(const hreg_tok_block_t *p, const Block &a, const Plan &q, void *stream) {
    bool vec = a.C % 8 == 0;  // rows and parameters in 16-byte steps
    for (const void *v : {a.x, a.f, a.gate, a.post_w, a.post_b, a.pre_w, a.pre_b, a.dy, a.dh, (const void *)a.y,
                          (const void *)a.h, (const void *)a.dx, (const void *)a.df, (const void *)a.dgate})
        vec = vec && aligned16(v);
    const bool usual = a.f && a.post && a.pre && (!BACK || (a.dy && a.dh && a.dx && a.df));
    const int mode = !vec ? SINGLE : usual && a.C == 8 * row_threads(a.C) ? WHOLE : ALIGNED;
    return p->dtype == HREG_TOK_F32 ? by_width<BACK, float>(a, mode, q, stream) : by_width<BACK, __bf16>(a, mode, q, stream);
}

}  // namespace

extern "C" {

int hreg_tok_dropout(const void *x, void *y, int64_t n, int dtype, uint32_t step, uint64_t seed,
                     const uint64_t *seed_dev, uint32_t site, void *stream) {
    if (n < 0 || step > 65535 || (dtype != HREG_TOK_F32 && dtype != HREG_TOK_BF16)) return HREG_ERR_INVALID;
    if (n == 0) return HREG_OK;
    if (!x || !y) return HREG_ERR_INVALID;
    const int64_t grid = (n + 8 * NT - 1) / (8 * NT);
    if (grid > (int64_t)65535 << 21) return HREG_ERR_UNSUPPORTED;
    const Rng g = make_rng(step, seed, seed_dev, site);
    const bool vec = aligned16(x) && aligned16(y);
    const hipStream_t st = as_stream(stream);
    if (dtype == HREG_TOK_F32) {
        const float *s = static_cast<const float *>(x);
        float *d = static_cast<float *>(y);
        if (vec) hipLaunchKernelGGL((dropout_kernel<float, true>), grid_of(grid), dim3(NT), 0, st, s, d, n, g);
        else hipLaunchKernelGGL((dropout_kernel<float, false>), grid_of(grid), dim3(NT), 0, st, s, d, n, g);
    } else {
        const __bf16 *s = static_cast<const __bf16 *>(x);
        __bf16 *d = static_cast<__bf16 *>(y);
        if (vec) hipLaunchKernelGGL((dropout_kernel<__bf16, true>), grid_of(grid), dim3(NT), 0, st, s, d, n, g);
        else hipLaunchKernelGGL((dropout_kernel<__bf16, false>), grid_of(grid), dim3(NT), 0, st, s, d, n, g);
    }
    HREG_CHECK_LAUNCH();
    return HREG_OK;
}

size_t hreg_tok_block_ws_bytes(const hreg_tok_block_t *p) {
    if (!p || p->R < 1 || p->C < 1 || (p->gate && (p->gate_rows < 1 || p->R % p->gate_rows))) return 0;
    const Plan q = plan_of(p);
    const bool sums = p->gate && p->gate_rows > 1;
    return part_bytes(p, q) + (sums ? (size_t)q.groups * q.splits * p->C * 4 : 0);
}

int hreg_tok_block_fwd(const hreg_tok_block_t *p, void *stream) {
    Block a;
    const int rc = take(p, a);
    if (rc != HREG_OK) return rc;
    if (a.R == 0) return HREG_OK;
    if (!a.x || (a.f && !a.y) || (a.pre && !a.h) || (!a.f && !a.pre) || (a.stats && !aligned16(a.stats))) return HREG_ERR_INVALID;
    return by_type<false>(p, a, Plan{}, stream);
}

int hreg_tok_block_bwd(const hreg_tok_block_t *p, void *stream) {
    Block a;
    int rc = take(p, a);
    if (rc != HREG_OK) return rc;
    const bool post = a.R == 0 || (a.f && a.post), pre = a.R == 0 || a.pre;
    void *const out[4] = {post ? p->dpost_w : nullptr, pre ? p->dpre_w : nullptr, post ? p->dpost_b : nullptr,
                          pre ? p->dpre_b : nullptr};
    for (int s = 0; s < 4; ++s) a.want |= (out[s] != nullptr) << s;
    Plan q{1, 1, 0};
    if (a.R > 0) {
        if (!a.stats || !aligned16(a.stats) || (a.pre && !a.y)) return HREG_ERR_INVALID;
        const size_t need = hreg_tok_block_ws_bytes(p);
        if (!p->ws || p->ws_bytes < need || reinterpret_cast<uintptr_t>(p->ws) % 256) return HREG_ERR_INVALID;
        q = plan_of(p);
        a.splits = q.splits;
        a.part = static_cast<float *>(p->ws);
        if (a.gate && a.gate_rows > 1 && a.dgate) a.gpart = reinterpret_cast<float *>(static_cast<char *>(p->ws) + part_bytes(p, q));
        rc = by_type<true>(p, a, q, stream);
        if (rc != HREG_OK) return rc;
    }
    const int cols = (a.C + 31) / 32;
    if (a.want) {  // zero rows too: the sums are zero
        Reduce r{a.part, {out[0], out[1], out[2], out[3]}, a.C, (int64_t)4 * a.C, 0, a.R > 0 ? q.splits * q.flight : 0, a.C,
                 a.param_f32};
        hipLaunchKernelGGL(sum_parts, dim3(cols, 4), dim3(NT), 0, as_stream(stream), r);
        HREG_CHECK_LAUNCH();
    }
    for (int g0 = 0; a.gpart && g0 < q.groups; g0 += 65535) {  // the gate's rows
        const int n = q.groups - g0 < 65535 ? q.groups - g0 : 65535;
        const size_t es = p->dtype == HREG_TOK_F32 ? 4 : 2;
        Reduce r{a.gpart + (int64_t)g0 * q.splits * a.C, {static_cast<char *>(a.dgate) + (size_t)g0 * a.C * es},
                 (int64_t)q.splits * a.C, a.C, a.C, q.splits, a.C, p->dtype == HREG_TOK_F32};
        hipLaunchKernelGGL(sum_parts, dim3(cols, n), dim3(NT), 0, as_stream(stream), r);
        HREG_CHECK_LAUNCH();
    }
    return HREG_OK;
}

}  // extern "C"
