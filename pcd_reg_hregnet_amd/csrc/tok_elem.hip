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

// the 16 bits of elements first .. first + 7, two a word; first need not be a multiple of eight
__device__ __forceinline__ u32x4 bits_of(uint64_t first, uint32_t site, uint64_t seed) {
    const u32x4 a = philox(first >> 3, site, seed);
    const int off = first & 7;
    if (off == 0) return a;
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
__device__ __forceinline__ void mask_of(const Rng &g, uint64_t first, uint64_t seed, float (&m)[8]) {
    const u32x4 w = bits_of(first, g.site, seed);
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

template <class T, bool VEC>
__global__ __launch_bounds__(NT) void dropout_kernel(const T *__restrict__ x, T *__restrict__ y, int64_t n, Rng g) {
    const int64_t at = ((int64_t)blockIdx.x * NT + threadIdx.x) * 8;
    if (at >= n) return;
    float v[8], m[8];
    const int have = (int)min((int64_t)8, n - at);
    if (VEC && have == 8) load8<true>(x + at, 8, v);
    else load8<false>(x + at, have, v);
    mask_of(g, at, rng_seed(g), m);
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
    int R, C, gate_rows, post, pre, param_f32, splits, want;  // want: bit k = column sum k
    float scale, eps;
    Rng rng;
};

// a parameter's elements c .. c + 7, `other` where there is no such parameter
template <bool VEC>
__device__ __forceinline__ void param8(const void *p, int f32, int c, int n, float other, float (&v)[8]) {
    if (!p) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = other;
    } else if (f32) load8<VEC>(static_cast<const float *>(p) + c, n, v);
    else load8<VEC>(static_cast<const __bf16 *>(p) + c, n, v);
}

// sum over the TPR threads of a row, in every one of them
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float *lds) {
    if constexpr (TPR == 16) return row_sum16(v);
    v = row_sum16(v);
    v = fadd_rn(v, __shfl_xor(v, 16));
    if constexpr (TPR >= 64) v = fadd_rn(v, __shfl_xor(v, 32));
    if constexpr (TPR > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = fadd_rn(fadd_rn(lds[0], lds[1]), fadd_rn(lds[2], lds[3]));
    }
    return v;
}

// mean and 1 / deviation of a row held in registers (two passes: the mean, then the squares
// around it)
template <int TPR, int NCH>
__device__ __forceinline__ void row_stats(const float (&v)[NCH][8], int kind, int C, int c0, float eps, float &mu, float &rs,
                                          float *lds) {
    mu = 0.f;
    if (kind == 2) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < NCH; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) s += v[k][i];  // 0 beyond C
        mu = row_sum<TPR>(s, lds) / (float)C;
    }
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < NCH; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float d = c0 + k * TPR * 8 + i < C ? v[k][i] - mu : 0.f;
            s = __builtin_fmaf(d, d, s);
        }
    rs = 1.f / sqrtf(row_sum<TPR>(s, lds) / (float)C + eps);
}

// One row a TPR threads, NCH groups of eight elements a thread: every input is read once and
// stays in registers through both norms.  Bound by its bytes.
template <class T, int TPR, int NCH, bool VEC>
__global__ __launch_bounds__(NT) void block_fwd(Block a) {
    __shared__ float lds[4];
    const int r = blockIdx.x * (NT / TPR) + threadIdx.x / TPR, C = a.C, c0 = threadIdx.x % TPR * 8;
    if (TPR <= 64 && r >= a.R) return;
    const int64_t row = (int64_t)r * C;
    float y[NCH][8];
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
        const int c = c0 + k * TPR * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) y[k][i] = 0.f;
        if (c < C) load8<VEC>(static_cast<const T *>(a.x) + row + c, C - c, y[k]);
    }
    float mu = 0.f, rs = 1.f, mu2 = 0.f, rs2 = 1.f;
    if (a.f) {
        float u[NCH][8];
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            const int c = c0 + k * TPR * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i) u[k][i] = 0.f;
            if (c < C) load8<VEC>(static_cast<const T *>(a.f) + row + c, C - c, u[k]);
        }
        if (a.post) row_stats<TPR, NCH>(u, a.post, C, c0, a.eps, mu, rs, lds);
        const uint64_t seed = a.rng.step ? rng_seed(a.rng) : 0;
        const int64_t grow = a.gate ? (int64_t)(r / a.gate_rows) * C : 0;
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            const int c = c0 + k * TPR * 8;
            if (c >= C) continue;
            float w[8], b[8], g[8], m[8];
            if (a.post) {
                param8<VEC>(a.post_w, a.param_f32, c, C - c, 1.f, w);
                param8<VEC>(a.post_b, a.param_f32, c, C - c, 0.f, b);
#pragma unroll
                for (int i = 0; i < 8; ++i) u[k][i] = __builtin_fmaf((u[k][i] - mu) * rs, w[i], b[i]);
            }
            if (a.rng.step) {
                mask_of(a.rng, row + c, seed, m);
#pragma unroll
                for (int i = 0; i < 8; ++i) u[k][i] = m[i] != 0.f ? u[k][i] * m[i] : 0.f;
            }
            if (a.gate) {
                load8<VEC>(static_cast<const T *>(a.gate) + grow + c, C - c, g);
#pragma unroll
                for (int i = 0; i < 8; ++i) u[k][i] *= g[i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) y[k][i] = c + i < C ? __builtin_fmaf(a.scale, u[k][i], y[k][i]) : 0.f;
            store8<VEC>(static_cast<T *>(a.y) + row + c, C - c, y[k]);
        }
    }
    if (a.pre) {
        row_stats<TPR, NCH>(y, a.pre, C, c0, a.eps, mu2, rs2, lds);
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            const int c = c0 + k * TPR * 8;
            if (c >= C) continue;
            float w[8], b[8];
            param8<VEC>(a.pre_w, a.param_f32, c, C - c, 1.f, w);
            param8<VEC>(a.pre_b, a.param_f32, c, C - c, 0.f, b);
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = __builtin_fmaf((y[k][i] - mu2) * rs2, w[i], b[i]);
            store8<VEC>(static_cast<T *>(a.h) + row + c, C - c, w);
        }
    }
    if (a.stats && threadIdx.x % TPR == 0) *reinterpret_cast<f32x4_m *>(a.stats + 4 * (int64_t)r) = f32x4{mu, rs, mu2, rs2};
}

// Column sums of the backward pass, in this order: the four parameters' and the gate's.
enum { S_POST_W, S_POST_B, S_PRE_W, S_PRE_B, S_GATE, NSUM };

// Rows first + slot, first + slot + slots, ... < last: gradients of the rows, column sums in
// registers.  The statistics are the forward pass's; everything else is computed again.
// Bound by its bytes (f, y, dy, dh and the gate read, dx, df and the gate's gradient written).
template <class T, int TPR, int NCH, bool VEC>
__device__ __forceinline__ void back_row(const Block &a, int r, int c0, uint64_t seed, bool direct_gate, float *lds,
                                         float (&sum)[NSUM][NCH][8]) {
    const int C = a.C;
    const int64_t row = (int64_t)r * C;
    const f32x4 st = *reinterpret_cast<const f32x4_m *>(a.stats + 4 * (int64_t)r);
    float dx[NCH][8], n[NCH][8], g[NCH][8];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
        const int c = c0 + k * TPR * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) dx[k][i] = n[k][i] = g[k][i] = 0.f;
        if (c >= C) continue;
        if (a.dy) load8<VEC>(static_cast<const T *>(a.dy) + row + c, C - c, dx[k]);
        if (a.pre && a.dh) {
            float w[8];
            load8<VEC>(static_cast<const T *>(a.dh) + row + c, C - c, g[k]);
            load8<VEC>(static_cast<const T *>(a.y) + row + c, C - c, n[k]);
            param8<VEC>(a.pre_w, a.param_f32, c, C - c, 1.f, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                n[k][i] = c + i < C ? (n[k][i] - st[2]) * st[3] : 0.f;
                sum[S_PRE_W][k][i] = __builtin_fmaf(g[k][i], n[k][i], sum[S_PRE_W][k][i]);
                sum[S_PRE_B][k][i] += g[k][i];
                g[k][i] *= w[i];
                if (c + i >= C) g[k][i] = 0.f;
                s1 = __builtin_fmaf(g[k][i], n[k][i], s1);
                s2 += g[k][i];
            }
        }
    }
    if (a.pre && a.dh) {
        s1 = row_sum<TPR>(s1, lds) / (float)C;
        s2 = a.pre == 2 ? row_sum<TPR>(s2, lds) / (float)C : 0.f;
#pragma unroll
        for (int k = 0; k < NCH; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) dx[k][i] += st[3] * (g[k][i] - n[k][i] * s1 - s2);
    }
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
        const int c = c0 + k * TPR * 8;
        if (c < C && a.dx) store8<VEC>(static_cast<T *>(a.dx) + row + c, C - c, dx[k]);
    }
    if (!a.f) return;
    s1 = s2 = 0.f;
    const int64_t grow = a.gate ? (int64_t)(r / a.gate_rows) * C : 0;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
        const int c = c0 + k * TPR * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) n[k][i] = g[k][i] = 0.f;
        if (c >= C) continue;
        float w[8], b[8], m[8], q[8];
        load8<VEC>(static_cast<const T *>(a.f) + row + c, C - c, n[k]);
        param8<VEC>(a.post_w, a.param_f32, c, C - c, 1.f, w);
        param8<VEC>(a.post_b, a.param_f32, c, C - c, 0.f, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) g[k][i] = c + i < C ? dx[k][i] * a.scale : 0.f;
        if (a.rng.step) {
            mask_of(a.rng, row + c, seed, m);
#pragma unroll
            for (int i = 0; i < 8; ++i) g[k][i] = m[i] != 0.f ? g[k][i] * m[i] : 0.f;
        }
        if (a.post) {
#pragma unroll
            for (int i = 0; i < 8; ++i) n[k][i] = c + i < C ? (n[k][i] - st[0]) * st[1] : 0.f;
        }
        if (a.gate) {
            load8<VEC>(static_cast<const T *>(a.gate) + grow + c, C - c, q);
            float dg[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                dg[i] = g[k][i] * (a.post ? __builtin_fmaf(n[k][i], w[i], b[i]) : n[k][i]);
                g[k][i] *= q[i];
            }
            if (direct_gate) {
                if (a.dgate) store8<VEC>(static_cast<T *>(a.dgate) + row + c, C - c, dg);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) sum[S_GATE][k][i] += dg[i];
            }
        }
        if (a.post) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                sum[S_POST_W][k][i] = __builtin_fmaf(g[k][i], n[k][i], sum[S_POST_W][k][i]);
                sum[S_POST_B][k][i] += g[k][i];
                g[k][i] = c + i < C ? g[k][i] * w[i] : 0.f;
                s1 = __builtin_fmaf(g[k][i], n[k][i], s1);
                s2 += g[k][i];
            }
        }
    }
    if (a.post) {
        s1 = row_sum<TPR>(s1, lds) / (float)C;
        s2 = a.post == 2 ? row_sum<TPR>(s2, lds) / (float)C : 0.f;
    }
    if (!a.df) return;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
        const int c = c0 + k * TPR * 8;
        if (c >= C) continue;
        if (a.post)
#pragma unroll
            for (int i = 0; i < 8; ++i) g[k][i] = st[1] * (g[k][i] - n[k][i] * s1 - s2);
        store8<VEC>(static_cast<T *>(a.df) + row + c, C - c, g[k]);
    }
}

// One column sum of the workgroup's row slots, in slot order, to out[C] (f32)
template <int TPR, int NCH>
__device__ __forceinline__ void write_sum(float (&v)[NCH][8], float *out, int C, int c0, float *lds) {
    constexpr int SLOTS = NT / TPR;
    if constexpr (SLOTS > 1) {
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 8; ++i) lds[threadIdx.x * 8 + i] = v[k][i];
            __syncthreads();
            for (int e = threadIdx.x; e < TPR * 8; e += NT) {
                const int c = k * TPR * 8 + e;
                float s = 0.f;
                for (int t = 0; t < SLOTS; ++t) s += lds[t * TPR * 8 + e];
                if (c < C) out[c] = s;
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < NCH; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c0 + k * TPR * 8 + i < C) out[c0 + k * TPR * 8 + i] = v[k][i];
    }
#pragma unroll
    for (int k = 0; k < NCH; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[k][i] = 0.f;
}

// grid (splits, groups in flight).  A gate row's rows (all rows without a gate) are cut into
// `splits` runs; the gate's column sum ends with each run, the parameters' run on.  With a gate
// for each row the workgroups share all rows and write its gradient directly.
template <class T, int TPR, int NCH, bool VEC>
__global__ __launch_bounds__(NT) void block_bwd(Block a) {
    __shared__ float lds[NT * 8];
    constexpr int SLOTS = NT / TPR;
    const int c0 = threadIdx.x % TPR * 8, slot = threadIdx.x / TPR;
    const uint64_t seed = a.rng.step ? rng_seed(a.rng) : 0;
    float sum[NSUM][NCH][8];
#pragma unroll
    for (int s = 0; s < NSUM; ++s)
#pragma unroll
        for (int k = 0; k < NCH; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[s][k][i] = 0.f;
    const bool direct = a.gate && a.gate_rows == 1;
    const int len = direct || !a.gate ? a.R : a.gate_rows, groups = a.R / len;
    for (int g = blockIdx.y; g < groups; g += gridDim.y) {
        const int run = (len + a.splits - 1) / a.splits;
        const int first = min((int)blockIdx.x * run, len), last = min(first + run, len);
        for (int r = first + slot; r < last; r += SLOTS)
            back_row<T, TPR, NCH, VEC>(a, g * len + r, c0, seed, direct, lds, sum);
        if (a.gpart)
            write_sum<TPR, NCH>(sum[S_GATE], a.gpart + ((int64_t)g * a.splits + blockIdx.x) * a.C, a.C, c0, lds);
    }
    const int64_t part = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
#pragma unroll
    for (int s = 0; s < S_GATE; ++s)
        if (a.want >> s & 1) write_sum<TPR, NCH>(sum[s], a.part + (part * 4 + s) * a.C, a.C, c0, lds);
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

// how the backward pass divides its rows: splits of a gate row's rows, gate rows in flight
struct Plan { int splits, flight, groups; };
Plan plan_of(int R, int gate_rows, bool gate) {
    const int len = gate && gate_rows > 1 ? gate_rows : R, groups = len ? R / len : 0;
    Plan p;
    p.groups = groups;
    p.flight = groups < 512 ? (groups > 0 ? groups : 1) : 512;
    p.splits = 512 / p.flight;
    if (p.splits > (len + 7) / 8) p.splits = (len + 7) / 8;
    if (p.splits < 1) p.splits = 1;
    return p;
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

template <bool BACK, class T, int TPR, int NCH, bool VEC>
int go(const Block &a, const Plan &q, void *stream) {
    if constexpr (BACK) {
        hipLaunchKernelGGL((block_bwd<T, TPR, NCH, VEC>), dim3(q.splits, q.flight), dim3(NT), 0, as_stream(stream), a);
    } else {
        constexpr int SLOTS = NT / TPR;
        hipLaunchKernelGGL((block_fwd<T, TPR, NCH, VEC>), dim3((a.R + SLOTS - 1) / SLOTS), dim3(NT), 0, as_stream(stream), a);
    }
    HREG_CHECK_LAUNCH();
    return HREG_OK;
}

template <bool BACK, class T, bool VEC>
int by_width(const Block &a, const Plan &q, void *stream) {
    if (a.C <= 128) return go<BACK, T, 16, 1, VEC>(a, q, stream);
    if (a.C <= 256) return go<BACK, T, 32, 1, VEC>(a, q, stream);
    if (a.C <= 512) return go<BACK, T, 64, 1, VEC>(a, q, stream);
    if (a.C <= 1024) return go<BACK, T, 64, 2, VEC>(a, q, stream);
    if (a.C <= 2048) return go<BACK, T, 256, 1, VEC>(a, q, stream);
    if (a.C <= 4096) return go<BACK, T, 256, 2, VEC>(a, q, stream);
    return go<BACK, T, 256, 4, VEC>(a, q, stream);
}

template <bool BACK>
int by_type(const hreg_tok_block_t *p, const Block &a, const Plan &q, void *stream) {
    bool vec = a.C % 8 == 0;  // rows and parameters in 16-byte steps
    for (const void *v : {a.x, a.f, a.gate, a.post_w, a.post_b, a.pre_w, a.pre_b, a.dy, a.dh, (const void *)a.y,
                          (const void *)a.h, (const void *)a.dx, (const void *)a.df, (const void *)a.dgate})
        vec = vec && aligned16(v);
    if (p->dtype == HREG_TOK_F32)
        return vec ? by_width<BACK, float, true>(a, q, stream) : by_width<BACK, float, false>(a, q, stream);
    return vec ? by_width<BACK, __bf16, true>(a, q, stream) : by_width<BACK, __bf16, false>(a, q, stream);
}

}  // namespace

extern "C" {

int hreg_tok_dropout(const void *x, void *y, int64_t n, int dtype, uint32_t step, uint64_t seed,
                     const uint64_t *seed_dev, uint32_t site, void *stream) {
    if (n < 0 || step > 65535 || (dtype != HREG_TOK_F32 && dtype != HREG_TOK_BF16)) return HREG_ERR_INVALID;
    if (n == 0) return HREG_OK;
    if (!x || !y) return HREG_ERR_INVALID;
    const int64_t grid = (n + 8 * NT - 1) / (8 * NT);
    if (grid > INT32_MAX) return HREG_ERR_UNSUPPORTED;
    const Rng g = make_rng(step, seed, seed_dev, site);
    const bool vec = aligned16(x) && aligned16(y);
    const hipStream_t st = as_stream(stream);
    if (dtype == HREG_TOK_F32) {
        const float *s = static_cast<const float *>(x);
        float *d = static_cast<float *>(y);
        if (vec) hipLaunchKernelGGL((dropout_kernel<float, true>), dim3(grid), dim3(NT), 0, st, s, d, n, g);
        else hipLaunchKernelGGL((dropout_kernel<float, false>), dim3(grid), dim3(NT), 0, st, s, d, n, g);
    } else {
        const __bf16 *s = static_cast<const __bf16 *>(x);
        __bf16 *d = static_cast<__bf16 *>(y);
        if (vec) hipLaunchKernelGGL((dropout_kernel<__bf16, true>), dim3(grid), dim3(NT), 0, st, s, d, n, g);
        else hipLaunchKernelGGL((dropout_kernel<__bf16, false>), dim3(grid), dim3(NT), 0, st, s, d, n, g);
    }
    HREG_CHECK_LAUNCH();
    return HREG_OK;
}

size_t hreg_tok_block_ws_bytes(const hreg_tok_block_t *p) {
    if (!p || p->R < 1 || p->C < 1 || (p->gate && (p->gate_rows < 1 || p->R % p->gate_rows))) return 0;
    const Plan q = plan_of(p->R, p->gate_rows, p->gate != nullptr);
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
    void *const out[4] = {post ? p->dpost_w : nullptr, post ? p->dpost_b : nullptr, pre ? p->dpre_w : nullptr,
                          pre ? p->dpre_b : nullptr};
    for (int s = 0; s < 4; ++s) a.want |= (out[s] != nullptr) << s;
    Plan q{1, 1, 0};
    if (a.R > 0) {
        if (!a.stats || !aligned16(a.stats) || (a.pre && !a.y)) return HREG_ERR_INVALID;
        const size_t need = hreg_tok_block_ws_bytes(p);
        if (!p->ws || p->ws_bytes < need || reinterpret_cast<uintptr_t>(p->ws) % 256) return HREG_ERR_INVALID;
        q = plan_of(p->R, p->gate_rows, p->gate != nullptr);
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
