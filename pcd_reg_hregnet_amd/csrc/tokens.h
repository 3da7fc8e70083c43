// tokens.h -- what the token operators (tok_attn.hip, tok_elem.hip) share: element types,
// the exact bf16 pieces of f32 values, swizzled LDS tiles and their MFMA fragments.
#pragma once

#include "common.h"

namespace hreg_tok {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
// LDS and global memory are read and written through these, whatever their declared type
typedef u32x4 __attribute__((may_alias)) u32x4_m;
typedef u32x2 __attribute__((may_alias)) u32x2_m;
typedef f32x4 __attribute__((may_alias)) f32x4_m;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(1))) const void glob_void;

// A product of two T values is NP * (NP + 1) / 2 bf16 matrix products of their pieces: one
// for bf16; six for f32, whose values are the exact sum of three bf16 pieces.  The pieces are cut, not
// rounded: the second lies below 2^-7 of the first, the third below 2^-15.  The three smallest of the
// nine piece products are left out: each below 2^-22 of the largest, together up to just above 2^-21 of the
// product and 0.7 x 2^-24 on average (normal values), always of the product's own sign.
template <class T> struct Elem;
template <> struct Elem<__bf16> { static constexpr int NP = 1; };
template <> struct Elem<float> { static constexpr int NP = 3; };

// rounds to nearest even: bf16 storage of an f32 result, off by at most 2^-8 of it
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const bf16x2 v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.f;
    return z;
}

// eight values as the NP operand pieces of one lane of a 16-deep product chunk.  NP = 1 rounds
// to bf16; NP = 2 rounds, and rounds the rest; NP = 3 cuts 8 + 8 + 8 significant bits (exact for
// normal f32).
template <int NP>
__device__ __forceinline__ void to_pieces(const float (&x)[8], bf16x8 (&p)[NP]) {
    u32x4 w[NP];
    if constexpr (NP == 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[0][i] = pack_bf16(x[2 * i], x[2 * i + 1]);
    } else if constexpr (NP == 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[0][i] = pack_bf16(x[2 * i], x[2 * i + 1]);
            w[1][i] = pack_bf16(x[2 * i] - bf16_lo(w[0][i]), x[2 * i + 1] - bf16_hi(w[0][i]));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
            for (int s = 0; s < NP; ++s) {
                const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
                w[s][i] = __builtin_amdgcn_perm(ub, ua, 0x07060302u);
                if (s + 1 < NP) {
                    a = fsub_rn(a, __uint_as_float(ua & 0xffff0000u));
                    b = fsub_rn(b, __uint_as_float(ub & 0xffff0000u));
                }
            }
        }
    }
#pragma unroll
    for (int s = 0; s < NP; ++s) p[s] = __builtin_bit_cast(bf16x8, w[s]);
}

// acc += A B on v_mfma_f32_32x32x16_bf16 (A bf16 itself, B in NB pieces, or both f32).  Lane l: column / row l & 31, depth 8 (l >> 5) + i;
// result register r: row 8 (r >> 2) + 4 (l >> 5) + (r & 3), column l & 31.  Smallest first.
template <int NP, int NB>
__device__ __forceinline__ void mma(f32x16 &acc, const bf16x8 (&a)[NP], const bf16x8 (&b)[NB]) {
    static_assert(NP == NB || NP == 1, "pieces");
    if constexpr (NP == 1) {
#pragma unroll
        for (int s = NB - 1; s >= 0; --s) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[s], acc, 0, 0, 0);
        return;
    }
#pragma unroll
    for (int s = NP - 1; s >= 0; --s)
#pragma unroll
        for (int i = 0; i <= s; ++i) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b[s - i], acc, 0, 0, 0);
}

// The order in which a run of MFMA matrix products with READS LDS reads before each is issued: AHEAD
// products' reads first, then one product and the next reads in turn, so that a product finds its
// operands there.  (Left to itself the compiler waits for the reads right before each product.)
template <int MFMA, int READS, int AHEAD>
__device__ __forceinline__ void interleave() {
    __builtin_amdgcn_sched_group_barrier(0x100, READS * AHEAD, 0);
#pragma unroll
    for (int i = 0; i < MFMA - AHEAD; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, AHEAD, 0);
}

// ------------------------------------------------------------------- LDS tiles --
// [rows][DP] bf16, 16-byte chunks permuted in each row so that both reads below touch every
// bank once: 16 rows at one chunk (row fragments), and 4 rows x 4 chunks (column fragments).
template <int DP>
__device__ __forceinline__ int swz(int r) {
    if constexpr (DP == 128) return ((r & 3) << 2) | ((r >> 2) & 3);
    else if constexpr (DP == 64) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    else return (r >> 2) & 3;
}
template <int DP>
__device__ __forceinline__ int tile_at(int r, int chunk) { return r * DP + ((chunk ^ swz<DP>(r)) << 3); }

// Where a lane's fragments start in a tile.  The permutation only flips bits of the chunk, so every
// other fragment is this one with constant bits flipped and a constant added.  opaque() keeps the
// compiler from holding all those addresses in registers across a loop.
template <int DP>
struct Lane {
    int row, col;
    __device__ __forceinline__ Lane(int lane) {
        row = tile_at<DP>(lane & 31, lane >> 5);
        const int i = lane & 15, g = lane >> 4;
        col = tile_at<DP>(4 * (g >> 1) + (i >> 2), 2 * (g & 1) + ((i & 3) >> 1)) + (i & 1) * 4;
    }
    __device__ __forceinline__ void opaque() { asm volatile("" : "+v"(row), "+v"(col)); }
};

// operand with one tile row per lane (depth along the row): rows row0 .. +31, depth chunk c
template <int DP, int NP>
__device__ __forceinline__ void row_frag(const uint16_t *t, int plane, int row0, int c, const Lane<DP> &at, bf16x8 (&p)[NP]) {
    const uint16_t *from = t + (at.row ^ (c << 4)) + row0 * DP;
#pragma unroll
    for (int s = 0; s < NP; ++s) p[s] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4_m *>(from + s * plane));
}

// operand with one tile column per lane (depth along the rows): columns col0 .. +31, rows row0
// .. +15 in the order in which an MFMA result holds them (registers 8c .. 8c + 7 of half h are
// rows 16c + 4h + {0..3, 8..11}), so a result is the other operand without any exchange.
template <int DP, int NP>
__device__ __forceinline__ void col_frag(const uint16_t *t, int plane, int row0, int col0, const Lane<DP> &at, bf16x8 (&p)[NP]) {
    const uint16_t *from = t + (at.col ^ col0) + row0 * DP, *next = t + (at.col ^ col0 ^ 16) + (row0 + 8) * DP;
#pragma unroll
    for (int s = 0; s < NP; ++s) {
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(from + s * plane));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(next + s * plane));
        p[s] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
}

// 16 bytes a lane from global memory straight into LDS: lane l's to `to` + 16 l (`to` alike in the
// wave), nothing where a lane is inactive.  Counted by vmcnt.
__device__ __forceinline__ void global_to_lds(const void *from, const uint16_t *to) {
    __builtin_amdgcn_global_load_lds((glob_void *)from, (lds_void *)to, 16, 0, 0);
}

// eight consecutive elements in registers
template <class T> struct Chunk;
template <> struct Chunk<__bf16> {
    u32x4 w;
    __device__ __forceinline__ void zero() { w = u32x4{0, 0, 0, 0}; }
    __device__ __forceinline__ void load(const __bf16 *p) { w = *reinterpret_cast<const u32x4_m *>(p); }
    __device__ __forceinline__ void negate() { w ^= 0x80008000u; }
    __device__ __forceinline__ void pieces(bf16x8 (&p)[1]) const { p[0] = __builtin_bit_cast(bf16x8, w); }
    __device__ __forceinline__ float dot(const Chunk &o) const {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) s += bf16_lo(w[i]) * bf16_lo(o.w[i]) + bf16_hi(w[i]) * bf16_hi(o.w[i]);
        return s;
    }
};
template <> struct Chunk<float> {
    f32x4 a, b;
    __device__ __forceinline__ void zero() { a = b = f32x4{0.f, 0.f, 0.f, 0.f}; }
    __device__ __forceinline__ void load(const float *p) {
        a = *reinterpret_cast<const f32x4_m *>(p);
        b = *reinterpret_cast<const f32x4_m *>(p + 4);
    }
    __device__ __forceinline__ void negate() { a = -a, b = -b; }
    __device__ __forceinline__ void pieces(bf16x8 (&p)[3]) const {
        const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        to_pieces<3>(x, p);
    }
    __device__ __forceinline__ float dot(const Chunk &o) const {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) s += a[i] * o.a[i] + b[i] * o.b[i];
        return s;
    }
};

// four consecutive elements of a result row
__device__ __forceinline__ void store4(__bf16 *p, float a, float b, float c, float d) {
    *reinterpret_cast<u32x2_m *>(p) = u32x2{pack_bf16(a, b), pack_bf16(c, d)};
}
__device__ __forceinline__ void store4(float *p, float a, float b, float c, float d) {
    *reinterpret_cast<f32x4_m *>(p) = f32x4{a, b, c, d};
}

}  // namespace hreg_tok
