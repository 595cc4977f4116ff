// jl_fp8.h — 8-bit rows: e4m3 values (OCP: 448 is the largest, no infinities) with a scale for each block of 128 columns, shared by the launches that make them (jl_fp8.hip) and the products that
// read or make them (jl_fp8_linear.hip).
//
// A block's scale is a power of two (E8: one byte, the exponent + 127; what gfx950's matrix instructions apply by themselves) or a float.  With a the block's largest magnitude:
//   E8     s = the least 2^e >= a / 448, e >= -126;  q = x / s to the nearest e4m3, ties to even (the division is exact)
//   float  s = max(a, 448 * 2^-126) / 448;           q = x * 448 / a to the nearest e4m3, from the quotient rounded once to 32 bits
// A block that holds an infinity or a NaN is all NaN, its scale among it.
#ifndef JL_FP8_H
#define JL_FP8_H

#include "jl_common.h"

constexpr int Q8_BLOCK = 128;
constexpr int Q8_MAX_COLS = 1 << 30;                                // columns stay within 32 bits with what a wavefront takes beyond them
constexpr uint32_t Q8_LEAST = 0x04e00000u;                          // 448 * 2^-126: a block of smaller values is scaled as if this were its largest

// whether workgroups of so many threads are more than a launch takes: fewer than 2^32 threads altogether
static inline bool q8_too_many(int64_t workgroups, int threads) { return workgroups > (int64_t)UINT32_MAX / threads; }

// the largest of |bits| over the 16 lanes of a row of the wavefront, in every one of them
__device__ __forceinline__ uint32_t q8_max16(uint32_t v) {
#define Q8_STEP(ctrl) { const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, ctrl, 0xF, 0xF, true); v = v > o ? v : o; }
    Q8_STEP(0xB1)                                                   // quad_perm [1, 0, 3, 2], [2, 3, 0, 1], half rows and rows mirrored
    Q8_STEP(0x4E)
    Q8_STEP(0x141)
    Q8_STEP(0x140)
#undef Q8_STEP
    return v;
}

__device__ __forceinline__ uint32_t q8_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// four floats within 448 as four bytes
__device__ __forceinline__ uint32_t q8_pack(float a, float b, float c, float d) {
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, p, true);
}

template <bool E8> struct q8_scale;
template <> struct q8_scale<true> {
    typedef uint8_t type;
    float by;
    uint8_t held;
    bool bad;
    __device__ __forceinline__ explicit q8_scale(uint32_t a) {      // the bits of the block's largest magnitude (a NaN's are above infinity's)
        int e = (int)(a >> 23) - 8 + ((a & 0x7fffffu) > 0x600000u ? 1 : 0);
        e = e < 1 ? 1 : e;
        bad = a >= 0x7f800000u;
        held = bad ? 255 : (uint8_t)e;
        by = __uint_as_float((uint32_t)(254 - (bad ? 127 : e)) << 23);
    }
    __device__ __forceinline__ float of(float x) const { return x * by; }
};
template <> struct q8_scale<false> {
    typedef float type;
    float to, least, inv, held;                                     // a = least * 2^e with least in [1, 2): x * 448 / a = (x * to) / least, to = 448 * 2^-e
    bool bad;
    __device__ __forceinline__ explicit q8_scale(uint32_t a) {
        bad = a >= 0x7f800000u;
        a = a < Q8_LEAST ? Q8_LEAST : a;
        held = bad ? __uint_as_float(0x7fc00000u) : __uint_as_float(a) / 448.0f;
        to = __uint_as_float(((262u - (bad ? 127u : a >> 23)) << 23) | 0x600000u);
        least = __uint_as_float(0x3f800000u | (a & 0x7fffffu));
        inv = 1.0f / least;
    }
    // The quotient rounded once: x * 448 is t + lo (it has up to 27 digits), and y is corrected by what it leaves over of both; the second rounding differs from the quotient's own only where that is
    // within 2^-23 of a step of the middle between two floats.  Without lo one in four quotients beside a border of e4m3 came out a step of 32 bits off, one in twenty on the border's other side
    __device__ __forceinline__ float of(float x) const {
        const float t = x * to, lo = __builtin_fmaf(x, to, -t), y = t * inv;
        return __builtin_fmaf(__builtin_fmaf(-y, least, t) + lo, inv, y);
    }
};

// A wavefront's 512 columns of a row: a lane has eight of them, U that follow one another (8: one load of 16-bit values; 4: two loads of floats), so that the lanes of a load lie side by side
__device__ __forceinline__ constexpr int q8_col(int U, int lane, int i) { return U == 8 ? lane * 8 + i : i / 4 * 256 + lane * 4 + i % 4; }

// those eight in 8 bits; a block is 16 lanes' values (U = 8) or 32 lanes' four (4), whose first lane leaves the scale.  `at`: the wavefront's first column, `wide` the row's with its padding
template <bool E8, int U> __device__ __forceinline__ void q8_leave(const float (&v)[8], int lane, int at, int wide, uint8_t *q, typename q8_scale<E8>::type *scale, int64_t s_ld) {
#pragma unroll
    for (int h = 0; h < 8; h += U) {
        uint32_t a = q8_bits(v[h]);
#pragma unroll
        for (int i = 1; i < U; ++i) { const uint32_t b = q8_bits(v[h + i]); a = a > b ? a : b; }
        a = q8_max16(a);
        if (U == 4) { const uint32_t b = (uint32_t)__shfl_xor((int)a, 16, 64); a = a > b ? a : b; }
        const q8_scale<E8> s(a);
        const int c = at + q8_col(U, lane, h);
        if (c >= wide) continue;
        uint32_t word[U / 4];
#pragma unroll
        for (int i = 0; i < U; i += 4) word[i / 4] = s.bad ? 0x7f7f7f7fu : q8_pack(s.of(v[h + i]), s.of(v[h + i + 1]), s.of(v[h + i + 2]), s.of(v[h + i + 3]));
        if constexpr (U == 8) *(uint2 *)(q + c) = make_uint2(word[0], word[1]);
        else *(uint32_t *)(q + c) = word[0];
        if (lane % (Q8_BLOCK / U) == 0) scale[c / Q8_BLOCK * s_ld] = s.held;
    }
}

typedef float q8_f32x4 __attribute__((ext_vector_type(4)));
// U values that follow one another, at any element's border (gfx950 takes wide accesses to global memory there)
template <typename T, int U> __device__ __forceinline__ void q8_take(const T *p, float *v) {
    if constexpr (sizeof(T) == 2) {
        uint32_t w[U / 2];
        __builtin_memcpy(w, p, 2 * U);
#pragma unroll
        for (int k = 0; k < U / 2; ++k) { v[2 * k] = __uint_as_float(w[k] << 16); v[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u); }
    } else
#pragma unroll
        for (int k = 0; k < U; k += 4) {                                // 16 bytes each: a copy of 32 comes out as 16, 12 and 4
            q8_f32x4 w;
            __builtin_memcpy(&w, p + k, 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[k + i] = w[i];
        }
}
template <typename T, int U> __device__ __forceinline__ void q8_give(T *p, const float *v) {
    if constexpr (sizeof(T) == 2) {
        __bf16 h[U];
#pragma unroll
        for (int k = 0; k < U; ++k) h[k] = (__bf16)v[k];
        __builtin_memcpy(p, h, 2 * U);
    } else
#pragma unroll
        for (int k = 0; k < U; k += 4) {
            const q8_f32x4 w = {v[k], v[k + 1], v[k + 2], v[k + 3]};
            __builtin_memcpy(p + k, &w, 16);
        }
}

// a lane's eight values from the wavefront's column `at` on of a row of W; zeros behind its end.  WHOLE: W is a multiple of eight
template <typename T, int U, bool WHOLE> __device__ __forceinline__ void q8_load(const T *row, int lane, int at, int W, float (&v)[8]) {
#pragma unroll
    for (int h = 0; h < 8; h += U) {
        const int c = at + q8_col(U, lane, h);
        if (WHOLE ? c < W : c + U <= W) q8_take<T, U>(row + c, v + h);
        else
#pragma unroll
            for (int i = 0; i < U; ++i) v[h + i] = !WHOLE && c + i < W ? ld_f(row + c + i) : 0.f;
    }
}
template <typename T, int U, bool WHOLE> __device__ __forceinline__ void q8_store(T *row, int lane, int at, int W, const float (&v)[8]) {
#pragma unroll
    for (int h = 0; h < 8; h += U) {
        const int c = at + q8_col(U, lane, h);
        if (WHOLE ? c < W : c + U <= W) q8_give<T, U>(row + c, v + h);
        else
#pragma unroll
            for (int i = 0; i < U; ++i)
                if (!WHOLE && c + i < W) st_f(row + c + i, v[h + i]);
    }
}

// jl_gated_act's unit, but that the caps of the clamped swish leave a NaN one, for its block to show it
__device__ __forceinline__ float q8_unit(float g, float u, int kind, float limit, float alpha, float shift) {
    if (kind != JL_ACT_CLAMPED_SWISH) return gated_unit_f<true>(g, u, kind, limit, alpha, shift);
    g = g > limit ? limit : g;
    u = u > limit ? limit : u < -limit ? -limit : u;
    return g * sigmoid_f<true>(alpha * g) * (u + shift);
}

struct Q8Out { uint8_t *q; int64_t ld; void *scale; int64_t s_ld; };      // rows of ld bytes; the scales of a block of columns side by side, s_ld from block to block

#endif
