// jl_fp8.hip — launches that leave 8-bit rows (jl_fp8.h): of a matrix, of a residual stream's norm, of a gated unit, and of weights in blocks of 128 x 128.
#include <type_traits>

#include "jl_fp8.h"

// ---- rows of a matrix, or of a unit of two column ranges of it: a wavefront takes 512 columns of a row ---------------------------------------------------
// Bound by memory: 8192 x 3584 of bfloat16 18.2 us (4.8 TB/s read and written; a large copy reaches 4.9), of floats 26.0 (5.6), with float scales 19.3 and 27.5; units of 4096 x 4864 21.9 - 23 (4.3 - 4.5), of
// 8192 x 18944 143 (5.4).  The unit's sigmoid on the hardware's exponential and reciprocal leaves as many values in 8 bits on the other side of a border as the library's functions do (60 million of gelu: 82 float scales, 137 plain torch; silu 90 / 90),
// and those take 26.7 us.  Rows that start anywhere: 8192 x 3585 of bfloat16 22.4 (a value at a time 49).
struct Q8Unit { int kind, g_col, u_col; float limit, alpha, shift; };      // u_col < 0: no linear branch

template <typename T, bool E8, int U, bool WHOLE, bool UNIT>
__global__ __launch_bounds__(256) void fp8_rows_kernel(const T *__restrict__ x, int64_t ld, int64_t N, int W, int chunks, Q8Unit unit, Q8Out out) {
    const int lane = threadIdx.x & 63;
    const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int64_t n = item / chunks;
    if (n >= N) return;
    const int at = (int)(item - n * chunks) * 512;
    float v[8];
    if constexpr (UNIT) {
        float g[8], u[8];
        q8_load<T, U, WHOLE>(x + n * ld + unit.g_col, lane, at, W, g);
        if (unit.u_col >= 0) q8_load<T, U, WHOLE>(x + n * ld + unit.u_col, lane, at, W, u);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = at + q8_col(U, lane, i) < W ? q8_unit(g[i], unit.u_col >= 0 ? u[i] : 1.0f, unit.kind, unit.limit, unit.alpha, unit.shift) : 0.f;
    } else q8_load<T, U, WHOLE>(x + n * ld, lane, at, W, v);
    typedef typename q8_scale<E8>::type S;
    q8_leave<E8, U>(v, lane, at, (W + Q8_BLOCK - 1) / Q8_BLOCK * Q8_BLOCK, out.q + n * out.ld, (S *)out.scale + n, out.s_ld);
}

static int q8_out_bad(const char *what, const Q8Out &o, int64_t N, int64_t W, int scale_type) {
    const int64_t wide = (W + Q8_BLOCK - 1) / Q8_BLOCK * Q8_BLOCK;
    if (!o.q || !o.scale || o.ld < wide || o.ld % 8 || ((uintptr_t)o.q & 7) || o.s_ld < N || W > Q8_MAX_COLS) return jl_fail(JL_E_INVALID, "%s: up to 2^30 columns, 8-bit rows of whole blocks at 8-byte borders, scales of all rows per block", what);
    if (scale_type != JL_SCALE_E8M0 && scale_type != JL_SCALE_F32) return jl_fail(JL_E_INVALID, "%s: unknown type of scales", what);
    return JL_OK;
}

template <bool UNIT>
static int fp8_rows_launch(const char *what, const void *x, int dtype, int64_t N, int64_t ld, int W, const Q8Unit &unit, const Q8Out &out, int scale_type, hipStream_t st) {
    const int chunks = (W + 511) / 512;
    const int64_t blocks = (N * chunks + 3) / 4;
    if (N > INT32_MAX || q8_too_many(blocks, 256)) return jl_fail(JL_E_INVALID, "%s: more rows than a launch takes", what);
    JL_DISPATCH(dtype, {
        auto go = [&](auto kern) { kern<<<(unsigned)blocks, 256, 0, st>>>((const T *)x, ld, N, W, chunks, unit, out); };
        constexpr int U = sizeof(T) == 2 ? 8 : 4;
        if (scale_type == JL_SCALE_E8M0) { if (W % 8 == 0) go(fp8_rows_kernel<T, true, U, true, UNIT>); else go(fp8_rows_kernel<T, true, U, false, UNIT>); }
        else { if (W % 8 == 0) go(fp8_rows_kernel<T, false, U, true, UNIT>); else go(fp8_rows_kernel<T, false, U, false, UNIT>); }
    });
    return jl_check_launch("fp8_rows_kernel");
}

extern "C" int jl_quantize_fp8(const void *x, int dtype, int64_t N, int64_t ld, int32_t W, uint8_t *q, int64_t q_ld, void *scale, int64_t s_ld, int scale_type, void *stream) {
    if (N <= 0 || W <= 0) return JL_OK;
    if (!x || ld < W || (dtype != JL_F32 && dtype != JL_BF16)) return jl_fail(JL_E_INVALID, "jl_quantize_fp8: null pointer or bad sizes");
    const Q8Out out = {q, q_ld, scale, s_ld};
    if (const int bad = q8_out_bad("jl_quantize_fp8", out, N, W, scale_type)) return bad;
    return fp8_rows_launch<false>("jl_quantize_fp8", x, dtype, N, ld, W, Q8Unit{}, out, scale_type, (hipStream_t)stream);
}

extern "C" int jl_gated_act_fp8(const void *z, int dtype, int64_t N, int64_t ld, int32_t g_col, int32_t u_col, int32_t F, int32_t kind, float limit, float alpha, float shift, uint8_t *q, int64_t q_ld,
                                void *scale, int64_t s_ld, int scale_type, void *stream) {
    if (N <= 0 || F <= 0) return JL_OK;
    if (!z || g_col < 0 || (int64_t)g_col + F > ld || (int64_t)u_col + F > ld || kind < JL_ACT_GELU_TANH || kind > JL_ACT_GELU_ERF || (dtype != JL_F32 && dtype != JL_BF16))
        return jl_fail(JL_E_INVALID, "jl_gated_act_fp8: null pointer, bad columns or kind");
    const Q8Out out = {q, q_ld, scale, s_ld};
    if (const int bad = q8_out_bad("jl_gated_act_fp8", out, N, F, scale_type)) return bad;
    return fp8_rows_launch<true>("jl_gated_act_fp8", z, dtype, N, ld, F, Q8Unit{kind, g_col, u_col < 0 ? -1 : u_col, limit, alpha, shift}, out, scale_type, (hipStream_t)stream);
}

// ---- residual update, norm, 8 bits -----------------------------------------------------------------------------------------------------------------------
// Bound by memory: 8192 x 3584 of a float stream 66.4 us (4.9 TB/s), of bfloat16 38.2 (5.4); 4096 x 8192 of floats 59 (6.3).  One row 3.8 (from memory 4.9): two waits for memory and a workgroup's sum.
// NW wavefronts share a row, 512 columns at a time in turn; a thread keeps its 8 * NC values between the sum of squares and the quantisation, so a row is read once and written once.  NC = 0: rows too
// wide for that are read again, from where the same thread has stored the update.
struct Q8Norm { int64_t x_ld; const void *y; int y_dtype; int64_t y_ld; const void *w; int w_dtype; float eps; int64_t N; int W; };

template <typename T, bool E8, int U, bool WHOLE, int NW, int NC>
__global__ __launch_bounds__(NW == 1 ? 256 : 64 * NW) void fp8_norm_kernel(T *__restrict__ x, Q8Norm p, Q8Out out) {
    constexpr int RB = NW == 1 ? 4 : 1, KEEP = NC ? NC : 1;
    __shared__ float red[NW];
    const int lane = threadIdx.x & 63, wave = NW == 1 ? 0 : threadIdx.x >> 6;
    const int64_t n = (int64_t)blockIdx.x * RB + (NW == 1 ? threadIdx.x >> 6 : 0);
    if (n >= p.N) return;                                             // whole wavefronts, and with more of them per row the whole workgroup
    T *row = x + n * p.x_ld;
    const int W = p.W, wide = (W + Q8_BLOCK - 1) / Q8_BLOCK * Q8_BLOCK, chunks = (W + 511) / 512;
    float v[KEEP][8], sum = 0.f;
    auto update = [&](int at, float (&a)[8]) {
        q8_load<T, U, WHOLE>(row, lane, at, W, a);
        if (!p.y) return;
        float b[8];
        if (p.y_dtype == JL_BF16) q8_load<bf16_t, U, WHOLE>((const bf16_t *)p.y + n * p.y_ld, lane, at, W, b);
        else q8_load<float, U, WHOLE>((const float *)p.y + n * p.y_ld, lane, at, W, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            a[i] += b[i];
            if (sizeof(T) == 2) a[i] = (float)(__bf16)a[i];         // the norm reads what the stream keeps
        }
        q8_store<T, U, WHOLE>(row, lane, at, W, a);
    };
    auto squares = [&](const float (&a)[8]) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s = __builtin_fmaf(a[i], a[i], s);
        sum += s;
    };
    if constexpr (NC > 0) {
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            if (wave + k * NW < chunks) update((wave + k * NW) * 512, v[k]);
            else
#pragma unroll
                for (int i = 0; i < 8; ++i) v[k][i] = 0.f;
            squares(v[k]);
        }
    } else
        for (int k = wave; k < chunks; k += NW) {
            update(k * 512, v[0]);
            squares(v[0]);
        }
    sum = wave_sum_f32(sum);
    if constexpr (NW > 1) {
        if (lane == 0) red[wave] = sum;
        __syncthreads();
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < NW; ++i) sum += red[i];
    }
    const float by = 1.0f / sqrtf(sum / (float)W + p.eps);
    auto leave = [&](int at, float (&a)[8]) {
        float f[8];
        if (p.w) {
            if (p.w_dtype == JL_BF16) q8_load<bf16_t, U, WHOLE>((const bf16_t *)p.w, lane, at, W, f);
            else q8_load<float, U, WHOLE>((const float *)p.w, lane, at, W, f);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            a[i] = p.w ? a[i] * by * f[i] : a[i] * by;
            if (at + 512 > W && at + q8_col(U, lane, i) >= W) a[i] = 0.f;      // behind the row's end: zero whatever the norm is
        }
        typedef typename q8_scale<E8>::type S;
        q8_leave<E8, U>(a, lane, at, wide, out.q + n * out.ld, (S *)out.scale + n, out.s_ld);
    };
    if constexpr (NC > 0) {
#pragma unroll
        for (int k = 0; k < NC; ++k)
            if (wave + k * NW < chunks) leave((wave + k * NW) * 512, v[k]);
    } else
        for (int k = wave; k < chunks; k += NW) {
            q8_load<T, U, WHOLE>(row, lane, k * 512, W, v[0]);
            leave(k * 512, v[0]);
        }
}

template <typename T, bool E8, int U, bool WHOLE> static int fp8_norm_launch(T *x, const Q8Norm &a, const Q8Out &out, hipStream_t st) {
    int rc = JL_OK;
    auto go = [&](auto kern, int waves) {
        const int64_t blocks = waves == 1 ? (a.N + 3) / 4 : a.N;
        const int threads = waves == 1 ? 256 : 64 * waves;
        if (a.N > INT32_MAX || q8_too_many(blocks, threads)) rc = jl_fail(JL_E_INVALID, "jl_add_rmsnorm_fp8: more rows than a launch takes");
        else kern<<<(unsigned)blocks, threads, 0, st>>>(x, a, out);
    };
    const int chunks = (a.W + 511) / 512;
    if (chunks <= 1) go(fp8_norm_kernel<T, E8, U, WHOLE, 1, 1>, 1);
    else if (chunks <= 2) go(fp8_norm_kernel<T, E8, U, WHOLE, 1, 2>, 1);
    else if (chunks <= 4) go(fp8_norm_kernel<T, E8, U, WHOLE, 4, 1>, 4);
    else if (chunks <= 8) go(fp8_norm_kernel<T, E8, U, WHOLE, 4, 2>, 4);
    else if (chunks <= 16) go(fp8_norm_kernel<T, E8, U, WHOLE, 4, 4>, 4);
    else if (chunks <= 64) go(fp8_norm_kernel<T, E8, U, WHOLE, 16, 4>, 16);
    else go(fp8_norm_kernel<T, E8, U, WHOLE, 16, 0>, 16);
    return rc != JL_OK ? rc : jl_check_launch("fp8_norm_kernel");
}

extern "C" int jl_add_rmsnorm_fp8(void *x, int dtype, int64_t x_ld, const void *y, int y_dtype, int64_t y_ld, const void *w, int w_dtype, float eps, int64_t N, int32_t W, uint8_t *q, int64_t q_ld,
                                  void *scale, int64_t s_ld, int scale_type, void *stream) {
    if (N <= 0 || W <= 0) return JL_OK;
    const auto known = [](int t) { return t == JL_F32 || t == JL_BF16; };
    if (!x || x_ld < W || (y && y_ld < W) || !known(dtype) || !known(y_dtype) || !known(w_dtype)) return jl_fail(JL_E_INVALID, "jl_add_rmsnorm_fp8: null pointer, bad sizes or types");
    const Q8Out out = {q, q_ld, scale, s_ld};
    if (const int bad = q8_out_bad("jl_add_rmsnorm_fp8", out, N, W, scale_type)) return bad;
    const Q8Norm a = {x_ld, y, y_dtype, y_ld, w, w_dtype, eps, N, W};
    const bool floats = dtype == JL_F32 || (y && y_dtype == JL_F32);      // loads of four values, or of eight
    JL_DISPATCH(dtype, {
        auto go = [&](auto e8, auto whole) {
            if (floats) return fp8_norm_launch<T, decltype(e8)::value, 4, decltype(whole)::value>((T *)x, a, out, (hipStream_t)stream);
            return fp8_norm_launch<T, decltype(e8)::value, 8, decltype(whole)::value>((T *)x, a, out, (hipStream_t)stream);
        };
        const std::true_type yes;
        const std::false_type no;
        if (scale_type == JL_SCALE_E8M0) return W % 8 == 0 ? go(yes, yes) : go(yes, no);
        return W % 8 == 0 ? go(no, yes) : go(no, no);
    });
}

// ---- weights: a scale for each block of 128 x 128, a workgroup's -----------------------------------------------------------------------------------------
// Bound by memory: 37888 x 3584 of bfloat16 79 us (5.1 TB/s read and written), of floats 129 (5.3).
template <typename T, bool E8>
__global__ __launch_bounds__(256) void fp8_weight_kernel(const T *__restrict__ w, int64_t ld, int64_t O, int K, Q8Out out) {
    __shared__ uint32_t most[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = blockIdx.x * Q8_BLOCK + (tid & 15) * 8;
    const int64_t o0 = (int64_t)blockIdx.y * Q8_BLOCK + (tid >> 4);
    float v[8][8];
    uint32_t a = 0;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        if (o0 + 16 * r < O) q8_load<T, 8, false>(w + (o0 + 16 * r) * ld, tid & 15, blockIdx.x * Q8_BLOCK, K, v[r]);
        else
#pragma unroll
            for (int i = 0; i < 8; ++i) v[r][i] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) { const uint32_t b = q8_bits(v[r][i]); a = a > b ? a : b; }
    }
    a = q8_max16(a);
#pragma unroll
    for (int off = 16; off < 64; off <<= 1) { const uint32_t b = (uint32_t)__shfl_xor((int)a, off, 64); a = a > b ? a : b; }
    if (lane == 0) most[wave] = a;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) a = a > most[i] ? a : most[i];
    const q8_scale<E8> s(a);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        if (o0 + 16 * r >= O) break;
        uint2 q = make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
        if (!s.bad) q = make_uint2(q8_pack(s.of(v[r][0]), s.of(v[r][1]), s.of(v[r][2]), s.of(v[r][3])), q8_pack(s.of(v[r][4]), s.of(v[r][5]), s.of(v[r][6]), s.of(v[r][7])));
        *(uint2 *)(out.q + (o0 + 16 * r) * out.ld + c) = q;
    }
    if (tid == 0) ((typename q8_scale<E8>::type *)out.scale)[blockIdx.y * out.s_ld + blockIdx.x] = s.held;
}

extern "C" int jl_quantize_weight_fp8(const void *w, int dtype, int64_t O, int64_t ld, int32_t K, uint8_t *q, int64_t q_ld, void *scale, int64_t s_ld, int scale_type, void *stream) {
    if (O <= 0 || K <= 0) return JL_OK;
    if (!w || ld < K || (dtype != JL_F32 && dtype != JL_BF16)) return jl_fail(JL_E_INVALID, "jl_quantize_weight_fp8: null pointer or bad sizes");
    const int64_t cols = (K + Q8_BLOCK - 1) / Q8_BLOCK, rows = (O + Q8_BLOCK - 1) / Q8_BLOCK;
    const Q8Out out = {q, q_ld, scale, s_ld};
    if (const int bad = q8_out_bad("jl_quantize_weight_fp8", out, cols, K, scale_type)) return bad;
    if (rows > 65535) return jl_fail(JL_E_INVALID, "jl_quantize_weight_fp8: up to 8388480 rows");
    JL_DISPATCH(dtype, {
        auto go = [&](auto kern) { kern<<<dim3((unsigned)cols, (unsigned)rows), 256, 0, (hipStream_t)stream>>>((const T *)w, ld, O, K, out); };
        if (scale_type == JL_SCALE_E8M0) go(fp8_weight_kernel<T, true>); else go(fp8_weight_kernel<T, false>);
    });
    return jl_check_launch("fp8_weight_kernel");
}
