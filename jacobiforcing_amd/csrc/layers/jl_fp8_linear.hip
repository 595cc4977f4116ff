// jl_fp8_linear.hip — products of 8-bit rows with 8-bit weights (jl_fp8.h): x has a scale for each row and 128 columns, W [O, K] one for each block of 128 x 128.
//   out[n, o] = sum over blocks b of sx[n, b] * sw[o / 128, b] * sum over k in b of x[n, k] * w[o, k]   (+ bias[o])
// One matrix instruction of 16 x 16 takes a block's 128 columns: scales that are powers of two go into it, float ones multiply what it leaves.  All sums are float.
#include <type_traits>

#include "jl_fp8.h"

typedef int f8_i32x8 __attribute__((ext_vector_type(8)));
typedef float f8_f32x4 __attribute__((ext_vector_type(4)));

struct Fp8Product {
    const uint8_t *x, *w;
    const void *xs, *ws;
    int64_t x_ld, xs_ld, w_ld, ws_ld;
    int N, O, blocks;
};
struct Fp8Result { const void *bias; int bias_dtype; void *out; int64_t out_ld; int out_dtype; };

// a block of 128 columns: 16 rows of W by 16 of x, each lane's operands its row's units of 16 bytes q and 4 + q (q = lane / 16; the sum does not go by their order)
__device__ __forceinline__ f8_i32x8 f8_operand(uint4 lo, uint4 hi) { return (f8_i32x8){(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w}; }
// The instruction lines the products of eight neighbouring columns up with the largest of them and keeps 13 binary digits behind its first (2^16 + 2^3 is whole, of 2^16 + 2^2 the 2^2 is gone), the
// same for its unscaled form: a sum is off by 2^-13 of the largest product of each eight at most, some 5e-5 .. 3e-4 of results of random operands, a rounding to bfloat16 4e-3.
// Scales of 2^(byte - 127), byte XB of `xs` and the lowest of `ws`
template <int XB> __device__ __forceinline__ f8_f32x4 f8_mma(f8_i32x8 w, f8_i32x8 x, f8_f32x4 c, int ws, int xs) { return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 0, 0, 0, ws, XB, xs); }
__device__ __forceinline__ f8_f32x4 f8_mma_plain(f8_i32x8 w, f8_i32x8 x) { return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, (f8_f32x4){0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0); }

template <bool E8> struct f8_scale_of { typedef uint8_t type; };
template <> struct f8_scale_of<false> { typedef float type; };

// acc[o][t]: rows o0 + 16 o .. of W by rows n0 + 16 t .. of x over the blocks b0 .. b1, operands straight from memory, AHEAD blocks on their way at once.  Rows that do not exist repeat the last
// one.  The 16 OT rows of W lie in one block of 128.
template <bool E8, int NT, int OT, int AHEAD>
__device__ __forceinline__ void f8_products(f8_f32x4 (&acc)[OT][NT], const Fp8Product &a, int64_t n0, int64_t o0, int b0, int b1, int lane) {
    typedef typename f8_scale_of<E8>::type S;
    const int l16 = lane & 15, quad = lane >> 4;
    const uint8_t *wp[OT], *xp[NT];
    const S *xs[NT], *ws = (const S *)a.ws + o0 / Q8_BLOCK * a.ws_ld;
#pragma unroll
    for (int o = 0; o < OT; ++o) {
        const int64_t r = o0 + 16 * o + l16;
        wp[o] = a.w + (r < a.O ? r : a.O - 1) * a.w_ld + 16 * quad;
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[o][t] = (f8_f32x4){0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int64_t n = n0 + 16 * t + l16, r = n < a.N ? n : a.N - 1;
        xp[t] = a.x + r * a.x_ld + 16 * quad;
        xs[t] = (const S *)a.xs + r;
    }
    for (int b = b0; b < b1; b += AHEAD) {
        uint4 wr[AHEAD][2][OT], xr[AHEAD][2][NT];
        S xf[AHEAD][NT], wf[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int c = b + i < b1 ? b + i : b1 - 1;              // behind the last block: the last one again, not multiplied
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int o = 0; o < OT; ++o) wr[i][h][o] = *(const uint4 *)(wp[o] + (int64_t)c * Q8_BLOCK + 64 * h);
#pragma unroll
                for (int t = 0; t < NT; ++t) xr[i][h][t] = *(const uint4 *)(xp[t] + (int64_t)c * Q8_BLOCK + 64 * h);
            }
            wf[i] = ws[c];
#pragma unroll
            for (int t = 0; t < NT; ++t) xf[i][t] = xs[t][c * a.xs_ld];
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (b + i >= b1) break;
#pragma unroll
            for (int o = 0; o < OT; ++o)
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const f8_i32x8 w = f8_operand(wr[i][0][o], wr[i][1][o]), x = f8_operand(xr[i][0][t], xr[i][1][t]);
                    if constexpr (E8) acc[o][t] = f8_mma<0>(w, x, acc[o][t], wf[i], xf[i][t]);
                    else {
                        const f8_f32x4 p = f8_mma_plain(w, x);
                        const float s = wf[i] * xf[i][t];
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[o][t][e] = __builtin_fmaf(s, p[e], acc[o][t][e]);
                    }
                }
        }
    }
}

// C consecutive columns from o of row n, and what is added to them
template <int C> __device__ __forceinline__ void f8_bias(const Fp8Result &r, int o, int O, float (&add)[C]) {
#pragma unroll
    for (int i = 0; i < C; ++i) add[i] = r.bias && o + i < O ? ld_any(r.bias, r.bias_dtype, o + i) : 0.f;
}
template <int C> __device__ __forceinline__ void f8_store(const Fp8Result &r, int64_t n, int o, int O, const float (&v)[C]) {
    auto leave = [&](auto *p) {
        typedef typename std::remove_pointer<decltype(p)>::type T;
        if (o + C <= O) q8_give<T, C>(p, v);                        // rows start at any element's border
        else
#pragma unroll
            for (int i = 0; i < C; ++i)
                if (o + i < O) st_f(p + i, v[i]);
    };
    if (r.out_dtype == JL_BF16) leave((bf16_t *)r.out + n * r.out_ld + o);
    else leave((float *)r.out + n * r.out_ld + o);
}
__device__ __forceinline__ void f8_store4(const Fp8Result &r, int64_t n, int o, int O, f8_f32x4 v, const float (&add)[4]) {
    const float f[4] = {v[0] + add[0], v[1] + add[1], v[2] + add[2], v[3] + add[3]};
    f8_store<4>(r, n, o, O, f);
}
__device__ __forceinline__ void f8_store8(const Fp8Result &r, int64_t n, int o, int O, f8_f32x4 lo, f8_f32x4 hi, const float (&add)[8]) {
    const float f[8] = {lo[0] + add[0], lo[1] + add[1], lo[2] + add[2], lo[3] + add[3], hi[0] + add[4], hi[1] + add[5], hi[2] + add[6], hi[3] + add[7]};
    f8_store<8>(r, n, o, O, f);
}

// ---- few rows: 16 NT of x by 16 OT of W per workgroup, whose NW wavefronts share the depth ------------------------------------------------------------
template <bool E8, int NT, int OT, int NW, int AHEAD>
__global__ __launch_bounds__(64 * NW) void fp8_few_kernel(Fp8Product a, Fp8Result r) {
    __shared__ f8_f32x4 part[NW][OT][NT][64];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int64_t o0 = (int64_t)blockIdx.x * 16 * OT, n0 = (int64_t)blockIdx.y * 16 * NT;
    f8_f32x4 acc[OT][NT];
    f8_products<E8, NT, OT, AHEAD>(acc, a, n0, o0, (int)((int64_t)a.blocks * wave / NW), (int)((int64_t)a.blocks * (wave + 1) / NW), lane);
#pragma unroll
    for (int o = 0; o < OT; ++o)
#pragma unroll
        for (int t = 0; t < NT; ++t) part[wave][o][t][lane] = acc[o][t];
    __syncthreads();
    for (int e = tid; e < OT * NT * 64; e += 64 * NW) {
        const int l = e & 63, t = (e >> 6) % NT, ot = (e >> 6) / NT;
        const int64_t n = n0 + 16 * t + (l & 15), o = o0 + 16 * ot + 4 * (l >> 4);
        f8_f32x4 s = part[0][ot][t][l];
#pragma unroll
        for (int i = 1; i < NW; ++i) s += part[i][ot][t][l];
        if (n >= a.N || o >= a.O) continue;
        float add[4];
        f8_bias(r, (int)o, a.O, add);
        f8_store4(r, n, (int)o, a.O, s, add);
    }
}

// ---- few rows of a gated unit: 16 NT of x by the 128 gates and 128 linear branches of a block of the result, a wavefront each 16 of them over the whole depth ------------
template <bool E8, int NT, int AHEAD>
__global__ __launch_bounds__(1024) void fp8_few_gated_kernel(Fp8Product a, int F, int kind, float limit, float alpha, float shift, Q8Out out) {
    __shared__ f8_f32x4 linear[8][NT][64];
    __shared__ uint32_t most[8][16 * NT];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, l16 = lane & 15, quad = lane >> 4;
    const int64_t f0 = (int64_t)blockIdx.x * Q8_BLOCK, n0 = (int64_t)blockIdx.y * 16 * NT;
    const int part = wave & 7;
    f8_f32x4 acc[1][NT];
    f8_products<E8, NT, 1, AHEAD>(acc, a, n0, (wave < 8 ? 0 : F) + f0 + 16 * part, 0, a.blocks, lane);
    if (wave >= 8)
#pragma unroll
        for (int t = 0; t < NT; ++t) linear[part][t][lane] = acc[0][t];
    __syncthreads();
    if (wave < 8)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const f8_f32x4 u = linear[part][t][lane];
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                acc[0][t][i] = q8_unit(acc[0][t][i], u[i], kind, limit, alpha, shift);
                const uint32_t b = q8_bits(acc[0][t][i]);
                m = m > b ? m : b;
            }
#pragma unroll
            for (int off = 16; off < 64; off <<= 1) { const uint32_t b = (uint32_t)__shfl_xor((int)m, off, 64); m = m > b ? m : b; }
            if (quad == 0) most[part][16 * t + l16] = m;
        }
    __syncthreads();
    if (wave >= 8) return;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int64_t n = n0 + 16 * t + l16;
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) { const uint32_t b = most[i][16 * t + l16]; m = m > b ? m : b; }
        const q8_scale<E8> s(m);
        if (n >= a.N) continue;
        *(uint32_t *)(out.q + n * out.ld + f0 + 16 * part + 4 * quad) = s.bad ? 0x7f7f7f7fu : q8_pack(s.of(acc[0][t][0]), s.of(acc[0][t][1]), s.of(acc[0][t][2]), s.of(acc[0][t][3]));
        if (part == 0 && quad == 0) ((typename q8_scale<E8>::type *)out.scale)[f0 / Q8_BLOCK * out.s_ld + n] = s.held;
    }
}

// ---- many rows: TM of x by TN of W per workgroup of WM x WN wavefronts -----------------------------------------------------------------------------------
// Stages of one block of 128 columns travel from memory into LDS while the stage before is multiplied.  XG rows of x that follow one another are the same lane's in XG tiles, so their scales are one word of
// LDS, and eight columns of the result that follow one another (32 h + 8 q + 4 e + i: accumulators 2 h + e of lanes of quad q) are a lane's whole store; for that the rows of a wavefront are
// permuted on their way into LDS.  Unit u of a row of LDS lies at u ^ (row / 2 % 8): the sixteen rows that are read at once meet different banks.
// GATED: the lower accumulators are gates, the others the linear branches of the same results.
// Tiles of 256 x 256, one workgroup per CU that takes tile after tile, the next one's first stage on its way while results are made: 8192 x 8192 by 8192 412 - 433 us (2540 - 2670 TFLOP/s), gated 8192 x 3584
// by 2 x 18944 870 - 930 by box (2390 - 2560; a workgroup for each tile 6 % more, a twentieth of it the units).  Float scales: 485 and 1085 - 1100.  Tiles of 128 x 256: 2048 x 18944 by 3584 130 us (2140), of
// 128 x 128 512 rows by 3584 by 4608 21.8.
// What bounds it: the way into a CU, some 60 GB/s of stages from L2 whatever the tile (a quarter of the loads left out of 128 x 128 and 128 x 256: 20 % less time; nothing loaded at all in 256 x 256: 15 % less),
// then the matrix cores (busy 67 % of the time in 8192 x 8192 by 8192, 60 % in the gated product, 47 % in 2048 x 18944 by 3584) and LDS (reads alone 27 %; what a stage's loads take is not counted there).
// Tiles are whole ones: where they fill the card once and a bit, as 4096 rows of 3584 by 4608 do (288 of 256 x 256, so 576 of 128 x 256 in three rounds), half of the time is lost.
// The gated tile of 256 x 256 needs more than its 256 registers: 13 vectors of offsets and constants, unused in the loop over the stages, are spilled and read back one by one in aim(), between tiles.
//   Lines from beyond L2 are touched a stage earlier (AHEAD: 458 -> 436; smaller tiles, whose rings are longer, lose by it).
//   The early barrier: 476 -> 459; no branch among the loads, so that they and the products stay in the order of the source: 459 -> 440; that order kept by force: 428 -> 418.
//   No loads into registers in the loop: the compiler waits for those with everything on its way (529 -> 458, with results in stores of 16 bytes).
//   Four wavefronts of 128 x 128 read a third less from LDS, but fill every register: 576; four of 128 x 64 in 128 x 256, one per SIMD, leave nobody to multiply while one waits: 145 for 122.
template <int I> struct f8_at { static constexpr int value = I; };
template <int XG> struct f8_word;
template <> struct f8_word<1> { typedef uint8_t type; };
template <> struct f8_word<2> { typedef uint16_t type; };
template <> struct f8_word<4> { typedef uint32_t type; };
constexpr int F8_MAX_BLOCKS = 1024;                                 // depths up to 131072: a tile's scales of W are in LDS from its beginning on

// 4 bytes per lane from base + off into LDS at `lds` + 4 * lane, as jl_load_lds; and from an address per lane
__device__ __forceinline__ void f8_load_lds4(const char *base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dword %1, %2" ::"s"(lds), "v"(off), "s"(base) : "m0", "memory");
}
// the same of the lanes whose bits are set alone (perhaps none), and of the first twelve with an address each: no branch, around which the compiler would gather products.  All 64 lanes are there where
// these are called, and again behind them
__device__ __forceinline__ void f8_load_lds4_of(uint32_t lanes_lo, uint32_t lanes_hi, const char *base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_mov_b32 exec_lo, %3\n\ts_mov_b32 exec_hi, %4\n\ts_nop 3\n\tglobal_load_lds_dword %1, %2\n\ts_mov_b64 exec, -1" ::"s"(lds), "v"(off), "s"(base), "s"(lanes_lo), "s"(lanes_hi) : "m0", "memory");
}
__device__ __forceinline__ void f8_load_far4_of12(const char *from, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_mov_b64 exec, 0xfff\n\ts_nop 3\n\tglobal_load_lds_dword %1, off\n\ts_mov_b64 exec, -1" ::"s"(lds), "v"(from) : "m0", "memory");
}
template <typename T> __device__ __forceinline__ uint32_t f8_lds(T *p) { return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)p); }

struct Fp8Tiles { int row_tiles, tiles, splits; float *parts; };   // splits > 1: shares of the depth, each its own sums [splits][N][O] for fp8_join_kernel
struct Fp8Unit { int kind; float limit, alpha, shift; };
// f with the kind of a unit as a constant
template <typename Fn> __device__ __forceinline__ void f8_unit_kind(int kind, Fn f) {
    if (kind == JL_ACT_SILU) f(f8_at<JL_ACT_SILU>{});
    else if (kind == JL_ACT_GELU_TANH) f(f8_at<JL_ACT_GELU_TANH>{});
    else if (kind == JL_ACT_GELU_ERF) f(f8_at<JL_ACT_GELU_ERF>{});
    else f(f8_at<JL_ACT_CLAMPED_SWISH>{});
}

template <bool E8, bool GATED, int TM, int TN, int WM, int WN, int RING>
__global__ __launch_bounds__(64 * WM * WN, (WM * WN >= 8 ? 1 : 2) * WM * WN / 4) void fp8_tile_kernel(Fp8Product a, Fp8Result res, Q8Out out8, Fp8Unit unit, Fp8Tiles t) {
    typedef typename f8_scale_of<E8>::type S;
    constexpr int NW = WM * WN, XT = TM / WM / 16, NT = TN / WN / 16, XG = XT < 4 ? XT : 4, BUF = (TM + TN) * 8, WTN = TN / WN;
    constexpr int HB = GATED ? NT / 2 : NT, WCOLS = 16 * HB, TCOLS = WN * WCOLS;      // accumulators that make up a wavefront's results, its columns of them, and the tile's
    // a stage's loads of a wavefront's 64 units of 16 bytes: rows of x, rows of W, words of x's scales.  Wavefronts below REST have one more
    constexpr int XI = TM / 8, WI = TN / 8, SWORDS = TM * (int)sizeof(S) / 4, SI = (SWORDS + 63) / 64, LOADS = XI + WI + SI, PER = (LOADS + NW - 1) / NW, REST = LOADS % NW ? LOADS % NW : NW;
    // EARLY: the barrier stands before a stage's last products; PAIR: its last two tiles of x are multiplied side by side, so that rows of W are free one by one for the next stage's (256 x 256 with bytes as scales:
    // 424 alone, 428 so).  WALK: a workgroup per CU takes tile after tile (float scales: no gain)
    constexpr bool AHEAD = TM == 256 && RING == 2, EARLY = XT >= 2 && (RING > 2 || XT == 8) && (XI + WI) % NW == 0, PAIR = EARLY && (XT < 8 || !E8), WALK = AHEAD && E8;
    static_assert(XT % XG == 0 && (HB == 1 || HB == 2 || HB == 4) && 128 % WTN == 0 && RING >= 2 && (!GATED || TCOLS == Q8_BLOCK), "tiles of whole parts");
    constexpr int SLOTS = PAIR ? (XT < 5 ? XT - 1 : 4) : XT < 4 ? XT : 4;      // parts of a stage's loads
    constexpr uint32_t SLO = SWORDS < 32 ? (1u << (SWORDS & 31)) - 1 : ~0u, SHI = SWORDS < 64 ? 0u : ~0u;
    extern __shared__ __attribute__((aligned(16))) uint4 ld8[];     // [RING][rows of x, rows of W][8 units]
    __shared__ __attribute__((aligned(16))) S xscale[RING][TM];
    __shared__ __attribute__((aligned(16))) S wscale[2][F8_MAX_BLOCKS + 4];
    __shared__ uint32_t touched[AHEAD ? NW : 1][64];
    __shared__ uint32_t most[GATED ? WN : 1][GATED ? TM : 1];
    // workgroups with the same remainder by 8 share an XCD; it walks strips of 1024 rows, column by column
    const int items = t.tiles * t.splits, per_xcd = (items + 7) / 8, slots = gridDim.x / 8, end = (blockIdx.x & 7) * per_xcd + per_xcd < items ? (blockIdx.x & 7) * per_xcd + per_xcd : items;
    int item = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
    if (item >= end) return;
    const int F = a.O / 2, rows_w = GATED ? F : a.O;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, l16 = lane & 15, quad = lane >> 4, wm = wave / WN, wn = wave % WN;
    auto swap = [](int row) { return (row >> 1) & 7; };
    auto x_row = [](int m) { const int p = m % (16 * XG); return m - p + p % 16 * XG + p / 16; };
    // row i of accumulator b's rows of W is this column of the wavefront's
    auto w_col = [](int b, int i) { return HB == 1 ? i : b / 2 * 32 + i / 4 * 8 + b % 2 * 4 + i % 4; };
    const uint32_t lds = f8_lds(ld8), lds_scale = f8_lds(xscale), lds_wscale = f8_lds(wscale), lds_touch = f8_lds(touched[AHEAD ? wave : 0]);
    int n0, o0, split, b0, last, first[2];
    const char *base[PER], *touch = nullptr;
    uint32_t off[PER], to[PER];
    // where a tile's operands lie; its scales of W, whole words from the one on that holds the first, go on their way in front of everything else: whoever waits for a stage has them
    auto aim = [&] {
        split = item / t.tiles;
        const int tile = item - split * t.tiles, cols = t.tiles / t.row_tiles, high = 1024 / TM < t.row_tiles ? 1024 / TM : t.row_tiles, strip = tile / (high * cols);
        const int here = t.row_tiles - strip * high < high ? t.row_tiles - strip * high : high, in_strip = tile - strip * high * cols;
        b0 = (int)((int64_t)a.blocks * split / t.splits);
        last = (int)((int64_t)a.blocks * (split + 1) / t.splits) - 1;
        n0 = (strip * high + in_strip % here) * TM;
        o0 = in_strip / here * TCOLS;
        const char *const xb = (const char *)a.x + n0 * a.x_ld, *const wb = (const char *)a.w + (int64_t)o0 * a.w_ld, *const wl = wb + (GATED ? F * a.w_ld : 0);
        auto x_off = [&](int m) { return (uint32_t)((n0 + m < a.N ? m : a.N - 1 - n0) * a.x_ld); };      // rows that do not exist repeat the last one
        auto w_off = [&](int o) { return (uint32_t)((o0 + o < rows_w ? o : rows_w - 1 - o0) * a.w_ld); };
        const int scale_end = (a.N - 1 - n0) * (int)sizeof(S) & ~3;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int j = NW * i + wave, row = 8 * (j < XI ? j : j - XI) + lane / 8, unit16 = (lane % 8 ^ swap(row)) * 16;
            if (j < XI) { base[i] = xb; off[i] = x_off(x_row(row)) + unit16; }
            else if (j < XI + WI) {
                const int b = row % WTN / 16, c = row / WTN * WCOLS + w_col(b % HB, row % 16);
                base[i] = GATED && 8 * (j - XI) % WTN / 16 >= HB ? wl : wb;
                off[i] = w_off(c) + unit16;
            } else {                                                // words behind the last row's repeat it
                const int at = (64 * (j - XI - WI) + lane) * 4;
                base[i] = (const char *)a.xs + (int64_t)n0 * sizeof(S);
                off[i] = at < scale_end ? at : scale_end;
            }
            to[i] = j < XI + WI ? lds + j * 1024 : lds_scale + (j - XI - WI) * 256;
        }
        // AHEAD: twelve lanes of a wavefront each touch a line of the stage after the next, so that it is in this XCD's L2 by then: of the 256 rows of x the 32 that are this tile's of the 8 that walk along
        // the same rows, of the 256 of W its 64 of 4
        if constexpr (AHEAD) {
            const int line = wave * 12 + (lane < 12 ? lane : 0), o = (in_strip % here * 64 + line - 32 + TN) % TN;
            if (line < 32) touch = xb + x_off((in_strip / here % 8 * 32 + line) % TM);
            else touch = (GATED && o >= TCOLS ? wl : wb) + w_off(GATED ? o % TCOLS : o);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int rb = GATED ? ((h ? F : 0) + o0) / Q8_BLOCK : o0 / Q8_BLOCK + h, bottom = (a.O - 1) / Q8_BLOCK;
            const char *from = (const char *)a.ws + ((rb < bottom ? rb : bottom) * a.ws_ld + b0) * sizeof(S);
            const int over = (int)((uintptr_t)from & 3), words = ((last + 1 - b0) * (int)sizeof(S) + over + 3) / 4;
            first[h] = over / (int)sizeof(S) - b0;
            for (int i = 64 * wave; i < words; i += 64 * NW)
                if (i + lane < words) f8_load_lds4(from - over, (i + lane) * 4, __builtin_amdgcn_readfirstlane(lds_wscale + h * (uint32_t)sizeof(wscale[0]) + i * 4));
        }
    };
    auto issue = [&](int s, int sel, int from, int upto) {      // behind the last stage: that one again, for the same number of loads on their way (nobody reads it)
        s = s < last ? s : last;
        const int64_t k = (int64_t)s * Q8_BLOCK, ks = s * a.xs_ld * (int64_t)sizeof(S);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (i < from || i >= upto) continue;
            const bool rows = NW * i + NW <= XI + WI, scales = NW * i >= XI + WI, any = i < PER - 1 || REST == NW;      // of every wavefront
            if (rows || (!scales && NW * i + wave < XI + WI)) jl_load_lds(base[i] + k, off[i], to[i] + sel * BUF * 16);
            else if (EARLY) f8_load_lds4_of(any ? SLO : __builtin_amdgcn_readfirstlane(wave < REST ? SLO : 0u), any ? SHI : __builtin_amdgcn_readfirstlane(wave < REST ? SHI : 0u), base[i] + ks, off[i], to[i] + sel * TM * (uint32_t)sizeof(S));
            else if ((any || wave < REST) && (SWORDS >= 64 || lane < SWORDS)) f8_load_lds4(base[i] + ks, off[i], to[i] + sel * TM * (uint32_t)sizeof(S));
        }
        if (AHEAD && upto == PER) f8_load_far4_of12(touch + (int64_t)(s + 1 < last ? s + 1 : last) * Q8_BLOCK, lds_touch);
    };
    f8_f32x4 acc[XT][NT];
    const int xr = (wm * (TM / WM) + l16) * 8, wr = (TM + wn * WTN + l16) * 8, p = swap(l16);
    // EARLY: a stage's first operands are read while the stage before multiplies its last tiles of x, which are in registers by then: the barrier that gives the memory back stands before those products
    f8_i32x8 wf[NT], xf[2];
    S ws[2], xs[XG];
    uint32_t word = 0;
    auto read_w = [&](int sel, int b) { const uint4 *B = ld8 + sel * BUF; wf[b] = f8_operand(B[wr + 128 * b + (quad ^ p)], B[wr + 128 * b + ((4 + quad) ^ p)]); };
    auto read_x = [&](int sel, int x) { const uint4 *B = ld8 + sel * BUF; xf[x & 1] = f8_operand(B[xr + 128 * x + (quad ^ p)], B[xr + 128 * x + ((4 + quad) ^ p)]); };
    auto read_xs = [&](int sel, int g) {
        const S *const from = xscale[sel] + wm * (TM / WM) + g * 16 * XG + XG * l16;
        if constexpr (E8) word = *(const typename f8_word<XG>::type *)from;
        else
#pragma unroll
            for (int i = 0; i < XG; ++i) xs[i] = from[i];
    };
    auto read_ws = [&](int s) {
        const int wblock = GATED ? 0 : (o0 % Q8_BLOCK + wn * WTN) / Q8_BLOCK;
        ws[0] = wscale[wblock][s + first[GATED ? 0 : wblock]];
        if (GATED) ws[1] = wscale[1][s + first[1]];
    };
    auto front = [&](int s, int sel) {
#pragma unroll
        for (int b = 0; b < NT; ++b) read_w(sel, b);
        read_x(sel, 0);
        read_xs(sel, 0);
        read_ws(s);
    };
    // behind(): the wait for the next stage; beside(x): loads among the products of tile x.  The order is kept as written (sched_barrier): left to itself the compiler moves products across the barrier and
    // loads in front of all of them
    auto products = [&](int s, int sel, auto behind, auto beside) {
        if (!EARLY) front(s, sel);
        const int next = sel == RING - 1 ? 0 : sel + 1;
#pragma unroll
        for (int g = 0; g < XT / XG; ++g) {
            if (g > 0) read_xs(sel, g);
            auto one = [&](auto at) {
                constexpr int I = decltype(at)::value;
                if constexpr (I < XG) {
                    const int x = g * XG + I;
                    auto product = [&](int x, auto i, int b, const S (&by)[2], uint32_t xw, const S (&xi)[XG]) {
                        constexpr int J = decltype(i)::value;
                        if constexpr (E8) acc[x][b] = f8_mma<J>(wf[b], xf[x & 1], acc[x][b], by[b >= HB], xw);
                        else {
                            const f8_f32x4 v = f8_mma_plain(wf[b], xf[x & 1]);
                            const float f = by[b >= HB] * xi[J];
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[x][b][e] = __builtin_fmaf(f, v[e], acc[x][b][e]);
                        }
                    };
                    if (x < XT - 1) read_x(sel, x + 1);
                    if constexpr (PAIR) if (x == XT - 2) return;
                    if (EARLY && x == XT - 1) {
                        __builtin_amdgcn_sched_barrier(0);
                        behind();
                        const S by[2] = {ws[0], ws[1]};
                        const uint32_t xw = word;
                        S xi[XG];
#pragma unroll
                        for (int i = 0; i < XG; ++i) xi[i] = xs[i];
                        read_xs(next, 0);
                        read_ws(s + 1);
                        if (PAIR) beside(x);
#pragma unroll
                        for (int b = 0; b < NT; ++b) {
                            if constexpr (PAIR) product(x - 1, f8_at<(I + XG - 1) % XG>{}, b, by, xw, xi);
                            if (b == (PAIR ? NT - 1 : 0)) read_x(next, 0);
                            product(x, f8_at<I>{}, b, by, xw, xi);
                            read_w(next, b);
                            if (!PAIR && b == 1) beside(x);
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    } else {
                        beside(x);
#pragma unroll
                        for (int b = 0; b < NT; ++b) product(x, f8_at<I>{}, b, ws, word, xs);
                        if (EARLY) __builtin_amdgcn_sched_barrier(0);
                    }
                    if constexpr (!E8 && XT * NT > 16) __builtin_amdgcn_sched_barrier(0);      // more products on their way at once take more registers than there are
                }
            };
            one(f8_at<0>{}); one(f8_at<1>{}); one(f8_at<2>{}); one(f8_at<3>{});
        }
        if (!EARLY) behind();
    };
    auto landed = [&] {                                             // all but the loads of the last RING - 2 stages (and one touch)
        if (RING == 2 || EARLY || REST == NW || wave < REST) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((RING - 2) * PER + (AHEAD ? 1 : 0)) : "memory");
        else asm volatile("s_waitcnt vmcnt(%0)" ::"n"((RING - 2) * (PER - 1) + (AHEAD ? 1 : 0)) : "memory");
    };
    int sel = 0;
    auto begin = [&] {
#pragma unroll
        for (int s = 0; s < RING - 1; ++s) issue(b0 + s, WALK ? sel : s, 0, PER);      // (WALK: not where the last stage's part of another may still land)
    };
    aim();
    begin();
    landed();
    __syncthreads();
    for (;;) {
#pragma unroll
        for (int x = 0; x < XT; ++x)
#pragma unroll
            for (int b = 0; b < NT; ++b) acc[x][b] = (f8_f32x4){0.f, 0.f, 0.f, 0.f};
        if (EARLY) {
            issue(b0 + RING - 1, sel == 0 ? RING - 1 : sel - 1, 0, PER / SLOTS);
            front(b0, sel);
        }
        for (int s = b0; s <= last; ++s) {
            products(s, sel, [&] { landed(); __syncthreads(); }, [&](int x) {
                if (!EARLY) { if (x == 0) issue(s + RING - 1, sel == 0 ? RING - 1 : sel - 1, 0, PER); }
                else {                                              // a part behind the barrier that gave the memory back, the others beside the first tiles
                    if (x < SLOTS - 1) issue(s + RING - 1, sel == 0 ? RING - 1 : sel - 1, (x + 1) * PER / SLOTS, (x + 2) * PER / SLOTS);
                    if (x == XT - 1) issue(s + RING, sel, 0, PER / SLOTS);
                }
            });
            sel = sel == RING - 1 ? 0 : sel + 1;
        }
        // WALK: the next tile's first stage travels while this one's results are made
        const int N0 = n0, O0 = o0;
        if (t.splits > 1) { res.out = t.parts + (int64_t)split * a.N * a.O; res.out_ld = a.O; res.out_dtype = JL_F32; res.bias = nullptr; }
        item += slots;
        const bool more = WALK && item < end;
        if (more) {
            aim();
            begin();
        }
        if constexpr (GATED) {
            f8_unit_kind(unit.kind, [&](auto kind) {
#pragma unroll
                for (int x = 0; x < XT; ++x) {
                    uint32_t m = 0;
#pragma unroll
                    for (int e = 0; e < 4 * HB; ++e) {
                        const float v = q8_unit(acc[x][e >> 2][e & 3], acc[x][HB + (e >> 2)][e & 3], decltype(kind)::value, unit.limit, unit.alpha, unit.shift);
                        acc[x][e >> 2][e & 3] = v;
                        const uint32_t b = q8_bits(v);
                        m = m > b ? m : b;
                    }
#pragma unroll
                    for (int o = 16; o < 64; o <<= 1) { const uint32_t b = (uint32_t)__shfl_xor((int)m, o, 64); m = m > b ? m : b; }
                    if (quad == 0) most[wn][wm * (TM / WM) + 16 * x + l16] = m;
                }
            });
            __syncthreads();
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");            // in front of the results, which need not be waited for; and nothing is on its way into LDS when the workgroup ends
        if constexpr (GATED) {
#pragma unroll
            for (int x = 0; x < XT; ++x) {
                const int64_t n = N0 + wm * (TM / WM) + x_row(16 * x + l16);
                uint32_t m = 0;
#pragma unroll
                for (int i = 0; i < WN; ++i) { const uint32_t b = most[i][wm * (TM / WM) + 16 * x + l16]; m = m > b ? m : b; }
                const q8_scale<E8> s(m);
                if (n >= a.N) continue;
                auto four = [&](const f8_f32x4 &v) { return s.bad ? 0x7f7f7f7fu : q8_pack(s.of(v[0]), s.of(v[1]), s.of(v[2]), s.of(v[3])); };
                uint8_t *q = out8.q + n * out8.ld + O0 + wn * WCOLS;
                if constexpr (HB == 1) *(uint32_t *)(q + 4 * quad) = four(acc[x][0]);
                else
#pragma unroll
                    for (int h = 0; h < HB; h += 2) *(uint2 *)(q + 16 * h + 8 * quad) = make_uint2(four(acc[x][h]), four(acc[x][h + 1]));
                if (wn == 0 && quad == 0) ((S *)out8.scale)[O0 / Q8_BLOCK * out8.s_ld + n] = s.held;
            }
        } else {
            auto rows = [&](auto store) {
#pragma unroll
                for (int x = 0; x < XT; ++x) {
                    const int64_t n = N0 + wm * (TM / WM) + x_row(16 * x + l16);
                    if (n < a.N) store(n, x);
                }
            };
            if constexpr (NT == 1) {
                const int o = O0 + wn * WTN + 4 * quad;
                float add[4];
                f8_bias(res, o, a.O, add);
                if (o < a.O) rows([&](int64_t n, int x) { f8_store4(res, n, o, a.O, acc[x][0], add); });
            } else
#pragma unroll
                for (int h = 0; h < NT / 2; ++h) {
                    const int o = O0 + wn * WTN + 32 * h + 8 * quad;
                    float add[8];
                    if (o >= a.O) continue;
                    f8_bias(res, o, a.O, add);
                    rows([&](int64_t n, int x) { f8_store8(res, n, o, a.O, acc[x][2 * h], acc[x][2 * h + 1], add); });
                }
        }
        if (!more) return;
        __syncthreads();                                            // everybody's loads of the first stage are in LDS
    }
}

// the sums of a depth's shares, in their order, to a result
__global__ __launch_bounds__(256) void fp8_join_kernel(const float *__restrict__ parts, int splits, int64_t N, int O, Fp8Result r) {
    const int per_row = (O + 3) / 4;
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, n = at / per_row;
    if (n >= N) return;
    const int o = (int)(at - n * per_row) * 4;
    f8_f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    const float *p = parts + n * O + o;
    if (o + 4 <= O)
#pragma unroll 4
        for (int s = 0; s < splits; ++s, p += N * O) {
            float v[4];
            q8_take<float, 4>(p, v);
            sum += (f8_f32x4){v[0], v[1], v[2], v[3]};
        }
    else
        for (int s = 0; s < splits; ++s, p += N * O)
            for (int i = 0; i < 4; ++i)
                if (o + i < O) sum[i] += p[i];
    float add[4];
    f8_bias(r, o, O, add);
    f8_store4(r, n, o, O, sum, add);
}

// How a product is cut: a kernel's tile, and shares of the depth
struct Fp8Plan { int tile, splits; };
enum { F8_16x64, F8_32x64, F8_64x64, F8_64x128, F8_128x128, F8_128x128_TWO, F8_128x256, F8_256x256, F8_16x128_MANY, F8_32x128_MANY, F8_64x128_MANY, F8_16x256, F8_32x256, F8_64x256, F8_FEW };

template <bool E8, bool GATED, int TM, int TN, int WM, int WN, int RING>
static int fp8_tile_launch(const Fp8Product &a, const Fp8Result &r, const Q8Out &out, const Fp8Unit &unit, int splits, float *parts, hipStream_t st) {
    constexpr int lds = RING * (TM + TN) * Q8_BLOCK;
    auto kern = fp8_tile_kernel<E8, GATED, TM, TN, WM, WN, RING>;
    const int64_t row_tiles = (a.N + TM - 1) / TM, tiles = row_tiles * (((int64_t)a.O + TN - 1) / TN);
    const int64_t items = (tiles * splits + 7) / 8 * 8, blocks = TM == 256 && E8 && items > 256 ? 256 : items;      // (256 CUs)
    if (tiles * splits > INT32_MAX / 2 || q8_too_many(blocks, 64 * WM * WN)) return jl_fail(JL_E_INVALID, "fp8_tile_kernel: more tiles than a launch takes");
    if (lds > 48 * 1024) {                                          // with the scales beside them beyond 64 KB
        const hipError_t e = hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return jl_fail(JL_E_LAUNCH, "fp8_tile_kernel: cannot get %d bytes of LDS: %s", lds, hipGetErrorString(e));
    }
    kern<<<(unsigned)blocks, 64 * WM * WN, lds, st>>>(a, r, out, unit, Fp8Tiles{(int)row_tiles, (int)tiles, splits, parts});
    return jl_check_launch("fp8_tile_kernel");
}

static int fp8_bad(const char *what, const jl_fp8_product *p) {
    if (!p || !p->x || !p->w || !p->x_scale || !p->w_scale) return jl_fail(JL_E_INVALID, "%s: null pointer", what);
    if (p->K <= 0 || p->K > Q8_MAX_COLS || p->K % Q8_BLOCK || p->x_ld < p->K || p->w_ld < p->K || p->x_ld % 16 || p->w_ld % 16 || (((uintptr_t)p->x | (uintptr_t)p->w) & 15))
        return jl_fail(JL_E_INVALID, "%s: whole blocks of 128 columns, rows at 16-byte borders", what);
    if (p->x_scale_ld < p->N || p->w_scale_ld < p->K / Q8_BLOCK) return jl_fail(JL_E_INVALID, "%s: x has a scale for each row and block, w for each 128 x 128", what);
    if (p->scale_type != JL_SCALE_E8M0 && p->scale_type != JL_SCALE_F32) return jl_fail(JL_E_INVALID, "%s: unknown type of scales", what);
    if (p->N > (1 << 21) || p->O > (1 << 30)) return jl_fail(JL_E_INVALID, "%s: up to 2097152 rows of x and 2^30 of w", what);
    return JL_OK;
}
// whether the tiles take it: rows within 32 bits of a tile's first, scales of W that fit, scales of x in whole words; others go straight from memory
static bool fp8_near(const jl_fp8_product *p) {
    return p->x_ld <= (1 << 24) && p->w_ld <= (1 << 24) && p->K / Q8_BLOCK <= F8_MAX_BLOCKS && (p->scale_type == JL_SCALE_F32 || (p->x_scale_ld % 4 == 0 && (uintptr_t)p->x_scale % 4 == 0));
}
static Fp8Product fp8_product(const jl_fp8_product *p) {
    return Fp8Product{(const uint8_t *)p->x, (const uint8_t *)p->w, p->x_scale, p->w_scale, p->x_ld, p->x_scale_ld, p->w_ld, p->w_scale_ld, (int)p->N, p->O, p->K / Q8_BLOCK};
}


// A product's time is its launch, rounds of one tile per CU (small tiles: several), a tile's start, end and stages, about as long whatever the others do, and for shares of the depth a launch of their sums,
// which are written and read once more.  us measured with weights from memory, by this rule / beside it: 100 rows of 3584 by 4608 11.6 (64 x 64) / 14.5 (32 x 64), 256 rows 17.1 (64 x 128) / 20 (64 x 64), 512
// rows 21.6 (128 x 128) / 28.8 (64 x 128), 1024 rows 31 (128 x 256) / 35.6 (128 x 128), 2048 rows 47 (256 x 256) / 57 (128 x 256); of 18944 by 3584 32 rows 18 (32 x 64 in 4) / 19.3 (64 x 128 in 8), 256 rows 35.5
// (128 x 128 in 4) / 36.6 (128 x 256 in 8), 1024 rows 76.7 (256 x 256 in 4) / 87.6 (128 x 128), 2048 rows 129 (128 x 256) / 137 (256 x 256 in 2), 4096 rows 217 (256 x 256) / 264 (in 2); 1298 rows of 15360 by
// 3646 100 (256 x 256 in 2) / 93 (128 x 256), the worst of some hundred.
// Wavefronts of 32 x 32 in 64 x 64 (four side by side over all its rows: 777 rows of 1920 by 1111 9.1, so 8.4); 128 x 128 with four, sixteen or turned round: as long or up to 13 % longer.
// Products of at most three blocks of depth, where a tile mostly starts and writes, have two tiles of 128 x 128 per CU, rings of two stages: 4096 rows of 128 by 16384 51 / 64 (256 x 256) / 79 (128 x 128), 1472 rows
// of 384 by 15680 28.8 / 33.9 (128 x 256); at four blocks, 8192 rows by 2048, 23.8 / 20.5 (256 x 256).
// Gated, whose tiles are 256 rows of W, by heights alone: 128 rows of 1024 by 2 x 2048 7.6 (16 high) / 12 (128), 256 rows of 3584 by 2 x 18944 55 (256) / 64 (128).
// Up to 16 rows are the few rows' launch's, but where they are deep (whose rows of x every workgroup reads: 16 rows of 18944 by 3584 20.6 / 18.4 (16 x 64 in 4), one row by 1024 15.6 / 13.1; 8 rows of 8192 by
// 8192 17.5 / 20.4) or have many columns (8 rows of 3584 by 152064 115.8 / 96.9 (16 x 128), two 90.6 / 92.7).
// Up to 64 rows by many columns have two or three workgroups per CU, at the rate of memory: 64 rows of 3584 by 152064 111 / 165 (64 x 64 in rings of 4).
struct Fp8Cost { int tile, rows, cols; float stage, rest; bool small; };
static Fp8Plan fp8_plan(const jl_fp8_product *p, bool gated) {
    const int64_t N = p->N, O = p->O, blocks = p->K / Q8_BLOCK;
    auto tiles = [&](int64_t tm, int64_t tn) { return (N + tm - 1) / tm * ((O + tn - 1) / tn); };
    if (!fp8_near(p)) return {F8_FEW, 1};
    if (!gated) {
        if (N <= 64 && tiles(64, 128) >= 512) return {N <= 2 ? F8_FEW : N <= 16 ? F8_16x128_MANY : N <= 32 ? F8_32x128_MANY : F8_64x128_MANY, 1};
        if (N <= 16) {
            const int64_t there = tiles(16, 64), most = there < 256 ? 256 / there : 1;
            if (blocks < 96 || (N <= 8 && O > 2048) || most == 1) return {F8_FEW, 1};
            return {F8_16x64, (int)(most < blocks / 4 ? most : blocks / 4)};
        }
        if (blocks <= 3 && tiles(128, 128) > 256) return {F8_128x128_TWO, 1};
    }
    static const Fp8Cost plain[] = {{F8_32x64, 32, 64, 0.28f, 1.5f, true}, {F8_64x64, 64, 64, 0.34f, 1.7f, true}, {F8_64x128, 64, 128, 0.42f, 3.3f, false}, {F8_128x128, 128, 128, 0.56f, 4.3f, false},
                                    {F8_128x256, 128, 256, 0.87f, 6.3f, false}, {F8_256x256, 256, 256, 1.42f, 8.f, false}};
    static const Fp8Cost units[] = {{F8_16x256, 16, 256, 0.30f, 1.5f, false}, {F8_32x256, 32, 256, 0.45f, 2.f, false}, {F8_64x256, 64, 256, 0.70f, 2.5f, false}, {F8_128x256, 128, 256, 1.0f, 4.f, false},
                                    {F8_256x256, 256, 256, 1.5f, 8.f, false}};
    Fp8Plan best = {0, 1};
    float least = 1e30f;
    for (int i = 0; i < (gated ? 5 : 6); ++i) {
        const Fp8Cost &t = gated ? units[i] : plain[i];
        const int64_t there = tiles(t.rows, t.cols), most = !gated && there < 256 ? 256 / there : 1;
        for (int64_t splits = 1; splits <= most; splits = splits < most && 2 * splits > most ? most : 2 * splits) {
            if (splits > 1 && blocks / splits < 4) break;
            const int64_t items = there * splits;
            const float rounds = t.small ? (items <= 256 ? 1.0f : items < 360 ? 1.4f : items / 256.0f) : (float)((items + 255) / 256);
            const float us = rounds * ((blocks + splits - 1) / splits * t.stage + t.rest) + (splits > 1 ? 3.5f + 0.3f * splits + N * O * splits * 1.25e-6f : 0.f);
            if (us < least) { least = us; best = {t.tile, (int)splits}; }
        }
    }
    return best;
}
extern "C" const char *jl_fp8_cut(const jl_fp8_product *p, int gated, int32_t *shares) {
    static const char *const names[] = {"16x64", "32x64", "64x64", "64x128", "128x128", "128x128 two", "128x256", "256x256", "16x128 many", "32x128 many", "64x128 many", "16x256", "32x256", "64x256", "rows"};
    static_assert(sizeof names / sizeof names[0] == F8_FEW + 1, "a name for each");
    const Fp8Plan plan = !p || p->N <= 0 || p->O <= 0 || p->K <= 0 ? Fp8Plan{F8_FEW, 1} : fp8_plan(p, gated != 0);
    if (shares) *shares = plan.splits;
    return names[plan.tile];
}
extern "C" int64_t jl_linear_fp8_floats(const jl_fp8_product *p) {
    if (!p || p->N <= 0 || p->O <= 0 || p->K <= 0) return 0;
    const Fp8Plan plan = fp8_plan(p, false);
    return plan.splits > 1 ? plan.splits * p->N * p->O : 0;
}

extern "C" int jl_linear_fp8(const jl_fp8_product *p, const void *bias, int bias_dtype, void *out, int64_t out_ld, int out_dtype, float *scratch, void *stream) {
    if (p && (p->N <= 0 || p->O <= 0)) return JL_OK;
    if (const int bad = fp8_bad("jl_linear_fp8", p)) return bad;
    const auto known = [](int t) { return t == JL_F32 || t == JL_BF16; };
    if (!out || out_ld < p->O || ((uintptr_t)out & 15) || !known(out_dtype) || (bias && !known(bias_dtype))) return jl_fail(JL_E_INVALID, "jl_linear_fp8: bad result or bias");
    const Fp8Product a = fp8_product(p);
    const Fp8Result r = {bias, bias_dtype, out, out_ld, out_dtype};
    hipStream_t st = (hipStream_t)stream;
    const bool e8 = p->scale_type == JL_SCALE_E8M0;
    const Fp8Plan plan = fp8_plan(p, false);
    if (plan.splits > 1 && (!scratch || ((uintptr_t)scratch & 15))) return jl_fail(JL_E_INVALID, "jl_linear_fp8: no room for %d shares of the depth (jl_linear_fp8_floats)", plan.splits);
#define F8_TILE(TM, TN, WM, WN, RING) (e8 ? fp8_tile_launch<true, false, TM, TN, WM, WN, RING>(a, r, Q8Out{}, Fp8Unit{}, plan.splits, scratch, st) : fp8_tile_launch<false, false, TM, TN, WM, WN, RING>(a, r, Q8Out{}, Fp8Unit{}, plan.splits, scratch, st))
    int rc = JL_OK;
    switch (plan.tile) {
    case F8_16x64: rc = F8_TILE(16, 64, 1, 4, 6); break;
    case F8_32x64: rc = F8_TILE(32, 64, 1, 4, 6); break;
    case F8_64x64: rc = F8_TILE(64, 64, 2, 2, 4); break;
    case F8_64x128: rc = F8_TILE(64, 128, 2, 4, 5); break;
    case F8_128x128: rc = F8_TILE(128, 128, 2, 4, 4); break;
    case F8_128x128_TWO: rc = F8_TILE(128, 128, 2, 4, 2); break;
    case F8_128x256: rc = F8_TILE(128, 256, 2, 4, 3); break;
    case F8_16x128_MANY: rc = F8_TILE(16, 128, 1, 4, 4); break;
    case F8_32x128_MANY: rc = F8_TILE(32, 128, 1, 4, 3); break;
    case F8_64x128_MANY: rc = F8_TILE(64, 128, 1, 4, 3); break;
    case F8_256x256: rc = F8_TILE(256, 256, 2, 4, 2); break;
    default: {
        auto go = [&](auto kern, int nt, int ot, int nw) {
            const int64_t cols = (p->O + 16 * (int64_t)ot - 1) / (16 * ot);
            if (q8_too_many(cols, 64 * nw)) return jl_fail(JL_E_INVALID, "jl_linear_fp8: more rows of w than a launch takes");
            kern<<<dim3((unsigned)cols, (unsigned)((p->N + 16 * nt - 1) / (16 * nt))), 64 * nw, 0, st>>>(a, r);
            return jl_check_launch("fp8_few_kernel");
        };
        if (e8) return p->N <= 16 ? go(fp8_few_kernel<true, 1, 1, 8, 4>, 1, 1, 8) : go(fp8_few_kernel<true, 4, 2, 4, 1>, 4, 2, 4);
        return p->N <= 16 ? go(fp8_few_kernel<false, 1, 1, 8, 4>, 1, 1, 8) : go(fp8_few_kernel<false, 4, 2, 4, 1>, 4, 2, 4);
    }
    }
#undef F8_TILE
    if (rc != JL_OK || plan.splits == 1) return rc;
    fp8_join_kernel<<<(unsigned)((p->N * ((p->O + 3) / 4) + 255) / 256), 256, 0, st>>>(scratch, plan.splits, p->N, p->O, r);
    return jl_check_launch("fp8_join_kernel");
}

extern "C" int jl_linear_gated_fp8(const jl_fp8_product *p, int32_t kind, float limit, float alpha, float shift, uint8_t *q, int64_t q_ld, void *scale, int64_t s_ld, void *stream) {
    if (p && (p->N <= 0 || p->O <= 0)) return JL_OK;
    if (const int bad = fp8_bad("jl_linear_gated_fp8", p)) return bad;
    const int F = p->O / 2;
    if (p->O % (2 * Q8_BLOCK) || kind < JL_ACT_GELU_TANH || kind > JL_ACT_GELU_ERF || !q || !scale || q_ld < F || q_ld % 8 || ((uintptr_t)q & 7) || s_ld < p->N)
        return jl_fail(JL_E_INVALID, "jl_linear_gated_fp8: gates and linear branches in whole blocks of 128, a known kind, a result of 8-bit rows");
    const Fp8Product a = fp8_product(p);
    const Q8Out out = {q, q_ld, scale, s_ld};
    const Fp8Unit unit = {kind, limit, alpha, shift};
    hipStream_t st = (hipStream_t)stream;
    const bool e8 = p->scale_type == JL_SCALE_E8M0;
#define F8_TILE(TM, TN, WM, WN, RING) (e8 ? fp8_tile_launch<true, true, TM, TN, WM, WN, RING>(a, Fp8Result{}, out, unit, 1, nullptr, st) : fp8_tile_launch<false, true, TM, TN, WM, WN, RING>(a, Fp8Result{}, out, unit, 1, nullptr, st))
    switch (fp8_plan(p, true).tile) {
    case F8_16x256: return F8_TILE(16, 256, 1, 8, 4);
    case F8_32x256: return F8_TILE(32, 256, 1, 8, 4);
    case F8_64x256: return F8_TILE(64, 256, 1, 8, 3);
    case F8_128x256: return F8_TILE(128, 256, 2, 4, 3);
    case F8_256x256: return F8_TILE(256, 256, 2, 4, 2);
    }
#undef F8_TILE
    auto go = [&](auto kern, int nt) {
        if (q8_too_many(F / Q8_BLOCK, 1024)) return jl_fail(JL_E_INVALID, "jl_linear_gated_fp8: more rows of w than a launch takes");
        kern<<<dim3((unsigned)(F / Q8_BLOCK), (unsigned)((p->N + 16 * nt - 1) / (16 * nt))), 1024, 0, st>>>(a, F, kind, limit, alpha, shift, out);
        return jl_check_launch("fp8_few_gated_kernel");
    };
    if (e8) return p->N <= 16 ? go(fp8_few_gated_kernel<true, 1, 4>, 1) : go(fp8_few_gated_kernel<true, 4, 1>, 4);
    return p->N <= 16 ? go(fp8_few_gated_kernel<false, 1, 4>, 1) : go(fp8_few_gated_kernel<false, 4, 1>, 4);
}
