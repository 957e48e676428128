// q48_w8.hpp — weights in 8 bits: what the product (q48_w8.hip) and the
// mixture-of-experts layer (q48_moe.hip) share.  Included by the HIP sources of
// libintllm_hip only.
//
// Codes lie in tiles of 16 rows x 64 columns, 1 KB: lane l of a wave holds the 16 codes
// of row l % 16 from column 16 (l / 16) on, which is the operand of
// v_mfma_i32_16x16x64_i8, so a wave reads a tile as 64 lanes x 16 contiguous bytes and
// multiplies it as it comes.  Rows past the last and columns past K are zero codes.
#pragma once

#include "q48_gemv_tiles.hpp"
#include "q48_quant.hpp"

typedef int v4i __attribute__((ext_vector_type(4)));

namespace {

// floor(S sa sw / 2^48) mod 2^64 for steps in [0, 2^63): the product of the three mod
// 2^128 holds the bits 48 .. 111 that are asked for.
__device__ __forceinline__ int64_t w8_scaled(int S, int64_t sa, int64_t sw)
{
    const q48_u128 p = (q48_u128)(uint64_t)sa * (uint64_t)sw;
    const q48_u128 v = p * (uint32_t)(S < 0 ? 0u - (uint32_t)S : (uint32_t)S);
    return (int64_t)(uint64_t)((q48_i128)(S < 0 ? 0 - v : v) >> 48);
}

// The same in FP64 rounding down (q48_round_down), as a double: sa and sw = step 2^-48 (inf
// for steps of 2^53 and more, w8_step_double).  P = sa sw and S P as rounded products and
// their exact remainders: the floor of the first, and of what the others add to its
// fraction.  Rounding down makes that sum (between -2 and 4) too small by less than 2^-49, so
// only a fraction next to 1 may hide a whole number: `sure` is false there (about one product
// in 2^40; w8_scaled then), and where h reaches 2^53 - 2^32: below that the sum of both
// floors is a whole number that a double holds, which next to 2^53 it need not be (2^32, of
// any margin past 4, for a constant whose low half is zero).
__device__ __forceinline__ double w8_scaled_double(int S, double sa, double sw, bool &sure)
{
#pragma clang fp contract(off)   // h as rounded
    const double p = sa * sw, pl = __builtin_fma(sa, sw, -p), s = (double)S;
    const double h = s * p, hl = __builtin_fma(s, p, -h), f = __builtin_floor(h);
    const double t = (h - f) + __builtin_fma(s, pl, hl), g = __builtin_floor(t);
    sure = (__builtin_fabs(h) < 0x1p53 - 0x1p32) & (t - g < 1.0 - 0x1p-40);
    return f + g;
}
__device__ __forceinline__ double w8_step_double(int64_t step)
{
    return (uint64_t)step < (uint64_t)1 << 53 ? (double)step : __builtin_inf();
}

// A constant that stays in a register: as a literal every fused operation that adds it
// would copy it into its result first.
__device__ __forceinline__ double w8_kept(double c)
{
    asm("" : "+v"(c));
    return c;
}

// All of v before anything behind: chains of operations that would else be scheduled one
// after the other.
__device__ __forceinline__ void w8_together(double (&v)[2])
{
    asm volatile("" : "+v"(v[0]), "+v"(v[1]));
}
__device__ __forceinline__ void w8_together(double (&v)[1]) {}

// fp_mul(fp_silu(g), u) (fp_math.h:911-921) of U pairs of whole numbers below 2^53 in FP64
// rounding down alone; false where the result passes 2^53.  The squares of fp_exp: the first
// 12 stay below 2^52 (two operations each, q48_exp_small), the last two, of at most e^10
// 2^48, are a rounded product and its exact remainder each, r = A + T with A a double and
// T < 2^13.  Rounding down makes the sums behind T too small by less than 2^-39: false is
// returned where that may hide a whole number (q48_silu then).  A quotient by A + T: an
// estimate as in q48_recip, its remainder 2^96 - q A exact (a multiple of A's last place,
// below 2^53 of them) and compared with A + (q + 1) T, whose product is below 2^53.  Past
// 10 in magnitude the sigmoid is 0 or 1.  About 90 operations (with 64-bit integers for the
// last squares and the quotients 160, a third of them of quarter rate), step by step for all
// pairs: one is a chain, and a wave alone on its SIMD waits for each of its links.
template <int U>
__device__ __forceinline__ bool w8_silu_mul(const double (&g)[U], const double (&u)[U], double (&out)[U])
{
#pragma clang fp contract(off)   // products as rounded
#define W8_EACH _Pragma("unroll") for (int j = 0; j < U; ++j)
    constexpr double ten = 10 * 0x1p48, unit = 0x1p-48;
    const double m28 = w8_kept(-0x1p28), p52 = w8_kept(0x1p52), r24 = w8_kept(0x1p-24);
    double h[U], y[U], A[U], T[U], r[U], q[U], c[U];
    bool sure = true, far = false;
    W8_EACH far |= __builtin_fabs(g[j]) > ten;
    W8_EACH h[j] = __builtin_fma(__builtin_fmin(__builtin_fabs(g[j]), ten), 0x1p-14, p52 + 0x1p48);
#pragma unroll
    for (int k = 0; k < 12; ++k) {
        W8_EACH y[j] = __builtin_fma(h[j], r24, m28);
        W8_EACH h[j] = __builtin_fma(y[j], y[j], p52);
        w8_together(h);
    }
    W8_EACH y[j] = __builtin_fma(h[j], r24, m28);
    W8_EACH r[j] = y[j] * y[j];   // square 13: A + T
    W8_EACH A[j] = __builtin_floor(r[j]);
    W8_EACH T[j] = __builtin_fma(y[j], y[j], -r[j]);
    W8_EACH T[j] = __builtin_floor((r[j] - A[j]) + T[j]);
    w8_together(T);
    W8_EACH A[j] *= r24;          // square 14
    W8_EACH T[j] *= r24;
    W8_EACH r[j] = A[j] * A[j];
    W8_EACH q[j] = __builtin_fma(A[j], A[j], -r[j]);
    W8_EACH q[j] = __builtin_fma(2 * A[j], T[j], q[j]);
    W8_EACH q[j] = __builtin_fma(T[j], T[j], q[j]);
    W8_EACH A[j] = __builtin_floor(r[j]);
    W8_EACH q[j] = (r[j] - A[j]) + q[j];
    W8_EACH T[j] = __builtin_floor(q[j]);
    W8_EACH sure &= q[j] - T[j] < 1.0 - 0x1p-30;
    w8_together(T);
    // what is divided by: e^g where g > 0, else 1 + e^-g
    W8_EACH c[j] = g[j] > 0 ? 0.0 : 0x1p48;
    W8_EACH r[j] = A[j] + c[j];
    W8_EACH T[j] += c[j] - (r[j] - A[j]);
    W8_EACH A[j] = r[j];
    W8_EACH r[j] = __builtin_amdgcn_rcp(A[j]);
    W8_EACH y[j] = __builtin_fma(-A[j], r[j], 1.0);
    W8_EACH y[j] = __builtin_fma(y[j], y[j], y[j]);
    W8_EACH r[j] = __builtin_fma(r[j], y[j], r[j]);
    w8_together(r);
    W8_EACH r[j] = __builtin_fma(-(r[j] * T[j]), r[j], r[j]);
    // the quotient in units of 2^-48, or a unit less
    const double p48 = w8_kept(0x1p48), low = w8_kept(16.0 - 0.5 * unit);
    W8_EACH q[j] = __builtin_fma(r[j], p48, low) - 16.0;
    W8_EACH y[j] = __builtin_fma(-q[j], A[j], p48);
    W8_EACH h[j] = q[j] + unit;
    W8_EACH y[j] = y[j] - A[j] * unit;
    W8_EACH q[j] = y[j] >= h[j] * T[j] ? h[j] : q[j];
    w8_together(q);
    // floor(2^96 / (1 + e^-g)) where g > 0: below 2^53, so the remainder is one operation
    W8_EACH A[j] = q[j] + 1.0;
    W8_EACH r[j] = __builtin_amdgcn_rcp(A[j]);
    W8_EACH y[j] = __builtin_fma(-A[j], r[j], 1.0);
    W8_EACH y[j] = __builtin_fma(y[j], y[j], y[j]);
    W8_EACH r[j] = __builtin_fma(r[j], y[j], r[j]);
    w8_together(r);
    W8_EACH r[j] = (r[j] + low) - 16.0;
    W8_EACH h[j] = r[j] + unit;
    W8_EACH r[j] = __builtin_fma(-h[j], A[j], 1.0) >= 0 ? h[j] : r[j];
    W8_EACH r[j] = c[j] == 0 ? w8_kept(r[j]) : q[j];   // (kept: else a branch around its making)
    if (__any(far))
        W8_EACH r[j] = g[j] > ten ? 1.0 : g[j] < -ten ? 0.0 : r[j];
    W8_EACH y[j] = __builtin_floor(g[j] * r[j]);
    W8_EACH out[j] = __builtin_floor(y[j] * (u[j] * unit));
    W8_EACH sure &= __builtin_fabs(out[j]) < 0x1p53;
#undef W8_EACH
    return sure;
}

// The words of whole numbers below 2^63: by their bits where a wave's are below 2^51
template <int U>
__device__ __forceinline__ void w8_words(const double (&v)[U], int64_t (&w)[U])
{
    bool wide = false;
#pragma unroll
    for (int j = 0; j < U; ++j)
        wide |= __builtin_fabs(v[j]) >= 0x1p51;
    if (__any(wide)) {
#pragma unroll
        for (int j = 0; j < U; ++j)
            w[j] = (int64_t)v[j];
    } else {
#pragma unroll
        for (int j = 0; j < U; ++j)
            w[j] = (int64_t)(__builtin_bit_cast(uint64_t, v[j] + 0x1.8p52) - 0x4338000000000000ull);
    }
}

// One product, and one SwiGLU of two, of steps in words
__device__ __forceinline__ int64_t w8_times(int S, int64_t sa, int64_t sw)
{
    bool sure;
    const double y = w8_scaled_double(S, w8_step_double(sa), w8_step_double(sw) * 0x1p-48, sure);
    return sure ? (int64_t)y : w8_scaled(S, sa, sw);
}
__device__ __forceinline__ int64_t w8_swiglu(int Sg, int Su, int64_t sa, int64_t sg, int64_t su)
{
    const double a = w8_step_double(sa);
    bool s1, s2;
    const double g[1] = {w8_scaled_double(Sg, a, w8_step_double(sg) * 0x1p-48, s1)};
    const double u[1] = {w8_scaled_double(Su, a, w8_step_double(su) * 0x1p-48, s2)};
    double y[1];
    if (w8_silu_mul<1>(g, u, y) & s1 & s2) {
        int64_t w[1];
        w8_words<1>(y, w);
        return w[0];
    }
    return q48_mul(q48_silu(w8_scaled(Sg, sa, sg)), w8_scaled(Su, sa, su));
}

// the step of a row whose largest magnitude is a, and its reciprocal
__device__ __forceinline__ uint64_t w8_step(uint64_t a, double &r)
{
    const uint64_t cap = (uint64_t)INT64_MAX / 127, s = (a + 126) / 127;
    const uint64_t step = s < cap ? s : cap;
    const double d = (double)step;
    r = __builtin_amdgcn_rcp(d);
    r = __builtin_fma(r, __builtin_fma(-d, r, 1.0), r);
    return step;
}

// byte of a code in a matrix's tiles
__device__ __forceinline__ size_t w8_at(int row, int col, int KT)
{
    return ((size_t)(row >> 4) * KT + (col >> 6)) * 1024 + ((col & 63) >> 4) * 256 +
           (row & 15) * 16 + (col & 15);
}

// Barrier of the block for what was written to LDS; loads from memory stay in flight.
__device__ __forceinline__ void lds_barrier()
{
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <int CTRL>
__device__ __forceinline__ int q48_dpp32(int v)
{
    return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, false);
}

// A row of words over the first NT threads of a block, in registers: thread i holds words
// C (i + NT j) + 0 .. C - 1 for j < J, zeros past K (at most NT C J).  Four waves, one a
// SIMD, for rows of up to 2048: what every wave does alike (its sums, the row's scalar, the
// step) was half of the work with sixteen.  norm and quantise have a barrier each: the
// block's other waves call lds_barrier for them.  With NT 64 every wave has a row of its
// own, and quantise no barrier.
//
// The arithmetic is FP64 rounding down (q48_round_down) where a wave's words allow it,
// integer elsewhere, per wave.  For integers below LIM: floor(x r / 2^48) is the floor of
// one rounded product, since rounding down passes no integer that a double holds; r is
// split where it has more than 53 bits (x is below 2^53 2^48 / r then, so its product with
// the low part is exact, and a fused operation rounds the sum once).  A code's quotient is
// an estimate that is at most one off, settled by a remainder that is exact.  Per word of
// norm and code some 35 operations of full rate, where the integers' 64-bit products are
// 12 of quarter rate and 90 others: a row of 2048, normed, to codes in LDS 3.3 us behind its
// load, with integers on sixteen waves 5.5.
template <int NT, int C, int J>
struct RowWords {
    static constexpr double LIM = 0x1p53 - 0x1p47;
    static constexpr uint64_t STEP_LIM = (uint64_t)1 << 46;   // LIM / 127 rounded up, and more
    union Word {
        int64_t i;
        double d;
    };
    Word v[J][C];
    bool dbl = false;   // the wave's words are doubles (uniform)

    static_assert((NT & (NT - 1)) == 0, "whole waves");
    __device__ __forceinline__ static int at(int j)
    {
        return C * (((int)threadIdx.x & (NT - 1)) + NT * j);
    }

    // x is on the boundary of its words only
    __device__ __forceinline__ void load(const int64_t *x, int K)
    {
        typedef int64_t words __attribute__((ext_vector_type(C), aligned(8)));
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int i = at(j);
            if (i + C <= K) {
                const words a = *(const words *)(x + i);
#pragma unroll
                for (int c = 0; c < C; ++c)
                    v[j][c].i = a[c];
            } else {
#pragma unroll
                for (int c = 0; c < C; ++c)
                    v[j][c].i = i + c < K ? x[i + c] : 0;
            }
        }
    }

    template <class F>
    __device__ __forceinline__ static void each(int K, F f)
    {
#pragma unroll
        for (int j = 0; j < J; ++j)
            if (C * NT * j < K)
#pragma unroll
                for (int c = 0; c < C; ++c)
                    f(j, c);
    }

    // words to doubles if all of the wave's are below LIM
    __device__ __forceinline__ void to_doubles(int K)
    {
        uint32_t m = 0;   // of the high halves
        each(K, [&](int j, int c) {
            const int hi = (int)(v[j][c].i >> 32);
            m = max(m, (uint32_t)(hi ^ (hi >> 31)));
        });
        static_assert(LIM == (double)(((uint64_t)1 << 53) - ((uint64_t)1 << 47)), "by halves");
        dbl = !__any(m >= (1u << 21) - (1u << 15));
        if (dbl)
            each(K, [&](int j, int c) { v[j][c].d = (double)v[j][c].i; });
    }
    __device__ __forceinline__ void to_words(int K)
    {
        if (dbl)
            each(K, [&](int j, int c) { v[j][c].i = (int64_t)v[j][c].d; });
        dbl = false;
    }

    __device__ __forceinline__ int64_t word(int j, int c) const
    {
        return dbl ? (int64_t)v[j][c].d : v[j][c].i;
    }

    // rmsnorm (llama_int.c:1048-1058) of the row x that was loaded, by weights w; red: two
    // words a wave
    __device__ __forceinline__ void norm(const int64_t *x, const int64_t *w, int K, uint64_t (*red)[2])
    {
        RowWords g;
        g.load(w, K);
        // squares of halves of 27 and 26 bits, three sums without a carry; of any words in
        // 128 bits
        uint32_t big = 0;
        int64_t hh = 0, hl = 0, ll = 0;
        each(K, [&](int j, int c) {
            const int64_t x = v[j][c].i;
            const int hi = (int)(x >> 32), l = (int)((uint32_t)x & 0x7ffffffu);
            const int h = (int)(x >> 27);
            big |= (uint32_t)(hi ^ (hi >> 31));
            hh += (int64_t)h * h;
            hl += (int64_t)h * l;
            ll += (int64_t)l * l;
        });
        q48_u128 ss = ((q48_u128)(q48_i128)hh << 54) + ((q48_u128)(q48_i128)hl << 28) + (uint64_t)ll;
        const bool fits = !__any(big >= 1u << 21);   // all below 2^53
        if (!fits) {
            ss = 0;
            each(K, [&](int j, int c) { ss += (q48_u128)q48_smul128(v[j][c].i, v[j][c].i); });
        }
        ss = q48_wave_sum128(ss);
        if ((threadIdx.x & 63) == 0) {
            red[threadIdx.x >> 6][0] = (uint64_t)ss;
            red[threadIdx.x >> 6][1] = (uint64_t)(ss >> 64);
        }
        lds_barrier();
        ss = 0;
#pragma unroll 4
        for (int i = 0; i < NT / 64; ++i)
            ss += ((q48_u128)red[i][1] << 64) | red[i][0];
        const int64_t r = rms_inv_of(ss, K);
        const int low = 11 - __builtin_clzll((uint64_t)r | 1);   // bits past 53
        const int64_t rl = low > 0 ? r & (((int64_t)1 << low) - 1) : 0;
        const double rh = (double)(r - rl) * 0x1p-48, rd = (double)rl * 0x1p-48;
        double m = 0;
        each(K, [&](int j, int c) {
            const double a = (double)v[j][c].i, b = (double)g.v[j][c].i;
            const double y = __builtin_floor(__builtin_fma(a, rh, a * rd));
            v[j][c].d = __builtin_floor(y * (b * 0x1p-48));
            m = __builtin_fmax(__builtin_fmax(m, __builtin_fabs(y)),
                               __builtin_fmax(__builtin_fabs(b), __builtin_fabs(v[j][c].d)));
        });
        dbl = fits && !__any(m >= LIM);
        if (!dbl) {   // the words once more
            load(x, K);
            each(K, [&](int j, int c) { v[j][c].i = q48_mul(q48_mul(v[j][c].i, r), g.v[j][c].i); });
        }
    }

    // The row's step; store(i, codes) gets C codes from column i on, bytes of an integer,
    // for every i below 64 KT.  red: a word a wave, not the words of norm's
    template <class Store>
    __device__ __forceinline__ int64_t quantise(int K, int KT, uint64_t *red, Store store)
    {
        uint64_t m = 0;
        if (!dbl)
            to_doubles(K);
        if (dbl) {
            double a = 0;
            each(K, [&](int j, int c) { a = __builtin_fmax(a, __builtin_fabs(v[j][c].d)); });
            m = (uint64_t)q48_wave_max64((int64_t)(uint64_t)a);
        } else {
            each(K, [&](int j, int c) {
                const uint64_t a = q48_magnitude(v[j][c].i);
                m = a > m ? a : m;
            });
            m = (uint64_t)q48_wave_max64((int64_t)(m - 1)) + 1;   // at most 2^63: in order less one
        }
        if constexpr (NT > 64) {
            if ((threadIdx.x & 63) == 0)
                red[threadIdx.x >> 6] = m;
            lds_barrier();
#pragma unroll 4
            for (int i = 0; i < NT / 64; ++i)
                m = red[i] > m ? red[i] : m;
        }
        double rc;
        const uint64_t step = w8_step(m, rc);
        if (step > STEP_LIM)   // another wave's words
            to_words(K);
        const double sd = (double)step, half = (double)(step >> 1);
        const bool d = dbl;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            if (at(j) >= 64 * KT)
                break;
            uint32_t codes = 0;
            if (C * NT * j < K && step) {
                if (d) {
#pragma unroll
                    for (int c = 0; c < C; ++c) {
                        const double n = __builtin_fabs(v[j][c].d) + half;
                        double q = __builtin_floor(n * rc);
                        const double rem = __builtin_fma(-q, sd, n);
                        q += rem < 0 ? -1.0 : rem >= sd ? 1.0 : 0.0;
                        q = __builtin_copysign(__builtin_fmin(q, 127.0), v[j][c].d);
                        codes |= (uint32_t)(uint8_t)(int)q << (8 * c);
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < C; ++c)
                        codes |= (uint32_t)(uint8_t)q48_code<127>(v[j][c].i, step, rc) << (8 * c);
                }
            }
            store(at(j), codes);
        }
        return (int64_t)step;
    }
};

} // namespace

// One multiplication by weights, as the kernels get it.
struct W8Mul {
    const uint8_t *A, *A2;        // weight tiles (of expert 0); A2: the up projection's
    const int64_t *sw, *sw2;      // steps of their rows
    size_t a_stride;              // bytes from one expert's tiles to the next one's
    int N, KT;                    // weight rows; tiles of 64 columns
    const uint8_t *B;             // row tiles
    const int64_t *sb;            // steps of the rows
    int T;                        // rows
    int64_t *Y;
    const int64_t *base;
    // experts: items {expert, first slot, slots (at most rows), 0}, a slot's token (-1: none)
    // and weight
    int rows;   // 16, 32, 64 or 128
    const int4 *items;
    const int *slot_tok;
    const int64_t *slot_w;
};

// Rows of words to 8 bits (k_w8_rows): tiles and steps; with norm_w after RMSNorm, whose
// words go to xn too if that is given.  tok: rows whose entry is negative are left out.
// With out, out[row] = base[row] (or zeros).
struct W8Rows {
    uint8_t *codes;
    int64_t *step;
    const int64_t *X, *norm_w;
    int64_t *xn;
    const int *tok;
    int64_t *out;
    const int64_t *base;
    int T, K;
};

// (blocks: 0, or T rounded up to 16: rows past T get zero codes)
int q48_launch_w8_rows(q48_ctx *c, const W8Rows &r, int blocks = 0);
// epi: 0 Y = base + product, 1 SwiGLU of two, 2 weighted adds to the tokens' rows of Y
int q48_launch_w8_mul(q48_ctx *c, const W8Mul &m, int epi, bool experts, int n_items);
// One row, or one slot an item, in one launch: X the words that are put into 8 bits on the
// way (experts: the slots' rows; gate and up of experts take codes, m.B).
inline bool q48_w8_one_ok(int K) { return K <= 8192; }
int q48_launch_w8_one(q48_ctx *c, const W8Mul &m, int epi, const int64_t *X,
                      const int64_t *norm_w, int K, int n_items);
// Grow the buffer that the 8-bit ops keep between launches (stream-synchronising).  Its
// first W8_TICKETS bytes are counters, zeros between launches.
int q48_w8_reserve(q48_ctx *c, size_t bytes);
bool q48_w8_ok(const q48_w8 *w);
// whether two arrays (or a null one) have bytes in common
inline bool q48_share(const void *a, size_t na, const void *b, size_t nb)
{
    return a && b && (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}

constexpr size_t W8_TICKETS = 8192;
constexpr int W8_MAX_K = 1 << 17;        // |S| <= 2^14 K stays below 2^31
constexpr int W8_MAX_N = 1 << 24;
constexpr int W8_MAX_COUNT = 1024;
constexpr int W8_MAX_T = 1 << 20;
inline int w8_kt(int K) { return (K + 63) / 64; }
inline size_t w8_tiles(int rows, int K) { return (size_t)((rows + 15) / 16) * w8_kt(K) * 1024; }
