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

// u^2 of |x|: three products
__device__ __forceinline__ q48_u128 w8_square(int64_t x)
{
    const uint64_t u = q48_magnitude(x);
    const uint32_t l = (uint32_t)u, h = (uint32_t)(u >> 32);
    const uint64_t ll = (uint64_t)l * l, lh = (uint64_t)l * h, hh = (uint64_t)h * h;
    return ((q48_u128)hh << 64) + ((q48_u128)lh << 33) + ll;
}

// A row of words over the first NT threads of a block, in registers: thread i holds words
// C (i + NT j) + 0 .. C - 1 for j < J, zeros past K (at most NT C J).  Four waves, one a
// SIMD, for rows of up to 2048: what every wave does alike (its sums, the row's scalar, the
// step) is half of the work with sixteen (norm and codes of 2048 words 5.4 us, of which
// 1.8 the words' own).  norm and quantise have a barrier each: the block's other waves
// call lds_barrier for them.
template <int NT, int C, int J>
struct RowWords {
    int64_t v[J][C];

    __device__ __forceinline__ static int at(int j) { return C * ((int)threadIdx.x + NT * j); }

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
                    v[j][c] = a[c];
            } else {
#pragma unroll
                for (int c = 0; c < C; ++c)
                    v[j][c] = i + c < K ? x[i + c] : 0;
            }
        }
    }

    // rmsnorm (llama_int.c:1048-1058) of the row by weights g; red: two words a wave
    __device__ __forceinline__ void norm(const RowWords &g, int K, uint64_t (*red)[2])
    {
        q48_u128 ss = 0;
#pragma unroll
        for (int j = 0; j < J; ++j)
            if (C * NT * j < K)
#pragma unroll
                for (int c = 0; c < C; ++c)
                    ss += w8_square(v[j][c]);
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
#pragma unroll
        for (int j = 0; j < J; ++j)
            if (C * NT * j < K)
#pragma unroll
                for (int c = 0; c < C; ++c)
                    v[j][c] = q48_mul(q48_mul(v[j][c], r), g.v[j][c]);
    }

    // The row's step; store(i, codes) gets C codes from column i on, bytes of an integer,
    // for every i below 64 KT.  red: a word a wave, not the words of norm's
    template <class Store>
    __device__ __forceinline__ int64_t quantise(int K, int KT, uint64_t *red, Store store)
    {
        uint64_t m = 0;
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const uint64_t a = q48_magnitude(v[j][c]);
                m = a > m ? a : m;
            }
        m = (uint64_t)q48_wave_max64((int64_t)(m - 1)) + 1;   // at most 2^63: in order less one
        if ((threadIdx.x & 63) == 0)
            red[threadIdx.x >> 6] = m;
        lds_barrier();
#pragma unroll 4
        for (int i = 0; i < NT / 64; ++i)
            m = red[i] > m ? red[i] : m;
        double rc;
        const uint64_t step = w8_step(m, rc);
#pragma unroll
        for (int j = 0; j < J; ++j) {
            if (at(j) >= 64 * KT)
                break;
            uint32_t q = 0;
            if (C * NT * j < K && step)
#pragma unroll
                for (int c = 0; c < C; ++c)
                    q |= (uint32_t)(uint8_t)q48_code<127>(v[j][c], step, rc) << (8 * c);
            store(at(j), q);
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
    // experts: items {expert, first slot, slots, 0}, a slot's token (-1: none) and weight
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

int q48_launch_w8_rows(q48_ctx *c, const W8Rows &r);
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
