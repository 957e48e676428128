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
// Grow the buffer that the 8-bit ops keep between launches (stream-synchronising).
int q48_w8_reserve(q48_ctx *c, size_t bytes);
bool q48_w8_ok(const q48_w8 *w);
// whether two arrays (or a null one) have bytes in common
inline bool q48_share(const void *a, size_t na, const void *b, size_t nb)
{
    return a && b && (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}

constexpr int W8_MAX_K = 1 << 17;        // |S| <= 2^14 K stays below 2^31
constexpr int W8_MAX_N = 1 << 24;
constexpr int W8_MAX_COUNT = 1024;
constexpr int W8_MAX_T = 1 << 20;
inline int w8_kt(int K) { return (K + 63) / 64; }
inline size_t w8_tiles(int rows, int K) { return (size_t)((rows + 15) / 16) * w8_kt(K) * 1024; }
