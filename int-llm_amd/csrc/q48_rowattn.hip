// q48_rowattn.hip — exact attention over a quantised cache (single tokens, rows)
// and of masked rows over the int64 cache (trees of drafted tokens); the
// arithmetic is the reference's exact attention path (llama_int.c:1502-1529,
// softmax 1060-1072) on the values the cache stands for.
#include <type_traits>

#include "q48_digits.hpp"
#include "q48_quant.hpp"

namespace {

constexpr int RA_MAX_POS = 32767;   // a softmax row's sum stays below 2^63
constexpr int RA_MAX_HEADS = 1024;  // the tiles of a launch stay below 65536 (a grid's y)

// The operands of one launch; k, v, ks, vs at the layer's row 0 (int64 words in
// k and v, and no steps, where the cache is not quantised).
struct RaArgs {
    int64_t *out;
    const int64_t *q;        // row t, head h: q + t ldq + h HD
    size_t ldq;
    const uint8_t *k, *v;
    const int64_t *ks, *vs;
    const uint64_t *mask;    // [T][words], or null: causal
    int64_t scale;
    const int *d_pos;        // decode: device position, or null: p0
    int p0, T, words, n_heads, n_kv, max_seq;
    // decode: the new token's key and value, and the RoPE tables (null: rotated)
    const int64_t *k_new, *v_new, *cos_t, *sin_t;
};

// dim d of a head's codes as the cache holds them
template <int BITS, int HD>
__device__ __forceinline__ int code_at(const uint8_t *row, int d)
{
    if (BITS == 8)
        return (int8_t)row[d];
    const int b = (int8_t)row[d & (HD / 2 - 1)];
    return d < HD / 2 ? (b << 28) >> 28 : b >> 4;
}

template <int BITS, int HD>
__device__ __forceinline__ int64_t value_at(const uint8_t *codes, const int64_t *steps, size_t row,
                                            int d)
{
    if constexpr (BITS == 64)
        return reinterpret_cast<const int64_t *>(codes)[row * HD + d];
    else
        return (int64_t)((uint64_t)(int64_t)code_at<BITS, HD>(codes + row * (HD * BITS / 8), d) *
                         (uint64_t)steps[row]);
}

// The new token's key (rotated where the tables are given) and value of KV head kh
// as the cache holds them, by 32 threads: into nk and nst, and into the cache's row.
template <int BITS, int HD>
__device__ __forceinline__ void new_row(const RaArgs &a, int pos, int kh, int tid,
                                        uint8_t (*nk)[HD], int64_t *nst, bool store)
{
    if constexpr (BITS != 64) {
        constexpr int N = HD / 32;
        const int l = tid & 15, i0 = l * N, isv = tid >> 4;
        const int64_t *x = (isv ? a.v_new : a.k_new) + (size_t)kh * HD;
        int64_t lo[N], hi[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            lo[i] = x[i0 + i];
            hi[i] = x[i0 + i + HD / 2];
            if (a.cos_t && !isv)
                q48_rope_pair(lo[i], hi[i], a.cos_t[(size_t)pos * (HD / 2) + i0 + i],
                              a.sin_t[(size_t)pos * (HD / 2) + i0 + i]);
        }
        q48_quantise_row<BITS, HD>(nk[isv], &nst[isv], l, lo, hi);
        if (store) {
            const size_t row = (size_t)pos * a.n_kv + kh;
            q48_quantise_row<BITS, HD>(
                const_cast<uint8_t *>(isv ? a.v : a.k) + row * (HD * BITS / 8),
                const_cast<int64_t *>(isv ? a.vs : a.ks) + row, l, lo, hi);
        }
    }
}

__device__ __forceinline__ int64_t row16_max64(int64_t v)
{
    int64_t o = (int64_t)q48_dpp64<Q48_DPP_XOR1>((uint64_t)v);
    v = o > v ? o : v;
    o = (int64_t)q48_dpp64<Q48_DPP_XOR2>((uint64_t)v);
    v = o > v ? o : v;
    o = (int64_t)q48_dpp64<Q48_DPP_HALF_MIRROR>((uint64_t)v);
    v = o > v ? o : v;
    o = (int64_t)q48_dpp64<Q48_DPP_MIRROR>((uint64_t)v);
    return o > v ? o : v;
}

// A launch's query vectors are, per KV head, v = (t - t0) G + g (row t, query
// head kh G + g), taken in tiles of up to 16 (the rows of one MFMA tile).  Two
// forms of the same phases:
//  - one launch: a block takes a tile over all its rows, scores in LDS (k_ra_tile);
//  - three launches over (chunk of rows, tile of 16, KV head) blocks with the
//    scores in the workspace (k_ra_score, k_ra_exp, k_ra_value), for spans past
//    LDS and where the tiles alone leave compute units idle.  The softmax of the
//    exact path needs the row's maximum before the first exponential and the whole
//    sum before the first quotient, and its truncations leave no way to rescale
//    later, so each of the two is a launch boundary.
struct RaPlan {
    int64_t *sc;     // [n_kv][tv tiles][spad]: scores, then exponentials
    int64_t *cm;     // [n_kv][tv tiles][n1]: a chunk's maximum
    uint64_t *cs;    // [n_kv][tv tiles][n2]: a chunk's sum of exponentials
    int *far;        // [n_kv][tiles][n1]: a visible score outside [-2^62, 2^62)
    int *odd;        // [n_kv][tiles][n2]: an exponential outside [0, ONE]
    int ch1, n1, ch2, n2, ch3, n3;   // rows a chunk, and chunks, of each launch
    int spad, tiles, t0, Tn;         // rows t0 .. t0 + Tn - 1 of the T
    int vb;                          // vectors a tile (one launch)
    int tv;                          // vectors a tile has room for: 16, or those of a single
                                     // tile of fewer
};

// rows [0, span) hold all that vectors up to vlast may see
template <bool DEC>
__device__ __forceinline__ int tile_span(const RaArgs &a, const RaPlan &p, int vlast, int G, int p0)
{
    if (DEC)
        return p0 + 1;
    if (a.mask)
        return p0 + a.T;
    const int last = vlast / G;
    return p0 + p.t0 + (last < p.Tn ? last + 1 : p.Tn);
}

// rows [0, clear) are seen by row t and every later row of its tile
template <bool DEC>
__device__ __forceinline__ int rows_clear(const RaArgs &a, int p0, int t)
{
    return DEC || (!a.mask) ? p0 + t + 1 : p0;
}

// whether row t sees cache row j (j < span)
template <bool DEC>
__device__ __forceinline__ bool sees(const RaArgs &a, int p0, int t, int j)
{
    if (DEC || j < p0)
        return true;
    if (a.mask)
        return j - p0 < a.T &&
               (a.mask[(size_t)t * a.words + ((j - p0) >> 6)] >> ((j - p0) & 63) & 1);
    return j - p0 <= t;
}

// whether any of the rows t0 .. t1 sees cache row j: a row that none sees (padding
// that was never stored) may hold anything
template <bool DEC>
__device__ __forceinline__ bool seen(const RaArgs &a, int p0, int t0, int t1, int j)
{
    if (DEC || j < p0 || !a.mask)
        return true;
    bool any = false;
    for (int t = t0; t <= t1; ++t)
        any |= sees<DEC>(a, p0, t, j);
    return any;
}

template <bool DEC>
__device__ __forceinline__ bool position(const RaArgs &a, int &p0)
{
    p0 = a.p0;
    if (DEC) {
        if (a.d_pos)
            p0 = *a.d_pos;
        return p0 >= 0 && p0 < a.max_seq;
    }
    return true;
}

// ---- keys as MFMA operands -----------------------------------------------------
// Lane (j = lane % 16, kq = lane / 16) holds dims 64 ks + 16 kq .. + 15 of its row,
// as loaded: int64 words, or the bytes of the codes (4 bits, HD 128: one load
// holds both ks, the low and the high halves).
template <int BITS, int HD>
struct KeyRow {
    static constexpr int KS = HD < 64 ? 1 : HD / 64, NL = BITS == 8 ? KS : 1;
    v4i w[NL];
    uint64_t step;
    __device__ __forceinline__ void load(const RaArgs &a, size_t row, int kq)
    {
        const uint8_t *k = a.k + row * (HD * BITS / 8);
#pragma unroll
        for (int n = 0; n < NL; ++n) {
            const int d0 = min(64 * n + 16 * kq, HD - 16);
            w[n] = *reinterpret_cast<const v4i *>(k + (BITS == 8 ? d0 : d0 & (HD / 2 - 1)));
        }
        step = (uint64_t)a.ks[row];
    }
    __device__ __forceinline__ void fresh(const uint8_t *k, uint64_t st, int kq)
    {
#pragma unroll
        for (int n = 0; n < NL; ++n) {
            const int d0 = min(64 * n + 16 * kq, HD - 16);
            w[n] = *reinterpret_cast<const v4i *>(k + (BITS == 8 ? d0 : d0 & (HD / 2 - 1)));
        }
        step = st;
    }
    __device__ __forceinline__ v4i operand(int ks, int kq) const
    {
        if constexpr (BITS == 8) {
            return w[ks];
        } else {
            const int sh = min(64 * ks + 16 * kq, HD - 16) < HD / 2 ? 0 : 4;
            v4i o;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // a nibble n as a signed byte: (n ^ 8) - 8 without borrows
                const uint32_t n = ((uint32_t)w[0][i] >> sh) & 0x0F0F0F0Fu;
                o[i] = (int)(((n ^ 0x08080808u) + 0x78787878u) ^ 0x80808080u);
            }
            return o;
        }
    }
};

// bits 48 .. 111 of step * sum_d q_d c_d from the digit sums: with q = sum_a s_a
// 256^a + C (q48_digits.hpp), D = sum_d q_d c_d = sum_a 256^a acc[a] + C cs, below
// 2^80 (|acc| <= 128 127 128 < 2^21).  c0 and c1: the low and high word of C times cs =
// sum_d c_d, and 2^80 in all, 2^48 of it in c0, so that both halves and D + 2^80 are
// positive; step 2^32 comes off at the end.  22 operations (38 with signed words).
__device__ __forceinline__ int64_t code_dot(const v4i (&acc)[8], int i, int64_t c0, int64_t c1,
                                            uint64_t step)
{
    int64_t lo = mad_shl<0>(acc[0][i], c0), hi = mad_shl<0>(acc[4][i], c1);
    lo = mad_shl<8>(acc[1][i], lo);
    hi = mad_shl<8>(acc[5][i], hi);
    lo = mad_shl<16>(acc[2][i], lo);
    hi = mad_shl<16>(acc[6][i], hi);
    lo = mad_shl<24>(acc[3][i], lo);
    hi = mad_shl<24>(acc[7][i], hi);
    hi += (int64_t)(uint32_t)((uint64_t)lo >> 32);
    // words n0, n1, n2 of the sum, s0 and s1 of the step (below 2^61)
    const uint32_t n0 = (uint32_t)lo, n1 = (uint32_t)hi, n2 = (uint32_t)((uint64_t)hi >> 32);
    const uint32_t s0 = (uint32_t)step, s1 = (uint32_t)(step >> 32);
    const uint64_t t = (uint64_t)n0 * s1 + __umulhi(n0, s0);   // from bit 32, below 2^62
    uint64_t u;                                                // n1 s0 + t, and its carry
    uint32_t carry;
    asm("v_mad_u64_u32 %0, vcc, %2, %3, %4\n\t"
        "s_nop 1\n\t"
        "v_addc_co_u32_e64 %1, vcc, 0, 0, vcc"
        : "=&v"(u), "=v"(carry)
        : "v"(n1), "v"(s0), "v"(t)
        : "vcc");
    uint64_t w = (uint64_t)n1 * s1 + (((uint64_t)carry << 32) | (uint32_t)(u >> 32));
    w += (uint64_t)n2 * s0;                                    // from bit 64, 48 bits needed
    const uint32_t w1 = (uint32_t)(w >> 32) + n2 * s1;
    return (int64_t)(((uint64_t)(__builtin_amdgcn_alignbit(w1, (uint32_t)w, 16) - s0) << 32) |
                     __builtin_amdgcn_alignbit((uint32_t)w, (uint32_t)u, 16));
}

// int64 keys as loaded, 16 dims a lane (dims past the head give digits of zero)
template <int HD>
struct WordRow {
    uint64_t x[HD < 64 ? 16 : HD / 4];
    __device__ __forceinline__ void load(const RaArgs &a, size_t row, int kq)
    {
        const uint64_t *k = reinterpret_cast<const uint64_t *>(a.k) + row * HD;
#pragma unroll
        for (int ks = 0; ks < (HD < 64 ? 1 : HD / 64); ++ks)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int d = 64 * ks + 16 * kq;
                x[16 * ks + e] = d < HD ? k[d + e] : kDig;
            }
    }
};

// Digits of a tile's queries as the A operands of the score products, and C sum_d
// q_d for int64 keys, by NT threads; qs: rotated queries in LDS, or null.
template <int BITS, int HD, int NT>
__device__ __forceinline__ void query_digits(const RaArgs &a, const RaPlan &p,
                                             v4i (*dig)[8][64], q48_u128 *cq, int v0, int vlast,
                                             int G, int kh, const int64_t *qs, int tid)
{
    constexpr int KS = HD < 64 ? 1 : HD / 64;
    for (int it = tid; it < KS * 64; it += NT) {
        const int ks = it >> 6, l = it & 63;
        const int v = min(v0 + (l & 15), vlast), d0 = 64 * ks + 16 * (l >> 4);
        uint64_t x[16];
        if (d0 < HD) {
            const int64_t *q =
                qs ? qs + (v - v0) * HD + d0
                   : a.q + (size_t)(p.t0 + v / G) * a.ldq + (size_t)(kh * G + v % G) * HD + d0;
#pragma unroll
            for (int e = 0; e < 16; ++e)
                x[e] = (uint64_t)q[e];
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e)
                x[e] = kDig;   // digits of zero
        }
        if constexpr (BITS == 64) {
            q48_u128 sum = 0;
            if (d0 < HD)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    sum += (q48_u128)(q48_i128)(int64_t)x[e];
            sum += shfl_xor128(sum, 16);   // the four lanes of a row are in one wave
            sum += shfl_xor128(sum, 32);
            if (l < 16)
                cq[16 * ks + l] = sum * kDig;
        }
        v4i o[8];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const uint64_t x4[4] = {x[4 * g], x[4 * g + 1], x[4 * g + 2], x[4 * g + 3]};
            uint32_t wd[8];
            digits4(x4, wd);
#pragma unroll
            for (int d = 0; d < 8; ++d)
                o[d][g] = (int)wd[d];
        }
#pragma unroll
        for (int d = 0; d < 8; ++d)
            dig[ks][d][l] = o[d];
    }
}

// A tile's scores before the scale: s[i] = (sum_d q_d k_d) >> 48 of row j's key and
// the tile's vector 4 kq + i.
template <int HD>
__device__ __forceinline__ void code_scores(int64_t (&s)[4], const v4i (*dig)[8][64],
                                            const v4i (&B)[HD < 64 ? 1 : HD / 64], int64_t c0,
                                            int64_t c1, uint64_t step, int lane, int nrow)
{
    constexpr int KS = HD < 64 ? 1 : HD / 64;
    v4i acc[8];
#pragma unroll
    for (int d = 0; d < 8; ++d)
        acc[d] = (v4i){0, 0, 0, 0};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int d = 0; d < 8; ++d)
            acc[d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(dig[ks][d][lane], B[ks], acc[d], 0, 0,
                                                          0);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i == 0 || i < nrow)   // a short tile has no vector 4 kq + i
            s[i] = code_dot(acc, i, c0, c1, step);
}

// C's low and high word times sum_d c_d of the operand's row (and the bias code_dot wants),
// on every lane: a product with a row of ones
template <int HD>
__device__ __forceinline__ void code_sum(int64_t &c0, int64_t &c1,
                                         const v4i (&B)[HD < 64 ? 1 : HD / 64], int kq)
{
    v4i sum = {0, 0, 0, 0};
#pragma unroll
    for (int ks = 0; ks < (HD < 64 ? 1 : HD / 64); ++ks) {
        const int o = 64 * ks + 16 * kq < HD ? 0x01010101 : 0;
        sum = __builtin_amdgcn_mfma_i32_16x16x64_i8((v4i){o, o, o, o}, B[ks], sum, 0, 0, 0);
    }
    c0 = (int64_t)(uint32_t)kDig * sum[0] + ((int64_t)1 << 48);
    c1 = (int64_t)(uint32_t)(kDig >> 32) * sum[0] + ((int64_t)1 << 48) - (1 << 16);
    // the product's other three words are not reused while it may still write them
    asm("" : : "v"(sum), "v"(c0), "v"(c1));
}

// Operands of 16 int64 key rows (eight digit planes), and C sum_d k_d - HD C^2
template <int HD>
__device__ __forceinline__ q48_u128 key_digits(v4i (&B)[HD < 64 ? 1 : HD / 64][8],
                                               const WordRow<HD> &k, int kq)
{
    constexpr int KS = HD < 64 ? 1 : HD / 64;
    q48_u128 ck = 0;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const bool in = 64 * ks + 16 * kq < HD;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            uint64_t x4[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x4[e] = k.x[16 * ks + 4 * g + e];
                if (in)
                    ck += (q48_u128)(q48_i128)(int64_t)x4[e];
            }
            uint32_t wd[8];
            digits4(x4, wd);
#pragma unroll
            for (int d = 0; d < 8; ++d)
                B[ks][d][g] = (int)wd[d];
        }
    }
    ck += shfl_xor128(ck, 16);
    ck += shfl_xor128(ck, 32);
    return ck * kDig - (q48_u128)kDig * kDig * (q48_u128)HD;
}

// The 63 digit products by the weight of their sum, 256^d: two chains at a time, and
// each sum joins the score as soon as it is whole, under the next pair's products.  All 14
// at once would take 56 registers for their sums alone, where the operands of both sides
// leave k_ra_score two waves a SIMD (222 registers) as it is.
template <int HD>
__device__ __forceinline__ void word_scores(int64_t (&s)[4], const v4i (*dig)[8][64],
                                            const v4i (&B)[HD < 64 ? 1 : HD / 64][8],
                                            const q48_u128 *cq, q48_u128 ck, int lane, int nrow)
{
    constexpr int KS = HD < 64 ? 1 : HD / 64;
    v4i A[KS][8];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int x = 0; x < 8; ++x)
            A[ks][x] = dig[ks][x][lane];
    uint32_t c[4][4], w1[4], w2[4];
    int64_t cur[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int m = 4 * (lane >> 4) + i;
        q48_u128 t = cq[m] + ck;
        if (KS == 2)
            t += cq[16 + m];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            c[i][k] = (uint32_t)(t >> (32 * k));
        cur[i] = (int64_t)c[i][0];
    }
    v4i acc[2][2];
#pragma unroll
    for (int d = 0; d < 16; d += 2) {
        // the products of this pair of weights, under the last pair's sums
        v4i(&now)[2] = acc[d / 2 & 1];
        if (d < 14) {
            now[0] = now[1] = (v4i){0, 0, 0, 0};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int x = 0; x < 8; ++x)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        if (d + e - x >= 0 && d + e - x < 8)
                            now[e] = __builtin_amdgcn_mfma_i32_16x16x64_i8(
                                A[ks][x], B[ks][d + e - x], now[e], 0, 0, 0);
        }
        if (d > 0) {
            const v4i(&was)[2] = acc[d / 2 - 1 & 1];
            const int k = d - 2;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (k == 4 || k == 8 || k == 12) {   // bits 8 k on, with the carry
                    if (k == 8)
                        w1[i] = (uint32_t)cur[i];
                    if (k == 12)
                        w2[i] = (uint32_t)cur[i];
                    cur[i] = (cur[i] >> 32) + (int64_t)c[i][k / 4];
                }
                // |was| <= 8 KS 64 128 128 = 2^24: four stay below 2^49
                cur[i] = (k & 2) ? mad_shl<24>(was[1][i], mad_shl<16>(was[0][i], cur[i]))
                                 : mad_shl<8>(was[1][i], mad_shl<0>(was[0][i], cur[i]));
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i == 0 || i < nrow)
            s[i] = (int64_t)(((uint64_t)__builtin_amdgcn_alignbit((uint32_t)cur[i], w2[i], 16)
                              << 32) |
                             __builtin_amdgcn_alignbit(w2[i], w1[i], 16));
}

// whether the next rows' keys are loaded ahead (int64: where the registers allow)
constexpr bool keys_ahead(int bits, int hd, int tb) { return bits != 64 || (hd < 128 && tb == 1); }

// Scores of TB tiles (vectors v0 .. of 16 each) over rows [begin, end), 16 rows a
// wave at a time (wave w of NW); put(tb, m, j, s) takes vector m's score, and mx
// and far gather each tile's maxima over the rows seen and far scores.
template <int BITS, int HD, int TB, int NW, bool DEC, typename Put>
__device__ __forceinline__ void score_rows(const RaArgs &a, const v4i (*dig)[HD < 64 ? 1 : HD / 64][8][64],
                                           const q48_u128 (*cq)[HD < 64 ? 16 : HD / 4],
                                           const int *vt, int ntile, int nrow, int kh, int p0,
                                           int begin, int end, const uint8_t *nk, int64_t nst,
                                           int clear, int w, int lane, int64_t (&mx)[TB][4],
                                           uint32_t (&far)[TB],
                                           std::conditional_t<BITS == 64, WordRow<HD>,
                                                              KeyRow<BITS == 64 ? 8 : BITS, HD>> &next,
                                           Put put)
{
    constexpr int KS = HD < 64 ? 1 : HD / 64;
    const int rl = lane & 15, kq = lane >> 4;
    constexpr bool AHEAD = keys_ahead(BITS, HD, TB);
    for (int j0 = begin + 16 * w; j0 < end; j0 += 16 * NW) {
        const int j = j0 + rl, jc = min(j, end - 1);
        const bool all = j0 + 16 <= clear;   // (clear <= end)
        const size_t row = (size_t)jc * a.n_kv + kh;
        v4i B[KS][BITS == 64 ? 8 : 1];
        q48_u128 ck = 0;
        int64_t c0 = 0, c1 = 0;
        uint64_t step = 0;
        v4i C[KS];
        if constexpr (BITS == 64) {
            if (!AHEAD)
                next.load(a, row, kq);
            ck = key_digits<HD>(B, next, kq);
            if (AHEAD && j0 + 16 * NW < end)
                next.load(a, (size_t)min(j + 16 * NW, end - 1) * a.n_kv + kh, kq);
        } else {
            KeyRow<BITS, HD> now = next;
            if (j0 + 16 * NW < end)
                next.load(a, (size_t)min(j + 16 * NW, end - 1) * a.n_kv + kh, kq);
            if (DEC && jc == p0)
                now.fresh(nk, (uint64_t)nst, kq);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
                C[ks] = now.operand(ks, kq);
            step = now.step;
            code_sum<HD>(c0, c1, C, kq);
        }
#pragma unroll
        for (int tb = 0; tb < TB; ++tb) {
            if (tb >= ntile)
                break;
            int64_t s[4];
            if constexpr (BITS == 64) {
                word_scores<HD>(s, dig[tb], B, cq[tb], ck, lane, nrow);
            } else
                code_scores<HD>(s, dig[tb], C, c0, c1, step, lane, nrow);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (i > 0 && i >= nrow)
                    break;
                const int m = 4 * kq + i;
                // the scale of 64-wide heads is 2^45: a shift
                s[i] = HD == 64 ? s[i] >> 3 : q48_mul(s[i], a.scale);
                if (all || j < end)
                    put(tb, m, j, s[i]);
                if (all || (j < end && sees<DEC>(a, p0, vt[tb * 16 + m], j))) {
                    far[tb] |= (uint32_t)((uint64_t)s[i] >> 32) + 0x40000000u;
                    mx[tb][i] = s[i] > mx[tb][i] ? s[i] : mx[tb][i];
                }
            }
        }
    }
}

// ---- values as doubles ------------------------------------------------------------

// v[n] = c[n] st of lane n of each row of 16 lanes (exact below 2^53), n < 16:
// row_newbcast hands a row's steps to its lanes.  The four moves cover the wait
// states between a vector write of st and its DPP read.
__device__ __forceinline__ void scale16(double (&v)[16], const double (&c)[16], double st)
{
#define RA_MUL4(A, B, C, D)                                                                      \
    asm("v_mov_b64_e32 %0, 0\n\t"                                                                \
        "v_mov_b64_e32 %1, 0\n\t"                                                                \
        "v_mov_b64_e32 %2, 0\n\t"                                                                \
        "v_mov_b64_e32 %3, 0\n\t"                                                                \
        "v_fmac_f64_dpp %0, %4, %5 row_newbcast:" #A " row_mask:0xf bank_mask:0xf\n\t"          \
        "v_fmac_f64_dpp %1, %4, %6 row_newbcast:" #B " row_mask:0xf bank_mask:0xf\n\t"          \
        "v_fmac_f64_dpp %2, %4, %7 row_newbcast:" #C " row_mask:0xf bank_mask:0xf\n\t"          \
        "v_fmac_f64_dpp %3, %4, %8 row_newbcast:" #D " row_mask:0xf bank_mask:0xf"              \
        : "=&v"(v[A]), "=&v"(v[B]), "=&v"(v[C]), "=&v"(v[D])                                     \
        : "v"(st), "v"(c[A]), "v"(c[B]), "v"(c[C]), "v"(c[D]))
    RA_MUL4(0, 1, 2, 3);
    RA_MUL4(4, 5, 6, 7);
    RA_MUL4(8, 9, 10, 11);
    RA_MUL4(12, 13, 14, 15);
#undef RA_MUL4
}

// Where a lane's values are: byte offsets from the first row of a group of CP rows,
// for its 16 rows vp + n at dim vd (a byte of 4-bit codes holds dims b and b + HD /
// 2), made once: the loads then take a scalar base and these.
template <int BITS, int HD>
struct ValueRows {
    static constexpr int DL = HD == 128 ? 2 : 1, CP = HD == 32 ? 32 : 16, RB = HD * BITS / 8;
    uint32_t off[16];
    uint32_t at;
    int vp, sh;
    const uint8_t *base;
    __device__ __forceinline__ ValueRows(const RaArgs &a, int kh, int lane)
    {
        const int vd = HD == 32 ? lane & 31 : lane;
        vp = HD == 32 ? 16 * (lane >> 5) : 0;
        sh = vd < HD / 2 ? 0 : 4;
        at = BITS == 64 ? 8 * vd : BITS == 8 ? vd : vd & (HD / 2 - 1);
        base = a.v + (size_t)kh * RB;
#pragma unroll
        for (int n = 0; n < 16; ++n)
            off[n] = (uint32_t)(vp + n) * (uint32_t)(a.n_kv * RB) + at;
    }
    // The values of rows j + vp + n (past last: that row's), on their way; j is the
    // wave's.  rl: the lane's place in its row of 16.
    int64_t x[BITS == 64 ? DL : 1][BITS == 64 ? 16 : 1];
    int b[BITS == 64 ? 1 : 16], b2[BITS == 8 && HD == 128 ? 16 : 1];
    int64_t step;
    __device__ __forceinline__ void fetch(const RaArgs &a, int kh, int j, int last, int rl)
    {
        const uint8_t *g = base + (size_t)j * (size_t)(a.n_kv * RB);
        if (j + CP - 1 > last)   // the wave's last group: the offsets are not used again
#pragma unroll
            for (int n = 0; n < 16; ++n)
                off[n] = (uint32_t)min(vp + n, last - j) * (uint32_t)(a.n_kv * RB) + at;
        if constexpr (BITS == 64) {
#pragma unroll
            for (int n = 0; n < 16; ++n)
#pragma unroll
                for (int l = 0; l < DL; ++l)
                    x[l][n] = *reinterpret_cast<const int64_t *>(g + off[n] + 512 * l);
        } else {
#pragma unroll
            for (int n = 0; n < 16; ++n) {
                b[n] = (int8_t)g[off[n]];
                if constexpr (BITS == 8 && HD == 128)
                    b2[n] = (int8_t)g[off[n] + 64];
            }
            step = a.vs[(size_t)min(j + vp + rl, last) * a.n_kv + kh];
        }
    }
    // What was fetched, as doubles; int64 words gather their range in big.  fresh (or
    // null): the codes and the step of row last, which the cache may not hold yet.
    __device__ __forceinline__ void take(double (&v)[DL][16], int j, int last, int rl,
                                         uint32_t &big, const uint8_t *fresh = nullptr,
                                         int64_t fresh_step = 0)
    {
        if constexpr (BITS == 64) {
#pragma unroll
            for (int n = 0; n < 16; ++n)
#pragma unroll
                for (int l = 0; l < DL; ++l)
                    v[l][n] = q48_f51(x[l][n], big);
        } else {
            if (fresh && j + CP - 1 >= last) {
                if (j + vp + rl >= last)
                    step = fresh_step;
#pragma unroll
                for (int n = 0; n < 16; ++n)
                    if (j + vp + n == last) {
                        b[n] = (int8_t)fresh[at];
                        if constexpr (BITS == 8 && HD == 128)
                            b2[n] = (int8_t)fresh[at + 64];
                    }
            }
            const double st = (double)step;
            double c[16];
#pragma unroll
            for (int n = 0; n < 16; ++n)
                c[n] = (double)(BITS == 8
                                    ? b[n]
                                    : (int)__builtin_amdgcn_sbfe(b[n], HD == 128 ? 0 : sh, 4));
            scale16(v[0], c, st);
            if constexpr (DL == 2) {
#pragma unroll
                for (int n = 0; n < 16; ++n) {
                    if constexpr (BITS == 8)
                        c[n] = (double)b2[n];
                    else
                        c[n] = (double)(b[n] >> 4);
                }
                scale16(v[1], c, st);
            }
        }
    }
};

// acc[l][r] += the 16 rows' values under vector r's weights (q(r): this lane's, row
// rl's weight), four vectors at a time, rounding down (q48_fsum4x4): one FP64
// operation a (vector, row, dim); absent vectors are skipped by fours.
template <int HD, typename Weight>
__device__ __forceinline__ void add_values(double (&acc)[HD == 128 ? 2 : 1][16],
                                           const double (&v)[HD == 128 ? 2 : 1][16], int nrow,
                                           Weight weight)
{
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
        if (r >= nrow)
            break;
        double q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            q[i] = weight(r + i);
#pragma unroll
        for (int l = 0; l < (HD == 128 ? 2 : 1); ++l) {
            auto f4 = [&](auto base) {
                constexpr int B = decltype(base)::value;
                const double x[4] = {v[l][B], v[l][B + 1], v[l][B + 2], v[l][B + 3]};
                q48_fsum4x4<B>(acc[l][r], acc[l][r + 1], acc[l][r + 2], acc[l][r + 3], q, x);
            };
            f4(std::integral_constant<int, 0>{});
            f4(std::integral_constant<int, 4>{});
            f4(std::integral_constant<int, 8>{});
            f4(std::integral_constant<int, 12>{});
        }
    }
}

// a step whose values all stay within [-2^51, 2^51), the lowest code's too, which a
// cache that was not quantised here may hold
template <int BITS>
__device__ __forceinline__ bool step_fits(int64_t step)
{
    return (uint64_t)step <= (uint64_t)1 << (52 - BITS);
}

// floor(x^2 / 2^48) for x below 2^56: with h the high word, 2 h and h 2^B fit 32 bits, so
// that the cross term and the high square are one multiply-add each (B <= 12, x below 2^52;
// else 8).
template <int B>
__device__ __forceinline__ uint64_t square_shr48(uint64_t x)
{
    const uint32_t l = (uint32_t)x;
    uint32_t h = (uint32_t)(x >> 32);
    asm("" : "+v"(h));   // (shifts of h, not parts of shifts of x)
    const uint64_t w = (uint64_t)l * (2 * h) + __umulhi(l, l);
    return (uint64_t)(h << B) * (h << (16 - B)) + (w >> 16);
}

// q48_exp_neg in fewer operations (98 -> 80, loads and sums of k_ra_exp included).  Its constants stand where v_fma_f64 takes them
// (a multiply-add whose addend is a constant otherwise copies it first).  The last two
// squares, of at most e^2.5 and e^5, have small high words.  The reciprocal of r takes one
// cubic step, y (1 + d + d^2) with d = 1 - r y: y off by 2^-20 becomes 2^-60, and rounding r
// and y down leaves it within 2^-52 of 1 / r.  Times 2^96 (1 - 2^-50) it is below 2^96 / r <=
// 2^48 by less than 2^-1, so q1 = floor of it, plus 1, is the quotient or one more; q1 r -
// 2^96 lies in (-r, r], and the sign of its low 64 bits tells.
__device__ __forceinline__ uint64_t exp_neg(uint64_t u)
{
    const uint64_t lim = (uint64_t)10 << 48;
    const bool in = u <= lim;
    double h = __builtin_bit_cast(double, 0x4330000000000000ull + (uint64_t)Q48_ONE +
                                              ((in ? u : lim) >> 14));
    const double k24 = 0x1p-24, k28 = -0x1p28, k52 = 0x1p52, k96 = 0x1.ffffffffffff8p95;
    const double one = 0x1p52 + 1;
#pragma unroll
    for (int k = 0; k < 12; ++k) {
        double y;
        asm("v_fma_f64 %0, %1, %2, %3" : "=v"(y) : "v"(h), "s"(k24), "v"(k28));
        asm("v_fma_f64 %0, %1, %1, %2" : "=v"(h) : "v"(y), "s"(k52));
    }
    const uint64_t r = square_shr48<8>(square_shr48<12>(q48_word_m52(h)));
    const double rd = (double)r;
    double y = __builtin_amdgcn_rcp(rd);
    const double d = __builtin_fma(-rd, y, 1.0);
    y = __builtin_fma(y, __builtin_fma(d, d, d), y);
    double q;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(q) : "v"(y), "s"(k96), "v"(one));
    const uint64_t q1 = q48_word_m52(q);
    return in ? q1 - ((int64_t)(q1 * r) > 0 ? 1 : 0) : 0;
}

// The exponentials of vector t's scores row[j], j = begin + l, + L, ..., in place: 0
// where it does not see j, up to `fill` >= end.  Two at a time where every row is
// seen: a chain of 24 dependent operations each.  Returns their sum; odd: one is
// outside [0, ONE] (far: scores whose differences may wrap).
template <bool DEC>
__device__ __forceinline__ uint64_t exp_rows(const RaArgs &a, int p0, int t, int64_t *row,
                                             int64_t m, bool far, int begin, int end, int fill,
                                             int l, int L, int &odd)
{
    uint64_t sum = 0;
    int j = begin + l;
    if (!far) {
        const int clear = min(end, rows_clear<DEC>(a, p0, t));
        for (; j + L < clear; j += 2 * L) {
            const uint64_t e0 = exp_neg((uint64_t)m - (uint64_t)row[j]);
            const uint64_t e1 = exp_neg((uint64_t)m - (uint64_t)row[j + L]);
            row[j] = (int64_t)e0;
            row[j + L] = (int64_t)e1;
            sum += e0 + e1;
        }
    }
    for (; j < fill; j += L) {
        int64_t e = 0;
        if (j < end && sees<DEC>(a, p0, t, j)) {
            if (!far) {
                e = (int64_t)exp_neg((uint64_t)m - (uint64_t)row[j]);
            } else {
                e = q48_safe_exp((int64_t)((uint64_t)row[j] - (uint64_t)m));
                odd |= (uint64_t)e > (uint64_t)Q48_ONE;
            }
        }
        row[j] = e;
        sum += (uint64_t)e;
    }
    return sum;
}

// 2^48 (1 - 2^-50) / d for the quotients of a softmax row (1 <= d < 2^63): as
// q48_divisor_of, whose bound of 2^62 a row past 16384 positions may pass, and always
// below 2^48 / d, by at most 6 units of 2^-52.
__device__ __forceinline__ double quotient_factor(uint64_t d)
{
    const double dd = (double)d;
    double y = __builtin_amdgcn_rcp(dd);
    y = __builtin_fma(y, __builtin_fma(-dd, y, 1.0), y);
    y = __builtin_fma(y, __builtin_fma(-dd, y, 1.0), y);
    return y * 0x1.ffffffffffff8p47;
}

// fp_div(e, den) 2^-48 for 0 <= e <= min(ONE, den), 1 <= den < 2^63, as the reciprocal in
// exp_neg: t = 2^52 + q1, q1 the quotient (at most 2^48) or one more, q1 den - e 2^48 in
// (-den, den]; 2^4 + 2^-48 is the double after 2^4.
__device__ __forceinline__ double quotient_scaled(uint64_t e, uint64_t den, double y48)
{
    const double ed = __builtin_bit_cast(double, e | 0x4330000000000000ull) - 0x1p52;
    const double one = 0x1p52 + 1, k48 = 0x1p-48;
    double t, p;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(t) : "v"(ed), "v"(y48), "v"(one));
    const int64_t over = (int64_t)(q48_word_m52(t) * den - (e << 48));
    const double less = __builtin_bit_cast(double, 0x4030000000000000ull | (over > 0 ? 1 : 0));
    asm("v_fma_f64 %0, %1, %2, -%3" : "=v"(p) : "v"(t), "s"(k48), "v"(less));
    return p;
}

// dim d of a vector's sum over rows [begin, end) in integers.  e: exponentials of
// any kind, the weights fp_div(e, sum) where the sum is positive, else e; or
// (scaled) the weights 2^-48 as doubles.
template <int BITS, int HD>
__device__ int64_t plain_sum(const RaArgs &a, const int64_t *e, int64_t sum, bool scaled, int kh,
                             int d, int begin, int end, const uint8_t *fresh = nullptr,
                             const int64_t *fresh_step = nullptr)
{
    const q48_divisor dv = q48_divisor_of(sum);
    uint64_t o = 0;
    for (int j = begin; j < end; ++j) {
        int64_t x = e[j];
        if (scaled)
            x = (int64_t)(__builtin_bit_cast(double, x) * 0x1p48);
        else if (sum > 0)
            x = q48_div_by(x, dv);
        o += (uint64_t)q48_mul(x, fresh && j == end - 1
                                      ? value_at<BITS, HD>(fresh, fresh_step, 0, d)
                                      : value_at<BITS, HD>(a.v, a.vs, (size_t)j * a.n_kv + kh, d));
    }
    return (int64_t)o;
}

template <int HD>
__device__ __forceinline__ int64_t *out_at(const RaArgs &a, const RaPlan &p, int v, int G, int kh)
{
    return a.out + ((size_t)(p.t0 + v / G) * a.n_heads + kh * G + v % G) * HD;
}

// The tile's queries of a decoded token into LDS (vectors v0 .. v0 + n - 1), rotated
// where the tables are given.
template <int HD, int NT>
__device__ __forceinline__ void decode_queries(const RaArgs &a, int64_t *qs, int v0, int n, int G,
                                               int kh, int p0, int tid)
{
    for (int it = tid; it < n * (HD / 2); it += NT) {
        const int m = it / (HD / 2), i = it % (HD / 2);
        const int64_t *q = a.q + (size_t)(kh * G + v0 + m) * HD;
        int64_t x0 = q[i], x1 = q[i + HD / 2];
        if (a.cos_t)
            q48_rope_pair(x0, x1, a.cos_t[(size_t)p0 * (HD / 2) + i],
                          a.sin_t[(size_t)p0 * (HD / 2) + i]);
        qs[m * HD + i] = x0;
        qs[m * HD + i + HD / 2] = x1;
    }
}

// ---- one launch ----------------------------------------------------------------------

// k_ra_tile's arrays beside the scores (digits, sums, queries, maxima, row sums, the
// rest rounded up), and what a compute unit's 160 KB of LDS leaves for the scores
constexpr size_t rt_static(int hd, int nw)
{
    return (size_t)(hd < 64 ? 1 : hd / 64) * (8 * 1024 + 256) + 16 * hd * 8 + 2 * 16 * nw * 8 +
           2 * hd + 512;
}
constexpr size_t rt_lds(int hd, int nw) { return 160 * 1024 - rt_static(hd, nw); }

// A tile of up to vb vectors over all its rows, the scores in LDS: they become
// exponentials, then weights in place.  8 or 16 waves; a wave takes 16 rows at a time for
// the scores and the values.
// Bound by vector issue where there are tiles for all compute units: 384 rows at 512 (32
// heads on 4 of 64, 8 bits), 8.7 M (vector, row) pairs, in 88 us, about 280 instructions
// per 64 pairs (64 the sums' FP64 operations, 80 the exponential, 20 the quotient) at 82%
// of the rate a SIMD issues FP64 and 64-bit integer operations (one in 4.3 cycles); of a
// block's 33 us the scores take 7, exponentials 11, quotients 3, values and their sums 12.
// Few vectors and rows are a chain of latencies: one token at 120 7.2 us, 1.5 of it the query
// and the new row, 1.3 the scores, 1.0 the exponentials, 0.8 the values.
// A visible step or value past the FP64 range sends the tile to plain_sum, a thread an
// output over all rows: with one value of 9.0 in each head the 384 rows take 1162 us, one
// token at 120 51, at 600 229 (13.9 without).
template <int BITS, int HD, bool DEC, int RT_NT>
__global__ __launch_bounds__(RT_NT) void k_ra_tile(RaArgs a, RaPlan p)
{
    constexpr int RT_NW = RT_NT / 64;
    q48_round_down();
    constexpr int KS = HD < 64 ? 1 : HD / 64;
    constexpr int PG = HD == 32 ? 2 : 1, CP = 16 * PG;
    extern __shared__ __align__(16) int64_t sc[];   // [vb][stride]
    __shared__ v4i dig[1][KS][8][64];
    __shared__ q48_u128 cq[1][16 * KS];
    __shared__ int vt[16];
    __shared__ int64_t mxs[RT_NW][16];
    __shared__ uint64_t psum[16][RT_NW];
    __shared__ int flags;                           // 1: a far score, 2: no plain softmax
    __shared__ __align__(16) uint8_t nk[2][HD];
    __shared__ int64_t nst[2];
    __shared__ uint64_t lam[16][HD];                // a decoded token's queries, then the sums

    static_assert(sizeof(dig) + sizeof(cq) + sizeof(vt) + sizeof(mxs) + sizeof(psum) +
                          sizeof(flags) + sizeof(nk) + sizeof(nst) + sizeof(lam) + 64 <=
                      rt_static(HD, RT_NW),
                  "k_ra_tile's LDS");

    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rl = lane & 15, kq = lane >> 4;
    const int kh = blockIdx.y, G = a.n_heads / a.n_kv, NV = p.Tn * G;
    const int v0 = ((int)gridDim.x - 1 - (int)blockIdx.x) * p.vb;   // the longest spans first
    const int nrow = min(p.vb, NV - v0), stride = p.spad + 4;   // 4 rows on: the other half of the banks
    int p0;
    if (!position<DEC>(a, p0))
        return;
    const int S = tile_span<DEC>(a, p, v0 + nrow - 1, G, p0);

    // the first keys on their way while the queries are split
    std::conditional_t<BITS == 64, WordRow<HD>, KeyRow<BITS == 64 ? 8 : BITS, HD>> next;
    if (keys_ahead(BITS, HD, 1) && 16 * w < S)
        next.load(a, (size_t)min(16 * w + rl, S - 1) * a.n_kv + kh, kq);
    if (tid < 16)
        vt[tid] = p.t0 + min(v0 + tid, NV - 1) / G;
    if (tid == 0)
        flags = 0;
    int64_t *qs = reinterpret_cast<int64_t *>(&lam[0][0]);
    if constexpr (DEC) {
        decode_queries<HD, RT_NT>(a, qs, v0, nrow, G, kh, p0, tid);
        if (tid >= RT_NT - 64 && tid < RT_NT - 32)
            new_row<BITS, HD>(a, p0, kh, tid - (RT_NT - 64), nk, nst, v0 == 0);
        __syncthreads();
    }
    query_digits<BITS, HD, RT_NT>(a, p, dig[0], cq[0], v0, v0 + nrow - 1, G, kh,
                                  DEC ? qs : nullptr, tid);
    __syncthreads();
    for (int i = tid; i < 16 * HD; i += RT_NT)
        (&lam[0][0])[i] = 0;

    {
        int64_t mx[1][4] = {{INT64_MIN, INT64_MIN, INT64_MIN, INT64_MIN}};
        uint32_t far[1] = {0};
        score_rows<BITS, HD, 1, RT_NW, DEC>(a, dig, cq, vt, 1, nrow, kh, p0, 0, S, nk[0],
                                            DEC && BITS != 64 ? nst[0] : 0,
                                            rows_clear<DEC>(a, p0, p.t0 + v0 / G), w, lane, mx,
                                            far, next, [&](int, int m, int j, int64_t s) {
                                                if (m < nrow)
                                                    sc[m * stride + j] = s;
                                            });
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t m = row16_max64(mx[0][i]);
            if (rl == 0)
                mxs[w][4 * kq + i] = m;
        }
        if (far[0] & 0x80000000u)
            atomicOr(&flags, 1);
    }
    __syncthreads();

    // exponentials: a wave takes whole vectors, or 8 / vb waves share one
    const int wr = p.vb >= RT_NW ? 1 : RT_NW / p.vb;   // waves a vector (vb a power of two)
    const int sub = w % wr;
    const int fill = (S + 31) & ~31;
    const bool far = flags & 1;
    int odd = 0;
    for (int r = w / wr; r < nrow; r += RT_NW / wr) {
        int64_t m = mxs[0][r];
#pragma unroll
        for (int u = 1; u < RT_NW; ++u)
            m = mxs[u][r] > m ? mxs[u][r] : m;
        uint64_t sum = exp_rows<DEC>(a, p0, vt[r], sc + r * stride, m, far, 0, S, fill,
                                     lane + 64 * sub, 64 * wr, odd);
        sum = (uint64_t)q48_wave_sum64((int64_t)sum);
        if (lane == 0)
            psum[r][sub] = sum;
    }
    if constexpr (BITS != 64)
        for (int j = tid; j < S; j += RT_NT) {
            const int64_t st = DEC && j == p0 ? nst[1] : a.vs[(size_t)j * a.n_kv + kh];
            odd |= !step_fits<BITS>(st) && seen<DEC>(a, p0, vt[0], vt[nrow - 1], j);
        }
    const bool slow = __syncthreads_or(odd);
    auto total = [&](int r) {
        uint64_t s = 0;
        for (int u = 0; u < wr; ++u)
            s += psum[r][u];
        return s;
    };
    uint32_t big = 0;
    if (!slow) {
        ValueRows<BITS, HD> rows(a, kh, lane);
        const int vd = HD == 32 ? lane & 31 : lane, vp = rows.vp;
        for (int r = w / wr; r < nrow; r += RT_NW / wr) {
            const uint64_t sum = total(r), den = sum ? sum : 1;   // (0: sees nothing)
            const double y48 = quotient_factor(den);
            int64_t *row = sc + r * stride;
#pragma unroll 2
            for (int j = lane + 64 * sub; j < fill; j += 64 * wr)
                row[j] = __builtin_bit_cast(int64_t,
                                            quotient_scaled((uint64_t)row[j], den, y48));
        }
        __syncthreads();
        double acc[HD == 128 ? 2 : 1][16];
#pragma unroll
        for (int l = 0; l < (HD == 128 ? 2 : 1); ++l)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                acc[l][r] = Q48_FSUM0;
        // the next rows' values on their way under the sums, where the registers allow
        constexpr bool AHEAD = BITS != 64 && RT_NT == 512;
        if (AHEAD && CP * w < S)
            rows.fetch(a, kh, CP * w, S - 1, rl);
        for (int j0 = CP * w; j0 < S; j0 += RT_NW * CP) {
            double v[HD == 128 ? 2 : 1][16];
            if (!AHEAD)
                rows.fetch(a, kh, j0, S - 1, rl);
            rows.take(v, j0, S - 1, rl, big, DEC && BITS != 64 ? nk[1] : nullptr,
                      DEC && BITS != 64 ? nst[1] : 0);
            if (AHEAD && j0 + RT_NW * CP < S)
                rows.fetch(a, kh, j0 + RT_NW * CP, S - 1, rl);
            add_values<HD>(acc, v, nrow, [&](int r) {
                if (r >= nrow)
                    return 0.0;
                return __builtin_bit_cast(double, sc[r * stride + j0 + vp + rl]);
            });
        }
#pragma unroll
        for (int r = 0; r < 16; ++r)
            if (r < nrow)
#pragma unroll
                for (int l = 0; l < (HD == 128 ? 2 : 1); ++l)
                    atomicAdd(reinterpret_cast<unsigned long long *>(&lam[r][vd + 64 * l]),
                              (unsigned long long)q48_fsum_total(acc[l][r]));
    }
    const bool redo = __syncthreads_or(q48_f51_big(big)) || slow;
    for (int i = tid; i < nrow * HD; i += RT_NT) {
        const int r = i / HD, d = i % HD;
        out_at<HD>(a, p, v0 + r, G, kh)[d] =
            redo ? plain_sum<BITS, HD>(a, sc + r * stride, (int64_t)total(r), !slow, kh, d, 0, S,
                                        DEC ? nk[1] : nullptr, nst + 1)
                 : (int64_t)lam[r][d];
    }
}

// ---- three launches ---------------------------------------------------------------------

// The scores of TB tiles of 16 vectors over one chunk, and each vector's maximum
// over the rows it sees: a row's operand is made once for all TB tiles.  DEC: the
// store of the new row too (by the blocks that own it).
// int64 keys: 63 products of 16 cycles for 16 x 16 pairs of 64 dims, and about 200 vector
// operations to add them up, of two waves a SIMD: 1.5 us a tile for both, 1.0 of it the
// matrix cores alone.  48 tokens at 4000 (32 heads on 4 of 64; 6.2 M pairs) 41 us, 15 of 8
// bits (26 at 2047, 1.7 M pairs; 8 products).
template <int BITS, int HD, int TB, bool DEC>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void
k_ra_score(RaArgs a, RaPlan p)
{
    q48_round_down();
    constexpr int KS = HD < 64 ? 1 : HD / 64;
    __shared__ v4i dig[TB][KS][8][64];
    __shared__ q48_u128 cq[TB][16 * KS];
    __shared__ int vt[TB * 16];
    __shared__ int64_t mxs[4][TB * 16];
    __shared__ int farw[TB];
    __shared__ __align__(16) uint8_t nk[2][HD];
    __shared__ int64_t nst[2];
    __shared__ int64_t qs[DEC ? 16 * HD : 1];

    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rl = lane & 15, kq = lane >> 4;
    const int kh = blockIdx.z, G = a.n_heads / a.n_kv, NV = p.Tn * G;
    const int tile0 = blockIdx.y * TB, ntile = min(TB, p.tiles - tile0);
    int p0;
    if (!position<DEC>(a, p0))
        return;
    const int begin = (int)blockIdx.x * p.ch1;
    const int end =
        min(begin + p.ch1, tile_span<DEC>(a, p, 16 * (tile0 + ntile) - 1, G, p0));
    if (begin >= end)
        return;

    std::conditional_t<BITS == 64, WordRow<HD>, KeyRow<BITS == 64 ? 8 : BITS, HD>> next;
    if (keys_ahead(BITS, HD, TB) && begin + 16 * w < end)
        next.load(a, (size_t)min(begin + 16 * w + rl, end - 1) * a.n_kv + kh, kq);
    if (tid < TB * 16)
        vt[tid] = p.t0 + min(16 * tile0 + tid, NV - 1) / G;
    if (tid < TB)
        farw[tid] = 0;
    if constexpr (DEC) {
        decode_queries<HD, 256>(a, qs, 16 * tile0, min(16, NV - 16 * tile0), G, kh, p0, tid);
        if (p0 >= begin && p0 < end && tid >= 192 && tid < 224)
            new_row<BITS, HD>(a, p0, kh, tid - 192, nk, nst, blockIdx.y == 0);
        __syncthreads();
    }
    // a.out of these tiles' vectors, for the sums that the chunks add
    if (p.n3 > 1 && blockIdx.x == 0)
        for (int i = tid; i < ntile * 16 * HD; i += 256) {
            const int v = 16 * tile0 + i / HD;
            if (v < NV)
                out_at<HD>(a, p, v, G, kh)[i % HD] = 0;
        }
    for (int tb = 0; tb < ntile; ++tb)
        query_digits<BITS, HD, 256>(a, p, dig[tb], cq[tb], 16 * (tile0 + tb), NV - 1, G, kh,
                                    DEC ? qs : nullptr, (tid + 256 - 64 * (tb & 3)) & 255);
    __syncthreads();

    int64_t mx[TB][4];
    uint32_t far[TB];
#pragma unroll
    for (int tb = 0; tb < TB; ++tb) {
        far[tb] = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            mx[tb][i] = INT64_MIN;
    }
    int64_t *sc = p.sc + ((size_t)kh * p.tiles + tile0) * p.tv * p.spad;
    score_rows<BITS, HD, TB, 4, DEC>(a, dig, cq, vt, ntile, min(16, NV - 16 * tile0), kh, p0,
                                     begin, end, nk[0], DEC && BITS != 64 ? nst[0] : 0,
                                     rows_clear<DEC>(a, p0, p.t0 + 16 * tile0 / G), w, lane, mx,
                                     far, next, [&](int tb, int m, int j, int64_t s) {
                                         if (m < NV - 16 * tile0)   // (tv rows)
                                             sc[(size_t)(16 * tb + m) * p.spad + j] = s;
                                     });
#pragma unroll
    for (int tb = 0; tb < TB; ++tb) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t m = row16_max64(mx[tb][i]);
            if (rl == 0)
                mxs[w][tb * 16 + 4 * kq + i] = m;
        }
        if (far[tb] & 0x80000000u)
            atomicOr(&farw[tb], 1);
    }
    __syncthreads();
    if (tid < ntile * p.tv) {   // (tv < 16: one tile)
        int64_t m = mxs[0][tid];
#pragma unroll
        for (int u = 1; u < 4; ++u)
            m = mxs[u][tid] > m ? mxs[u][tid] : m;
        p.cm[(((size_t)kh * p.tiles + tile0) * p.tv + tid) * p.n1 + blockIdx.x] = m;
    }
    if (tid < ntile)
        p.far[((size_t)kh * p.tiles + tile0 + tid) * p.n1 + blockIdx.x] = farw[tid];
}

// Exponentials in place of a chunk's scores (0 for rows a vector does not see,
// up to the next multiple of 32 rows) and their sums: 80 vector operations each, 24 of
// them the squarings.  6.2 M in 25 us, 75% of what issue allows; 1.7 M in 13, most of it
// the launch, the chunk maxima and the scores on their way from other dies' caches.
template <bool DEC>
__global__ __launch_bounds__(256) void k_ra_exp(RaArgs a, RaPlan p)
{
    q48_round_down();
    __shared__ int odds;
    const int tid = threadIdx.x, kh = blockIdx.z, tile = blockIdx.y;
    const int G = a.n_heads / a.n_kv, NV = p.Tn * G, nrow = min(16, NV - 16 * tile);
    int p0;
    if (!position<DEC>(a, p0))
        return;
    const int span = tile_span<DEC>(a, p, 16 * tile + 15, G, p0);
    const int begin = (int)blockIdx.x * p.ch2, end = min(begin + p.ch2, span);
    if (begin >= end)
        return;
    if (tid == 0)
        odds = 0;
    const int chunks = (span + p.ch1 - 1) / p.ch1;
    // lanes of a vector: 16, or 32 or 64 where the tile has few vectors
    const int lg = nrow > 8 ? 4 : nrow > 4 ? 5 : 6, L = 1 << lg;
    const int r = tid >> lg, l = tid & (L - 1);
    const size_t vec = ((size_t)kh * p.tiles + tile) * p.tv + min(r, nrow - 1);
    const int *farp = p.far + ((size_t)kh * p.tiles + tile) * p.n1;
    const int64_t *cm = p.cm + vec * p.n1;
    int64_t *sc = p.sc + vec * p.spad;
    // the lane's first scores on their way while the maximum is found
    int64_t ahead[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        ahead[i] = sc[min(begin + l + i * L, end - 1)];
    int far = 0;
    int64_t m = INT64_MIN;
    for (int c = l; c < chunks; c += L) {
        far |= farp[c];
        m = cm[c] > m ? cm[c] : m;
    }
    far = __any(far);
    m = row16_max64(m);
    for (int o = 16; o < L; o <<= 1) {
        const int64_t x = __shfl_xor(m, o);
        m = x > m ? x : m;
    }
    __syncthreads();   // odds
    if (r < nrow) {
        const int t = p.t0 + (16 * tile + r) / G;
        const int fill = min(begin + p.ch2, (end + 31) & ~31);
        const int clear = far ? begin : min(end, rows_clear<DEC>(a, p0, t));
        int odd = 0;
        uint64_t sum = 0;
        int from = begin;
        if (begin + 4 * L <= clear) {
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                const uint64_t e0 = exp_neg((uint64_t)m - (uint64_t)ahead[i]);
                const uint64_t e1 = exp_neg((uint64_t)m - (uint64_t)ahead[i + 1]);
                sc[begin + l + i * L] = (int64_t)e0;
                sc[begin + l + (i + 1) * L] = (int64_t)e1;
                sum += e0 + e1;
            }
            from = begin + 4 * L;
        }
        sum += exp_rows<DEC>(a, p0, t, sc, m, far, from, end, fill, l, L, odd);
        sum = group_sum64<16>(sum);
        for (int o = 16; o < L; o <<= 1)
            sum += __shfl_xor(sum, o);
        if (l == 0)
            p.cs[vec * p.n2 + blockIdx.x] = sum;
        if (odd)
            atomicOr(&odds, 1);
    }
    __syncthreads();
    if (tid == 0)
        p.odd[((size_t)kh * p.tiles + tile) * p.n2 + blockIdx.x] = odds;
}

// The values of a chunk under its weights, added to out.  Wave w takes the
// 16-row groups w, w + 4, ... by itself (head_dim 32: 32 rows, 16 for each half of
// the wave): the quotients of its vectors (four a lane) go through LDS so that
// lane l of every row of 16 lanes holds row l % 16's weights.  A chunk with a value
// outside [-2^51, 2^51), or weights that are no plain softmax, multiplies in
// integers.
// Bound by FP64 issue: 16 rows of 16 vectors of 64 dims are 256 sums, 80 operations of
// quotients and 70 of conversions, 1.9 us for two waves a SIMD and no less.  48 tokens at
// 4000 over int64 rows 38 us, 25 of it this loop; 26 at 2047 of 8 bits 16 (7 the loop).
// A chunk that multiplies in integers is one thread an output and makes a quotient a term:
// with a value of 9.0 in each head whole calls take 1428 us (92 without) and 444 (43).
template <int BITS, int HD, bool DEC>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(HD == 128 ? 1 : 2))) void
k_ra_value(RaArgs a, RaPlan p)
{
    q48_round_down();
    constexpr int DL = HD == 128 ? 2 : 1, PG = HD == 32 ? 2 : 1, CP = 16 * PG;
    __shared__ double pw[4][16][CP];
    __shared__ uint64_t lam[16][HD];
    __shared__ uint64_t dens[16];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rl = lane & 15, g = lane >> 4;
    const int kh = blockIdx.z, tile = blockIdx.y;
    const int G = a.n_heads / a.n_kv, NV = p.Tn * G, nrow = min(16, NV - 16 * tile);
    int p0;
    if (!position<DEC>(a, p0))
        return;
    const int span = tile_span<DEC>(a, p, 16 * tile + 15, G, p0);
    const int begin = (int)blockIdx.x * p.ch3, end = min(begin + p.ch3, span);
    if (begin >= end)
        return;
    const int chunks = (span + p.ch2 - 1) / p.ch2;
    const size_t vec0 = ((size_t)kh * p.tiles + tile) * p.tv;
    const int64_t *sc = p.sc + vec0 * p.spad;
    // the wave's first exponentials and values on their way while the sums are joined
    ValueRows<BITS, HD> rows(a, kh, lane);
    uint64_t er[4 * PG];
    auto load_e = [&](int j0) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (4 * i < nrow)
#pragma unroll
                for (int u = 0; u < PG; ++u)
                    er[PG * i + u] =
                        (uint64_t)sc[(size_t)min(4 * i + g, nrow - 1) * p.spad + j0 + 16 * u + rl];
    };
    constexpr bool AHEAD = BITS != 64;   // (registers)
    if (begin + CP * w < end) {
        load_e(begin + CP * w);
        if (AHEAD)
            rows.fetch(a, kh, begin + CP * w, end - 1, rl);
    }
    {
        const int r = tid >> 4, l = tid & 15;
        uint64_t s = 0;
        if (r < nrow)
            for (int c = l; c < chunks; c += 16)
                s += p.cs[(vec0 + r) * p.n2 + c];
        s = group_sum64<16>(s);
        if (l == 0)
            dens[r] = s;
    }
    for (int i = tid; i < 16 * HD; i += 256)
        (&lam[0][0])[i] = 0;
    int slow = 0;
    for (int c = tid; c < chunks; c += 256)
        slow |= p.odd[((size_t)kh * p.tiles + tile) * p.n2 + c];
    if constexpr (BITS != 64)
        for (int j = begin + tid; j < end; j += 256)
            slow |= !step_fits<BITS>(a.vs[(size_t)j * a.n_kv + kh]) &&
                    seen<DEC>(a, p0, p.t0 + 16 * tile / G, p.t0 + (16 * tile + nrow - 1) / G, j);
    slow = __syncthreads_or(slow);   // dens and lam too
    uint32_t big = 0;
    if (!slow) {
        double y48[4];
        uint64_t den[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            den[i] = dens[4 * i + g];
            den[i] = den[i] ? den[i] : 1;   // (0: sees nothing)
            y48[i] = quotient_factor(den[i]);
        }
        const int vd = HD == 32 ? lane & 31 : lane, vp = rows.vp;
        double acc[DL][16];
#pragma unroll
        for (int l = 0; l < DL; ++l)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                acc[l][r] = Q48_FSUM0;
        for (int j0 = begin + CP * w; j0 < end; j0 += 4 * CP) {
            double v[DL][16];
            if (!AHEAD)
                rows.fetch(a, kh, j0, end - 1, rl);
            rows.take(v, j0, end - 1, rl, big);
            if (AHEAD && j0 + 4 * CP < end)
                rows.fetch(a, kh, j0 + 4 * CP, end - 1, rl);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (4 * i < nrow)
#pragma unroll
                    for (int u = 0; u < PG; ++u) {
                        const int r = 4 * i + g;
                        const double x = quotient_scaled(er[PG * i + u], den[i], y48[i]);
                        pw[w][r][16 * u + rl] = r < nrow ? x : 0.0;
                    }
            if (j0 + 4 * CP < end)
                load_e(j0 + 4 * CP);
            // the wave's own LDS writes before its reads
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            add_values<HD>(acc, v, nrow, [&](int r) { return pw[w][r][vp + rl]; });
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }
#pragma unroll
        for (int r = 0; r < 16; ++r)
            if (r < nrow)
#pragma unroll
                for (int l = 0; l < DL; ++l)
                    atomicAdd(reinterpret_cast<unsigned long long *>(&lam[r][vd + 64 * l]),
                              (unsigned long long)q48_fsum_total(acc[l][r]));
    }
    const bool redo = __syncthreads_or(q48_f51_big(big)) || slow;
    for (int i = tid; i < nrow * HD; i += 256) {
        const int r = i / HD, d = i % HD;
        const uint64_t o = redo ? (uint64_t)plain_sum<BITS, HD>(a, sc + (size_t)r * p.spad,
                                                               (int64_t)dens[r], false, kh, d,
                                                               begin, end)
                                : lam[r][d];
        int64_t *out = out_at<HD>(a, p, 16 * tile + r, G, kh) + d;
        if (p.n3 > 1)
            atomicAdd(reinterpret_cast<unsigned long long *>(out), (unsigned long long)o);
        else
            *out = (int64_t)o;
    }
}

// floor(2^48 / sqrt(hd)), fp_inv_sqrt(fp_from_int(hd)) (fp_math.h:658-707) for
// head_dim 32, 64 and 128
int64_t score_scale(int hd)
{
    return hd == 32 ? 49758216191607LL : hd == 64 ? (int64_t)1 << 45 : 24879108095803LL;
}

// rows of queries, and whether out shares words with them
bool overlap(const int64_t *a, size_t na, const int64_t *b, size_t nb)
{
    return (uintptr_t)a < (uintptr_t)(b + nb) && (uintptr_t)b < (uintptr_t)(a + na);
}

// Estimated times of the two forms, in us, for rows that see `most` rows at most and
// `seen` on average:
//   one launch     o + (c0 + c1 vb) most, where every block has a compute unit of its own;
//                  k (a second block's waves fill gaps) a further round, and `seen`
//   three launches l + c3 vectors seen
// with the constants fitted to both forms' times from 150 to 2756 rows and 1 to 1000
// tokens of 8 heads on 2 of 32, 32 on 4 of 64, 32 on 8 of 128: the slower one is chosen by
// 0.7% on average.  us, one / three, 32 heads on 4 of 64, 8 bits: one token at 300 rows
// 10.1 / 14.9, at 1000 17.4 / 14.7; 16 tokens at 1000 20.8 / 23.2; 64 at 2000 54.5 / 63.5;
// 512 at 1500 372 / 320, 256 at 2500 404 / 214.  int64: 4 tokens at 300 16.4 / 20.5, 16 at
// 1000 38.8 / 28.9, 512 at 1500 556 / 387.
template <int BITS, int HD>
bool one_launch(int vb, int most, double seen, long vectors, long blocks, int cus)
{
    constexpr int h = HD == 32 ? 0 : HD == 64 ? 1 : 2, w = BITS == 64;
    constexpr double o[2] = {10.8, 14.2}, k[2] = {1.27, 1.31}, l[2] = {16.3, 19.7};
    constexpr double c0[2][3] = {{3.0e-3, 4.9e-3, 8.3e-3}, {9.9e-3, 11.9e-3, 27.9e-3}};
    constexpr double c1[2][3] = {{2.27e-3, 2.10e-3, 3.81e-3}, {2.47e-3, 2.78e-3, 4.01e-3}};
    constexpr double c3[2][3] = {{11.4e-6, 11.6e-6, 18.8e-6}, {15.7e-6, 16.1e-6, 31.5e-6}};
    const double rounds = (double)blocks / cus;
    const double rows = rounds <= 1 ? (double)most : seen * (1 + k[w] * (rounds - 1));
    return o[w] + rows * (c0[w][h] + c1[w][h] * vb) <= l[w] + (double)vectors * seen * c3[w][h];
}

// Rows of one launch: their scores, in whole tiles of every KV head, take at most this
// much workspace.  (A single row's 1024 vectors of 32767 scores always fit.)
constexpr size_t RA_WS_MAX = (size_t)1 << 30;

template <int BITS, int HD, bool DEC>
int launch_hd(q48_ctx *c, RaArgs &a)
{
    const int G = a.n_heads / a.n_kv;
    // positions a launch may reach: the cache's, where the device holds the position
    const int S = DEC ? (a.d_pos ? a.max_seq : a.p0 + 1) : a.p0 + a.T;
    RaPlan p = {};
    p.spad = (S + 63) & ~63;
    {
        // Tiles of the most vectors (a power of two) that still leave about a block a
        // compute unit, and whose scores fit LDS.  Of the tiles of 16 vectors, those of
        // 64-wide heads over codes take 16 waves (they keep their 128 registers each)
        // where a block is alone on its compute unit: there are as many blocks as units,
        // or two of 8 waves do not fit LDS.  us, 16 / 8 waves, 32 heads on 4, 8 bits: 128
        // rows (256 blocks) at 0 12.9 / 13.4, at 300 20.9 / 23.1, at 600 30.3 / 34.3; 256
        // at 200 41.8 / 46.9, 384 at 512 87.3 / 100.8 (4 bits 89.4 / 103.3); two blocks of
        // 8 waves a unit: 256 at 0 29.0 / 25.3, 256 at 192 37.9 / 33.8.  Tiles of fewer
        // vectors have 8 waves.
        int vb = 16;
        while (vb > 1 && ((a.T * G + vb - 1) / vb) * a.n_kv < c->cu_count)
            vb >>= 1;
        while (vb > 1 && (size_t)vb * (p.spad + 4) * 8 > rt_lds(HD, 16))
            vb >>= 1;
        const long tiles = (a.T * G + vb - 1) / vb;
        const size_t lds = (size_t)vb * (p.spad + 4) * 8;
        // (in step mode the position given says what to expect)
        const int most = a.p0 + a.T;
        const double seen = DEC || a.mask ? most : most - 0.5 * a.T;
        if (lds <= rt_lds(HD, 16) &&
            one_launch<BITS, HD>(vb, most, seen, (long)a.T * a.n_heads, tiles * a.n_kv,
                                 c->cu_count)) {
            constexpr bool WIDE = HD == 64 && BITS != 64 && !DEC;   // (decode: spills)
            p.Tn = a.T;
            p.vb = vb;
            const dim3 grid(tiles, a.n_kv);
            const bool alone = tiles * a.n_kv <= c->cu_count ||
                               2 * (lds + rt_static(HD, 8)) > 160 * 1024;
            if (WIDE && vb == 16 && alone)
                hipLaunchKernelGGL((k_ra_tile<BITS, HD, DEC, WIDE ? 1024 : 512>), grid, dim3(1024),
                                   lds, c->stream, a, p);
            else
                hipLaunchKernelGGL((k_ra_tile<BITS, HD, DEC, 512>), grid, dim3(512), lds,
                                   c->stream, a, p);
            return hipGetLastError() == hipSuccess ? Q48_OK : Q48_EHIP;
        }
    }
    long fit = (long)(RA_WS_MAX / ((size_t)a.n_kv * p.spad * 8));   // vectors a KV head
    if (fit > 16)
        fit &= ~15L;
    long Tn = fit / G;
    Tn = Tn < 1 ? 1 : Tn < a.T ? Tn : a.T;
    p.tiles = (int)((Tn * G + 15) / 16);
    p.tv = Tn * G < 16 ? (int)(Tn * G) : 16;
    const long tiles = (long)p.tiles * a.n_kv;
    constexpr int TB = DEC ? 1 : BITS == 64 && HD < 128 ? 4 : 2;
    // Chunks for about `want` blocks, of 64 rows at least, 128 past 4096: a later launch's
    // blocks read every chunk's maximum or sum, and the values' sums of all chunks meet in
    // atomics.  `want` is about what the compute units hold at once (8 exponential blocks
    // each, 4 score blocks, 2 of int64 keys; 2 value blocks, 1 of 128-wide int64 heads): a
    // few blocks more are a round more.  us with 512 / 1024 score blocks: 16 tokens at 3000
    // (8 bits) 40.7 / 37.5, 512 at 1500 319 / 305; int64 48 at 4000 96.7 / 99.9, 200 at 2000
    // 187 / 197.  1024 / 2048 exponential blocks: 48 at 4000 104 / 100, 512 at 1500 334 /
    // 319.  256 / 512 / 1024 value blocks: 26 at 2047 (8 bits) 46.8 / 43.1 / 48.8, 48 at
    // 4000 119 / 100 / 107, 16 at 2000 of 128-wide int64 heads 42.9 / 49.2 / 66.6.  One token
    // at 16000 with chunks of 128 / 64 rows 27 / 30 (any of the three).
    auto chunk = [&](long blocks, long want, int &ch, int &n) {
        long k = want / blocks, most = p.spad / (S > 4096 ? 128 : 64);
        k = k < most ? k : most;
        k = k < 1 ? 1 : k;
        ch = (int)(((S + k - 1) / k + 63) & ~63);
        n = (S + ch - 1) / ch;
    };
    chunk((tiles + TB - 1) / TB, BITS == 64 ? 512 : 1024, p.ch1, p.n1);
    chunk(tiles, 2048, p.ch2, p.n2);
    chunk(tiles, BITS == 64 && HD == 128 ? 256 : 512, p.ch3, p.n3);
    size_t o = 0;
    auto take = [&](size_t bytes) {
        const size_t at = o;
        o += (bytes + 255) & ~(size_t)255;
        return at;
    };
    const size_t vecs = (size_t)a.n_kv * p.tiles * p.tv;
    const size_t o_sc = take(vecs * p.spad * 8), o_cm = take(vecs * p.n1 * 8);
    const size_t o_cs = take(vecs * p.n2 * 8);
    const size_t o_far = take(tiles * p.n1 * 4), o_odd = take(tiles * p.n2 * 4);
    int rc = q48_ws_reserve(c, o);
    if (rc)
        return rc;
    uint8_t *ws = (uint8_t *)c->ws;
    p.sc = (int64_t *)(ws + o_sc);
    p.cm = (int64_t *)(ws + o_cm);
    p.cs = (uint64_t *)(ws + o_cs);
    p.far = (int *)(ws + o_far);
    p.odd = (int *)(ws + o_odd);
    for (p.t0 = 0; p.t0 < a.T; p.t0 += Tn) {
        p.Tn = Tn < a.T - p.t0 ? (int)Tn : a.T - p.t0;
        const int nt = (p.Tn * G + 15) / 16;
        hipLaunchKernelGGL((k_ra_score<BITS, HD, TB, DEC>),
                           dim3(p.n1, (nt + TB - 1) / TB, a.n_kv), dim3(256), 0, c->stream, a, p);
        hipLaunchKernelGGL((k_ra_exp<DEC>), dim3(p.n2, nt, a.n_kv), dim3(256), 0, c->stream, a, p);
        hipLaunchKernelGGL((k_ra_value<BITS, HD, DEC>), dim3(p.n3, nt, a.n_kv), dim3(256), 0,
                           c->stream, a, p);
    }
    return hipGetLastError() == hipSuccess ? Q48_OK : Q48_EHIP;
}

template <int BITS, bool DEC>
int launch(q48_ctx *c, RaArgs &a, int hd)
{
    a.scale = score_scale(hd);
    return hd == 32   ? launch_hd<BITS, 32, DEC>(c, a)
           : hd == 64 ? launch_hd<BITS, 64, DEC>(c, a)
                      : launch_hd<BITS, 128, DEC>(c, a);
}

int decode_qcache(q48_ctx *c, int64_t *out, const int64_t *q, const q48_qcache *qc,
                  const int64_t *k_new, const int64_t *v_new, int layer, int pos, int n_heads,
                  bool rope)
{
    if (!c || !out || !q || !k_new || !v_new || q48_off_words<8>(out, q, k_new, v_new) ||
        !q48_qcache_ok(qc) || layer < 0 ||
        layer >= qc->layers || n_heads <= 0 || n_heads > RA_MAX_HEADS || n_heads % qc->n_kv)
        return Q48_EINVAL;
    const size_t hd = qc->head_dim, qn = n_heads * hd, kn = qc->n_kv * hd;
    if (overlap(out, qn, q, qn) || overlap(out, qn, k_new, kn) || overlap(out, qn, v_new, kn))
        return Q48_EINVAL;
    if (rope && (!c->rope_cos || qc->head_dim != c->rope_head_dim || qc->max_seq > c->rope_max_seq))
        return Q48_ESTATE;
    if (pos < 0 || pos >= qc->max_seq)
        return Q48_ERANGE;
    q48_on_device on(c);
    const size_t rows = (size_t)layer * qc->max_seq * qc->n_kv;
    RaArgs a = {};
    a.out = out;
    a.q = q;
    a.k = (const uint8_t *)qc->k + rows * (hd * qc->bits / 8);
    a.v = (const uint8_t *)qc->v + rows * (hd * qc->bits / 8);
    a.ks = qc->k_step + rows;
    a.vs = qc->v_step + rows;
    a.d_pos = c->step_mode ? c->d_step + 1 : nullptr;
    a.p0 = pos;
    a.T = 1;
    a.n_heads = n_heads;
    a.n_kv = qc->n_kv;
    a.max_seq = qc->max_seq;
    a.k_new = k_new;
    a.v_new = v_new;
    a.cos_t = rope ? c->rope_cos : nullptr;
    a.sin_t = rope ? c->rope_sin : nullptr;
    return qc->bits == 8 ? launch<8, true>(c, a, qc->head_dim)
                         : launch<4, true>(c, a, qc->head_dim);
}

} // namespace

extern "C" {

int q48_attn_decode_qcache(q48_ctx *c, int64_t *out, const int64_t *q, const q48_qcache *qc,
                           const int64_t *k_new, const int64_t *v_new, int layer, int pos,
                           int n_heads)
{
    return decode_qcache(c, out, q, qc, k_new, v_new, layer, pos, n_heads, false);
}

int q48_attn_decode_rope_qcache(q48_ctx *c, int64_t *out, const int64_t *q, const q48_qcache *qc,
                                const int64_t *k_new, const int64_t *v_new, int layer, int pos,
                                int n_heads)
{
    return decode_qcache(c, out, q, qc, k_new, v_new, layer, pos, n_heads, true);
}

int q48_attn_rows_qcache(q48_ctx *c, int64_t *out, const int64_t *QKV, const q48_qcache *qc,
                         int layer, int p0, int T, int n_heads, const uint64_t *mask)
{
    if (!c || !out || !QKV || q48_off_words<8>(out, QKV, mask) || !q48_qcache_ok(qc) ||
        layer < 0 || layer >= qc->layers || T <= 0 ||
        n_heads <= 0 || n_heads > RA_MAX_HEADS || n_heads % qc->n_kv)
        return Q48_EINVAL;
    if (p0 < 0 || p0 >= qc->max_seq || T > qc->max_seq - p0)
        return Q48_ERANGE;
    const size_t hd = qc->head_dim, row = (size_t)(n_heads + 2 * qc->n_kv) * hd;
    if (overlap(out, T * n_heads * hd, QKV, T * row))
        return Q48_EINVAL;
    q48_on_device on(c);
    const size_t rows = (size_t)layer * qc->max_seq * qc->n_kv;
    RaArgs a = {};
    a.out = out;
    a.q = QKV;
    a.ldq = row;
    a.k = (const uint8_t *)qc->k + rows * (hd * qc->bits / 8);
    a.v = (const uint8_t *)qc->v + rows * (hd * qc->bits / 8);
    a.ks = qc->k_step + rows;
    a.vs = qc->v_step + rows;
    a.mask = mask;
    a.words = (T + 63) / 64;
    a.p0 = p0;
    a.T = T;
    a.n_heads = n_heads;
    a.n_kv = qc->n_kv;
    a.max_seq = qc->max_seq;
    return qc->bits == 8 ? launch<8, false>(c, a, qc->head_dim)
                         : launch<4, false>(c, a, qc->head_dim);
}

int q48_attn_tree(q48_ctx *c, int64_t *out, const int64_t *QKV, const int64_t *kcache,
                  const int64_t *vcache, int layer, int p0, int T, int n_heads, int n_kv,
                  int head_dim, int max_seq, const uint64_t *mask)
{
    if (!c || !out || !QKV || !kcache || !vcache ||
        q48_off_words<8>(out, QKV, kcache, vcache, mask) || layer < 0 || T <= 0 || n_heads <= 0 ||
        n_heads > RA_MAX_HEADS || n_kv <= 0 || n_heads % n_kv || max_seq <= 0 ||
        (head_dim != 32 && head_dim != 64 && head_dim != 128))
        return Q48_EINVAL;
    if (p0 < 0 || p0 >= max_seq || T > max_seq - p0 || p0 + T > RA_MAX_POS)
        return Q48_ERANGE;
    const size_t hd = head_dim, row = (size_t)(n_heads + 2 * n_kv) * hd;
    if (overlap(out, T * n_heads * hd, QKV, T * row))
        return Q48_EINVAL;
    q48_on_device on(c);
    const size_t at = (size_t)layer * max_seq * n_kv * hd;
    RaArgs a = {};
    a.out = out;
    a.q = QKV;
    a.ldq = row;
    a.k = (const uint8_t *)(kcache + at);
    a.v = (const uint8_t *)(vcache + at);
    a.mask = mask;
    a.words = (T + 63) / 64;
    a.p0 = p0;
    a.T = T;
    a.n_heads = n_heads;
    a.n_kv = n_kv;
    a.max_seq = max_seq;
    return launch<64, false>(c, a, head_dim);
}

} // extern "C"
