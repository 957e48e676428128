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
// head kh G + g), taken in tiles of 16 (one MFMA tile of rows); the cache rows in
// chunks of ch.  Three kernels, each a grid of (chunk, tile, KV head) blocks: the
// softmax of the exact path needs the row's maximum before the first exponential
// and the whole sum before the first quotient, and its truncations leave no way
// to rescale later, so each of the two is a launch boundary.
struct RaPlan {
    int64_t *sc;     // [n_kv][16 tiles][spad]: scores, then exponentials
    int64_t *cm;     // [n_kv][16 tiles][nchunk]: a chunk's maximum
    uint64_t *cs;    // [n_kv][16 tiles][nchunk]: a chunk's sum of exponentials
    int *far;        // [n_kv][tiles][nchunk]: a visible score outside [-2^62, 2^62)
    int *odd;        // [n_kv][tiles][nchunk]: an exponential outside [0, ONE]
    int ch, nchunk, spad, tiles, t0, Tn;   // rows t0 .. t0 + Tn - 1 of the T
};

// rows [0, span) hold all that a tile's vectors may see
template <bool DEC>
__device__ __forceinline__ int tile_span(const RaArgs &a, const RaPlan &p, int tile, int G, int p0)
{
    if (DEC)
        return p0 + 1;
    if (a.mask)
        return p0 + a.T;
    const int last = (16 * tile + 15) / G;
    return p0 + p.t0 + (last < p.Tn ? last + 1 : p.Tn);
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

// 16 codes as int8 MFMA operands: dims d0 .. d0 + 15 of a head's row
template <int BITS, int HD>
__device__ __forceinline__ v4i codes16(const uint8_t *row, int d0)
{
    if constexpr (BITS == 8) {
        return *reinterpret_cast<const v4i *>(row + d0);
    } else {
        v4i w = *reinterpret_cast<const v4i *>(row + (d0 & (HD / 2 - 1)));
        const int sh = d0 < HD / 2 ? 0 : 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // a nibble n as a signed byte: (n ^ 8) - 8 without borrows
            const uint32_t n = ((uint32_t)w[i] >> sh) & 0x0F0F0F0Fu;
            w[i] = (int)(((n ^ 0x08080808u) + 0x78787878u) ^ 0x80808080u);
        }
        return w;
    }
}

// bits 48 .. 111 of step * sum_d q_d c_d from the digit sums: with q = sum_a s_a
// 256^a + C (q48_digits.hpp), sum_d q_d c_d = sum_a 256^a acc[a] + C cs, below 2^80
__device__ __forceinline__ int64_t code_dot(const v4i (&acc)[8], int i, int cs, uint64_t step)
{
    int64_t lo = (int64_t)(uint32_t)kDig * cs, hi = (int64_t)(kDig >> 32) * cs;
    lo = mad_shl<0>(acc[0][i], lo);
    lo = mad_shl<8>(acc[1][i], lo);
    lo = mad_shl<16>(acc[2][i], lo);
    lo = mad_shl<24>(acc[3][i], lo);
    hi = mad_shl<0>(acc[4][i], hi);
    hi = mad_shl<8>(acc[5][i], hi);
    hi = mad_shl<16>(acc[6][i], hi);
    hi = mad_shl<24>(acc[7][i], hi);
    hi += lo >> 32;
    const uint64_t nl = ((uint64_t)hi << 32) | (uint32_t)lo;
    const int64_t nh = hi >> 32;
    const uint64_t ph = __umul64hi(nl, step) + (uint64_t)nh * step;
    return (int64_t)((ph << 16) | ((nl * step) >> 48));
}

// The scores of TB tiles of vectors over one chunk, and each vector's maximum
// over the rows it sees.  Wave w takes the 16-row tiles w, w + 4, ...: its lane
// (j = lane % 16) holds row j's 16 dims of MFMA operand once for all TB tiles; a
// query's digits come from LDS.  DEC: RoPE of the queries and the new key, and
// the store of the new row (by the blocks that own it).
template <int BITS, int HD, int TB, bool DEC>
__global__ __launch_bounds__(256) void k_ra_score(RaArgs a, RaPlan p)
{
    q48_round_down();
    constexpr int KS = HD < 64 ? 1 : HD / 64;
    __shared__ v4i dig[TB][KS][8][64];
    __shared__ q48_u128 cq[TB * 16];
    __shared__ int vt[TB * 16];
    __shared__ int64_t mxs[4][TB * 16];
    __shared__ int farw[TB];
    __shared__ __align__(16) uint8_t nk[2][HD];
    __shared__ int64_t nst[2];
    __shared__ int64_t qs[DEC ? 16 : 1][DEC ? HD : 1];

    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int rl = lane & 15, kq = lane >> 4;
    const int kh = blockIdx.z, G = a.n_heads / a.n_kv, NV = p.Tn * G;
    const int tile0 = blockIdx.y * TB, ntile = min(TB, p.tiles - tile0);
    int p0;
    if (!position<DEC>(a, p0))
        return;
    const int begin = (int)blockIdx.x * p.ch;
    const int end = min(begin + p.ch, tile_span<DEC>(a, p, tile0 + ntile - 1, G, p0));
    if (begin >= end)
        return;

    if (tid < TB * 16)
        vt[tid] = p.t0 + min(16 * tile0 + tid, NV - 1) / G;
    if (tid < TB)
        farw[tid] = 0;
    if constexpr (DEC) {
        for (int it = tid; it < 16 * (HD / 2); it += 256) {
            const int v = min(16 * tile0 + it / (HD / 2), NV - 1), i = it % (HD / 2);
            const int64_t *q = a.q + (size_t)(kh * G + v) * HD;
            int64_t x0 = q[i], x1 = q[i + HD / 2];
            if (a.cos_t)
                q48_rope_pair(x0, x1, a.cos_t[(size_t)p0 * (HD / 2) + i],
                              a.sin_t[(size_t)p0 * (HD / 2) + i]);
            qs[it / (HD / 2)][i] = x0;
            qs[it / (HD / 2)][i + HD / 2] = x1;
        }
        if (p0 >= begin && p0 < end && tid < 32)
            new_row<BITS, HD>(a, p0, kh, tid, nk, nst, blockIdx.y == 0);
        __syncthreads();
    }
    // a.out of this tile's vectors, for the sums that the chunks add
    if (p.nchunk > 1 && blockIdx.x == 0)
        for (int i = tid; i < ntile * 16 * HD; i += 256) {
            const int v = 16 * tile0 + i / HD;
            if (v < NV)
                a.out[((size_t)(p.t0 + v / G) * a.n_heads + kh * G + v % G) * HD + i % HD] = 0;
        }
    for (int it = tid; it < ntile * KS * 64; it += 256) {
        const int tb = it / (KS * 64), ks = it / 64 % KS, l = it & 63;
        const int v = min(16 * (tile0 + tb) + (l & 15), NV - 1), d0 = 64 * ks + 16 * (l >> 4);
        uint64_t x[16];
        q48_u128 sum = 0;
        if (d0 < HD) {
            const int64_t *q;
            if constexpr (DEC)
                q = &qs[l & 15][d0];
            else
                q = a.q + (size_t)(p.t0 + v / G) * a.ldq + (size_t)(kh * G + v % G) * HD + d0;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                x[e] = (uint64_t)q[e];
                if (BITS == 64)
                    sum += (q48_u128)(q48_i128)q[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e)
                x[e] = kDig;   // digits of zero
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
            dig[tb][ks][d][l] = o[d];
        if constexpr (BITS == 64) {
            // the four lanes of a row are in one wave; with KS = 2 its halves are
            // in different waves, so the second adds what it reads back below
            sum += shfl_xor128(sum, 16);
            sum += shfl_xor128(sum, 32);
            if (l < 16 && ks == 0)
                cq[tb * 16 + l] = sum * kDig;
        }
    }
    __syncthreads();
    if constexpr (BITS == 64 && KS == 2) {
        if (tid < ntile * 16) {
            const int v = min(16 * tile0 + tid, NV - 1);
            const int64_t *q =
                a.q + (size_t)(p.t0 + v / G) * a.ldq + (size_t)(kh * G + v % G) * HD + 64;
            q48_u128 sum = 0;
            for (int e = 0; e < 64; ++e)
                sum += (q48_u128)(q48_i128)q[e];
            cq[tid] += sum * kDig;
        }
        __syncthreads();
    }

    const bool pow2 = HD == 64;   // the scale is 2^45: a shift
    int64_t mx[TB][4];
    uint32_t far[TB];
#pragma unroll
    for (int tb = 0; tb < TB; ++tb) {
        far[tb] = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            mx[tb][i] = INT64_MIN;
    }
    const v4i ones = {0x01010101, 0x01010101, 0x01010101, 0x01010101};
    for (int j0 = begin + 16 * w; j0 < end; j0 += 64) {
        const int j = j0 + rl, jc = min(j, end - 1);
        const size_t row = (size_t)jc * a.n_kv + kh;
        v4i B[KS][BITS == 64 ? 8 : 1];
        q48_u128 ck = 0;
        int cs = 0;
        uint64_t step = 0;
        if constexpr (BITS == 64) {
            const int64_t *k = reinterpret_cast<const int64_t *>(a.k) + row * HD;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const int d0 = 64 * ks + 16 * kq;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    uint64_t x4[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x4[e] = d0 < HD ? (uint64_t)k[d0 + 4 * g + e] : kDig;
                        if (d0 < HD)
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
            ck = ck * kDig - (q48_u128)kDig * kDig * (q48_u128)HD;
        } else {
            const bool fresh = DEC && jc == p0;
            const uint8_t *k = a.k + row * (HD * BITS / 8);
            v4i sum = {0, 0, 0, 0};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const int d0 = min(64 * ks + 16 * kq, HD - 16);   // zero digits past HD
                B[ks][0] = fresh ? codes16<BITS, HD>(nk[0], d0) : codes16<BITS, HD>(k, d0);
                v4i one = ones;
                if (64 * ks + 16 * kq >= HD)
                    one = (v4i){0, 0, 0, 0};
                sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(one, B[ks][0], sum, 0, 0, 0);
            }
            cs = sum[0];
            step = (uint64_t)(fresh ? nst[0] : a.ks[row]);
        }
#pragma unroll
        for (int tb = 0; tb < TB; ++tb) {
            if (tb >= ntile)
                break;
            int64_t *sc = p.sc + (((size_t)kh * p.tiles + tile0 + tb) * 16) * p.spad;
            int64_t s[4];
            if constexpr (BITS == 64) {
                v4i acc[14];
#pragma unroll
                for (int d = 0; d < 14; ++d)
                    acc[d] = (v4i){0, 0, 0, 0};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        const v4i A = dig[tb][ks][x][lane];
#pragma unroll
                        for (int y = 0; y < 8; ++y)
                            if (x + y <= 13)
                                acc[x + y] = __builtin_amdgcn_mfma_i32_16x16x64_i8(
                                    A, B[ks][y], acc[x + y], 0, 0, 0);
                    }
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    s[i] = digits_shr48(acc, i, cq[tb * 16 + 4 * kq + i] + ck);
            } else {
                v4i acc[8];
#pragma unroll
                for (int d = 0; d < 8; ++d)
                    acc[d] = (v4i){0, 0, 0, 0};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int d = 0; d < 8; ++d)
                        acc[d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(
                            dig[tb][ks][d][lane], B[ks][0], acc[d], 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    s[i] = code_dot(acc, i, cs, step);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int m = 4 * kq + i;
                s[i] = pow2 ? s[i] >> 3 : q48_mul(s[i], a.scale);
                if (j < end)
                    sc[(size_t)m * p.spad + j] = s[i];
                if (j < end && sees<DEC>(a, p0, vt[tb * 16 + m], j)) {
                    far[tb] |= (uint32_t)((uint64_t)s[i] >> 32) + 0x40000000u;
                    mx[tb][i] = s[i] > mx[tb][i] ? s[i] : mx[tb][i];
                }
            }
        }
    }
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
    if (tid < ntile * 16) {
        int64_t m = mxs[0][tid];
#pragma unroll
        for (int u = 1; u < 4; ++u)
            m = mxs[u][tid] > m ? mxs[u][tid] : m;
        p.cm[(((size_t)kh * p.tiles + tile0) * 16 + tid) * p.nchunk + blockIdx.x] = m;
    }
    if (tid < ntile)
        p.far[((size_t)kh * p.tiles + tile0 + tid) * p.nchunk + blockIdx.x] = farw[tid];
}

// Exponentials in place of a chunk's scores (0 for rows a vector does not see,
// up to the next multiple of 32 rows) and their sums.
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
    const int span = tile_span<DEC>(a, p, tile, G, p0);
    const int begin = (int)blockIdx.x * p.ch, end = min(begin + p.ch, span);
    if (begin >= end)
        return;
    if (tid == 0)
        odds = 0;
    __syncthreads();
    const int chunks = (span + p.ch - 1) / p.ch;
    // lanes of a vector: 16, or 32 or 64 where the tile has few vectors
    const int lg = nrow > 8 ? 4 : nrow > 4 ? 5 : 6, L = 1 << lg;
    const int r = tid >> lg, l = tid & (L - 1);
    const int *farp = p.far + ((size_t)kh * p.tiles + tile) * p.nchunk;
    int far = 0;
    for (int c = l; c < chunks; c += L)
        far |= farp[c];
    far = __any(far);
    if (r < nrow) {
        const size_t vec = ((size_t)kh * p.tiles + tile) * 16 + r;
        const int64_t *cm = p.cm + vec * p.nchunk;
        int64_t m = INT64_MIN;
        for (int c = l; c < chunks; c += L)
            m = cm[c] > m ? cm[c] : m;
        m = row16_max64(m);
        for (int o = 16; o < L; o <<= 1) {
            const int64_t x = __shfl_xor(m, o);
            m = x > m ? x : m;
        }
        const int t = p.t0 + (16 * tile + r) / G;
        int64_t *sc = p.sc + vec * p.spad;
        uint64_t sum = 0;
        int odd = 0;
        const int fill = min(begin + p.ch, (end + 31) & ~31);
        for (int j = begin + l; j < fill; j += L) {
            int64_t e = 0;
            if (j < end && sees<DEC>(a, p0, t, j)) {
                const int64_t s = sc[j];
                if (!far) {
                    e = q48_exp_neg((uint64_t)m - (uint64_t)s);
                } else {
                    e = q48_safe_exp((int64_t)((uint64_t)s - (uint64_t)m));
                    odd |= (uint64_t)e > (uint64_t)Q48_ONE;
                }
            }
            sc[j] = e;
            sum += (uint64_t)e;
        }
        sum = group_sum64<16>(sum);
        for (int o = 16; o < L; o <<= 1)
            sum += __shfl_xor(sum, o);
        if (l == 0)
            p.cs[vec * p.nchunk + blockIdx.x] = sum;
        if (odd)
            atomicOr(&odds, 1);
    }
    __syncthreads();
    if (tid == 0)
        p.odd[((size_t)kh * p.tiles + tile) * p.nchunk + blockIdx.x] = odds;
}

// 2^48 / d for the quotients of a softmax row (1 <= d < 2^63; 0 for d = 0): as
// q48_divisor_of, whose bound of 2^62 a row past 16384 positions may pass.  The
// quotient's bound is the same there: e / d shrinks as d grows.
__device__ __forceinline__ double quotient_factor(uint64_t d)
{
    const double dd = (double)d;
    double y = __builtin_amdgcn_rcp(dd);
    y = __builtin_fma(y, __builtin_fma(-dd, y, 1.0), y);
    y = __builtin_fma(y, __builtin_fma(-dd, y, 1.0), y);
    return d ? y * 0x1p48 : 0.0;
}

// fp_div(e, den) 2^-48 for 0 <= e <= ONE <= den, or 0 for e = den = 0
__device__ __forceinline__ double quotient_scaled(uint64_t e, uint64_t den, double y48)
{
    const double ed = __builtin_bit_cast(double, e | 0x4330000000000000ull) - 0x1p52;
    const uint64_t q0 = q48_word_m52(__builtin_fma(ed, y48, 0x1p52 - 0.5));
    const uint64_t rem = (e << 48) - q0 * den;
    return q48_pscaled((int64_t)(q0 + (rem >= den ? 1 : 0)));
}

// The values of a chunk under its weights, added to out.  Wave w takes the
// 16-row groups w, w + 4, ... by itself: the quotients of 16 vectors (four a lane)
// go through LDS so that lane l of every row of 16 lanes holds row l % 16's
// weights, and row_newbcast hands them to the lanes, which hold one dim each
// (head_dim 128: two; 32: two groups of rows) of the values as doubles: one FP64
// operation a (vector, row, dim), rounding down (q48_fsum4x4).  Tiles of fewer
// vectors skip the sums of four absent ones.  A chunk with a value outside
// [-2^51, 2^51), or weights that are no plain softmax, multiplies in integers.
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
    const int span = tile_span<DEC>(a, p, tile, G, p0);
    const int begin = (int)blockIdx.x * p.ch, end = min(begin + p.ch, span);
    if (begin >= end)
        return;
    const int chunks = (span + p.ch - 1) / p.ch;
    const size_t vec0 = ((size_t)kh * p.tiles + tile) * 16;
    const int64_t *sc = p.sc + vec0 * p.spad;
    {
        const int r = tid >> 4, l = tid & 15;
        uint64_t s = 0;
        if (r < nrow)
            for (int c = l; c < chunks; c += 16)
                s += p.cs[(vec0 + r) * p.nchunk + c];
        s = group_sum64<16>(s);
        if (l == 0)
            dens[r] = s;
    }
    for (int i = tid; i < 16 * HD; i += 256)
        (&lam[0][0])[i] = 0;
    int slow = 0;
    for (int c = tid; c < chunks; c += 256)
        slow |= p.odd[((size_t)kh * p.tiles + tile) * p.nchunk + c];
    if constexpr (BITS != 64) {
        constexpr uint64_t top = ((uint64_t)1 << 51) / (BITS == 8 ? 127 : 7);
        for (int j = begin + tid; j < end; j += 256)
            slow |= (uint64_t)a.vs[(size_t)j * a.n_kv + kh] >= top;
    }
    slow = __syncthreads_or(slow);   // dens and lam too
    uint32_t big = 0;
    if (!slow) {
        double y48[4];
        uint64_t den[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            den[i] = dens[4 * i + g];
            y48[i] = quotient_factor(den[i]);
        }
        const int vd = HD == 32 ? lane & 31 : lane;
        const int vp = HD == 32 ? 16 * (lane >> 5) : 0;
        double acc[DL][16];
#pragma unroll
        for (int l = 0; l < DL; ++l)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                acc[l][r] = Q48_FSUM0;
        uint64_t er[4 * PG];
        auto load_e = [&](int j0) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (4 * i < nrow)
#pragma unroll
                    for (int u = 0; u < PG; ++u)
                        er[PG * i + u] = (uint64_t)sc[(size_t)(4 * i + g) * p.spad + j0 + 16 * u + rl];
        };
        if (begin + CP * w < end)
            load_e(begin + CP * w);
        for (int j0 = begin + CP * w; j0 < end; j0 += 4 * CP) {
            double v[DL][16];
            if constexpr (BITS == 64) {
                const int64_t *vb = reinterpret_cast<const int64_t *>(a.v) + (size_t)kh * HD + vd;
#pragma unroll
                for (int n = 0; n < 16; ++n)
#pragma unroll
                    for (int l = 0; l < DL; ++l)
                        v[l][n] = q48_f51(
                            vb[(size_t)min(j0 + vp + n, end - 1) * a.n_kv * HD + 64 * l], big);
            } else {
                // a lane's own row's step, handed to the lanes of its row group
                const double st =
                    (double)a.vs[(size_t)min(j0 + vp + rl, end - 1) * a.n_kv + kh];
                const uint8_t *vb = a.v + (size_t)kh * (HD * BITS / 8);
#pragma unroll
                for (int n = 0; n < 16; ++n) {
                    const uint8_t *vr =
                        vb + (size_t)min(j0 + vp + n, end - 1) * a.n_kv * (HD * BITS / 8);
                    const double sn = __shfl(st, (lane & 48) | n);
#pragma unroll
                    for (int l = 0; l < DL; ++l)
                        v[l][n] = (double)code_at<BITS, HD>(vr, vd + 64 * l) * sn;
                }
            }
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
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                if (r >= nrow)
                    break;
                double q[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    q[i] = pw[w][r + i][vp + rl];
#pragma unroll
                for (int l = 0; l < DL; ++l) {
                    auto f4 = [&](auto base) {
                        constexpr int B = decltype(base)::value;
                        const double x[4] = {v[l][B], v[l][B + 1], v[l][B + 2], v[l][B + 3]};
                        q48_fsum4x4<B>(acc[l][r], acc[l][r + 1], acc[l][r + 2], acc[l][r + 3], q,
                                       x);
                    };
                    f4(std::integral_constant<int, 0>{});
                    f4(std::integral_constant<int, 4>{});
                    f4(std::integral_constant<int, 8>{});
                    f4(std::integral_constant<int, 12>{});
                }
            }
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
    const bool redo = __syncthreads_or(q48_f51_big(big));
    for (int i = tid; i < nrow * HD; i += 256) {
        const int r = i / HD, d = i % HD, v = 16 * tile + r;
        uint64_t o = lam[r][d];
        if (slow || redo) {
            const int64_t sum = (int64_t)dens[r];
            const q48_divisor dv = q48_divisor_of(sum);
            o = 0;
            for (int j = begin; j < end; ++j) {
                int64_t e = sc[(size_t)r * p.spad + j];
                if (sum > 0)
                    e = q48_div_by(e, dv);
                o += (uint64_t)q48_mul(e, value_at<BITS, HD>(a.v, a.vs, (size_t)j * a.n_kv + kh, d));
            }
        }
        int64_t *out =
            a.out + ((size_t)(p.t0 + v / G) * a.n_heads + kh * G + v % G) * HD + d;
        if (p.nchunk > 1)
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

// Rows of one launch: their scores take at most this much workspace.
constexpr size_t RA_WS_MAX = (size_t)1 << 30;

template <int BITS, int HD, bool DEC>
int launch_hd(q48_ctx *c, RaArgs &a)
{
    const int G = a.n_heads / a.n_kv;
    // positions a launch may reach: the cache's, where the device holds the position
    const int S = DEC ? (a.d_pos ? a.max_seq : a.p0 + 1) : a.p0 + a.T;
    RaPlan p = {};
    p.spad = (S + 63) & ~63;
    const size_t row_bytes = (size_t)a.n_heads * p.spad * 8;
    int Tn = (int)(RA_WS_MAX / row_bytes);
    Tn = Tn < 1 ? 1 : Tn < a.T ? Tn : a.T;
    p.tiles = (Tn * G + 15) / 16;
    // chunks for about 512 blocks, of 64 rows at least
    const long blocks = (long)p.tiles * a.n_kv;
    int n = (int)(blocks >= 512 ? 1 : (512 + blocks - 1) / blocks);
    n = n < p.spad / 64 ? n : p.spad / 64;
    p.ch = ((S + n - 1) / n + 63) & ~63;
    p.nchunk = (S + p.ch - 1) / p.ch;
    size_t o = 0;
    auto take = [&](size_t bytes) {
        const size_t at = o;
        o += (bytes + 255) & ~(size_t)255;
        return at;
    };
    const size_t vecs = (size_t)a.n_kv * p.tiles * 16, ft = (size_t)a.n_kv * p.tiles * p.nchunk;
    const size_t o_sc = take(vecs * p.spad * 8), o_cm = take(vecs * p.nchunk * 8);
    const size_t o_cs = take(vecs * p.nchunk * 8), o_far = take(ft * 4), o_odd = take(ft * 4);
    int rc = q48_ws_reserve(c, o);
    if (rc)
        return rc;
    uint8_t *ws = (uint8_t *)c->ws;
    p.sc = (int64_t *)(ws + o_sc);
    p.cm = (int64_t *)(ws + o_cm);
    p.cs = (uint64_t *)(ws + o_cs);
    p.far = (int *)(ws + o_far);
    p.odd = (int *)(ws + o_odd);
    constexpr int TB = DEC ? 1 : BITS == 64 ? 4 : 2;
    for (p.t0 = 0; p.t0 < a.T; p.t0 += Tn) {
        p.Tn = Tn < a.T - p.t0 ? Tn : a.T - p.t0;
        const int tiles = (p.Tn * G + 15) / 16;
        const dim3 grid(p.nchunk, tiles, a.n_kv);
        hipLaunchKernelGGL((k_ra_score<BITS, HD, TB, DEC>),
                           dim3(p.nchunk, (tiles + TB - 1) / TB, a.n_kv), dim3(256), 0, c->stream,
                           a, p);
        hipLaunchKernelGGL((k_ra_exp<DEC>), grid, dim3(256), 0, c->stream, a, p);
        hipLaunchKernelGGL((k_ra_value<BITS, HD, DEC>), grid, dim3(256), 0, c->stream, a, p);
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
    if (!c || !out || !q || !k_new || !v_new || !q48_qcache_ok(qc) || layer < 0 ||
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
    if (!c || !out || !QKV || !q48_qcache_ok(qc) || layer < 0 || layer >= qc->layers || T <= 0 ||
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
    if (!c || !out || !QKV || !kcache || !vcache || layer < 0 || T <= 0 || n_heads <= 0 ||
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
