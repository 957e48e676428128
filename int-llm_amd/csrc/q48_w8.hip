// q48_w8.hip — weights in 8 bits with a step a row, and their product with rows that
// are put into 8 bits with a step a row (include/intllm_hip.h has the integer steps).
#include "q48_w8.hpp"

namespace {

__device__ __forceinline__ uint64_t block_umax(uint64_t v, uint64_t *red)
{
    // magnitudes are at most 2^63: as signed words, less one, in order
    const int64_t m = q48_wave_max64((int64_t)(v - 1));
    if ((threadIdx.x & 63) == 0)
        red[threadIdx.x >> 6] = (uint64_t)m + 1;
    __syncthreads();
    uint64_t t = 0;
    for (int w = 0; w < (int)blockDim.x / 64; ++w)
        t = red[w] > t ? red[w] : t;
    __syncthreads();
    return t;
}

// Row of block b of n: the blocks of one die (every eighth) take eight neighbouring rows,
// whose codes share lines of 128 bytes, so that its L2 has whole lines to write.  us,
// without and with: 2560 x 2048 words packed 12.2 / 9.6, 2048 x 5632 23.2 / 19.1.
__device__ __forceinline__ int w8_near(int b, int n)
{
    return (b | 63) < n ? (b & ~63) | (b & 7) << 3 | (b >> 3 & 7) : b;
}

// A block a row: sum of squares, largest magnitude, codes, each a pass over the row.  Rows
// past T: zero codes.  Bound by the one block's passes in integers: a row of 28672 63 us.
__global__ __launch_bounds__(256) void k_w8_rows(W8Rows a)
{
    q48_round_down();
    __shared__ uint64_t red[4], red_lo[4], red_hi[4];
    __shared__ int64_t r_sh;
    const int t = w8_near(blockIdx.x, gridDim.x), tid = threadIdx.x, K = a.K, KT = (K + 63) / 64;
    if (a.tok && a.tok[t] < 0)
        return;
    const int64_t *x = a.X + (size_t)t * K;
    const bool past = t >= a.T;
    int64_t r = 0;
    if (a.norm_w) {
        q48_u128 ss = 0;
        for (int i = tid; i < K; i += 256)
            ss += (q48_u128)q48_smul128(x[i], x[i]);
        ss = block_sum128<256>(ss, red_lo, red_hi);
        if (tid == 0)
            r_sh = rms_inv_of(ss, K);
        __syncthreads();
        r = r_sh;
    }
    auto at = [&](int i) {
        return past ? 0 : a.norm_w ? q48_mul(q48_mul(x[i], r), a.norm_w[i]) : x[i];
    };
    uint64_t m = 0;
    for (int i = tid; i < K; i += 256) {
        const int64_t v = at(i);
        if (a.xn)
            a.xn[(size_t)t * K + i] = v;
        if (a.out)
            a.out[(size_t)t * K + i] = a.base ? a.base[(size_t)t * K + i] : 0;
        const uint64_t g = q48_magnitude(v);
        m = g > m ? g : m;
    }
    m = block_umax(m, red);
    double rc;
    const uint64_t step = w8_step(m, rc);
    if (tid == 0 && !past)
        a.step[t] = (int64_t)step;
    for (int i = tid; i < KT * 64; i += 256)
        a.codes[w8_at(t, i, KT)] = i < K && step ? (uint8_t)q48_code<127>(at(i), step, rc) : 0;
}

// The same with the row in registers, read once, FP64 where the words allow (RowWords).
// Many rows are bound by memory: 2048 rows of 5632 19.0 us (104 MB, 5.5 TB/s), 2560 rows of
// weights of 2048 9.6; with the norm by vector issue too: 2048 rows of 2048 15.0 (6.1 M wave
// instructions, about 10 us of FP64).  Few rows are one block's chain: 26 of 5632 5.0.
template <int NT, int C, int J, bool NORM>
__global__ __launch_bounds__(NT) void k_w8_rows_r(W8Rows a)
{
    q48_round_down();
    __shared__ uint64_t red[NT / 64][2], top[NT / 64];
    const int t = w8_near(blockIdx.x, gridDim.x), K = a.K, KT = (K + 63) / 64;
    if (a.tok && a.tok[t] < 0)
        return;
    RowWords<NT, C, J> x;
    x.load(a.X + (size_t)t * K, t < a.T ? K : 0);
    if constexpr (NORM)
        x.norm(a.X + (size_t)t * K, a.norm_w, K, red);
    if (a.xn)
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (x.at(j) + c < K)
                    a.xn[(size_t)t * K + x.at(j) + c] = x.word(j, c);
    if (a.out)
        for (int i = threadIdx.x; i < K; i += NT)
            a.out[(size_t)t * K + i] = a.base ? a.base[(size_t)t * K + i] : 0;
    const int64_t step = x.quantise(K, KT, top, [&](int i, uint32_t q) {
        uint8_t *to = a.codes + w8_at(t, i, KT);
        if constexpr (C == 4)
            *(uint32_t *)to = q;
        else
            *(uint16_t *)to = (uint16_t)q;
    });
    if (threadIdx.x == 0 && t < a.T)
        a.step[t] = step;
}

// Codes and steps as they come, a row of weights at a time.  A byte a thread: 32000 x 2048
// 52 us (131 MB, 2.5 TB/s), 2560 x 2048 5.3.
__global__ __launch_bounds__(256) void k_w8_put(uint8_t *__restrict__ codes,
                                               int64_t *__restrict__ steps,
                                               const int8_t *__restrict__ from,
                                               const int64_t *__restrict__ from_step, int N, int K)
{
    const int tid = threadIdx.x, KT = (K + 63) / 64;
    const int rows = (N + 15) & ~15;
    for (int b = blockIdx.x; b < rows; b += gridDim.x) {
        const int n = w8_near(b, rows);
        if (tid == 0 && n < N)
            steps[n] = from_step[n] < 0 ? 0 : from_step[n];
        for (int i = tid; i < KT * 64; i += 256)
            codes[w8_at(n, i, KT)] = n < N && i < K ? (uint8_t)from[(size_t)n * K + i] : 0;
    }
}

// The way back: eight rows x 2048 columns a block, through LDS so that tiles and words are
// whole lines.  Bound by memory: 2560 x 2048 10.6 us, 47 MB at 4.5 TB/s.
__global__ __launch_bounds__(512) void k_w8_values(int64_t *__restrict__ out,
                                                  const uint8_t *__restrict__ codes,
                                                  const int64_t *__restrict__ steps, int N, int K)
{
    constexpr int LD = 2048 + 16;
    __shared__ __align__(16) uint8_t rows[8][LD];
    const int tid = threadIdx.x, w = tid >> 6, n = blockIdx.x * 8 + w, KT = (K + 63) / 64;
    const int k0 = blockIdx.y * 2048, nk = min(K - k0, 2048);
    const uint8_t *from = codes + ((size_t)(blockIdx.x >> 1) * KT + (k0 >> 6)) * 1024 +
                          (blockIdx.x & 1) * 128;
    for (int i = tid; i < (nk + 15) / 16 * 8; i += 512)
        *(v4i *)&rows[i & 7][(i >> 3) * 16] = *(const v4i *)(from + (i >> 3) * 256 + (i & 7) * 16);
    __syncthreads();
    if (n >= N)
        return;
    const uint64_t step = (uint64_t)steps[n];
    int64_t *to = out + (size_t)n * K + k0;
    typedef int64_t words __attribute__((ext_vector_type(2), aligned(8)));
    for (int i = 2 * (tid & 63); i < nk; i += 128) {
        const uint16_t c = *(const uint16_t *)&rows[w][i];
        const words v = {(int64_t)((uint64_t)(int64_t)(int8_t)c * step),
                         (int64_t)((uint64_t)(int64_t)(int8_t)(c >> 8) * step)};
        if (i + 1 < nk)
            *(words *)(to + i) = v;
        else
            to[i] = v.x;
    }
}

// A block 16 weight rows x 16 NB rows: its NW waves take every NW-th tile of 64 columns,
// straight from memory into the matrix instruction's operands, and add up in LDS.  What
// bounds it is the loads under way, and for many rows the weights read again for every 64:
// 26 rows x 2048 x 5632 5.2 us; 208 pairs of 64 experts, gate and up of 1024 x 2048 48 us
// (5.6 TB/s of codes), down 28.5 (4.7; a block's 16 KB are one turn of loads).
template <int NB, int EPI, bool EXPERTS, int NW>
__global__ __launch_bounds__(64 * NW) void k_w8_mul(W8Mul m)
{
    q48_round_down();
    constexpr int M = EPI == 1 ? 2 : 1, NT = 64 * NW;
    constexpr int P = 12 / (M + NB) > 4 ? 4 : 12 / (M + NB);    // tiles a turn
    constexpr int IT = (NB * 256 + NT - 1) / NT;                // outputs a thread
    __shared__ __align__(16) int red[M * NB * NW][256];
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    int expert = 0, row0 = blockIdx.y * 16 * NB, rows = m.T - row0;
    if constexpr (EXPERTS) {
        const int4 it = m.items[blockIdx.y];
        expert = it.x;
        row0 = it.y;
        rows = it.z;
        if (rows <= 0)
            return;
    }
    rows = min(rows, 16 * NB);
    const int KT = m.KT, n0 = blockIdx.x * 16;
    const size_t tile = (size_t)expert * m.a_stride + (size_t)blockIdx.x * KT * 1024 + lane * 16;
    const uint8_t *A[2] = {m.A + tile, M == 2 ? m.A2 + tile : nullptr};
    const uint8_t *B[NB];
#pragma unroll
    for (int g = 0; g < NB; ++g) {
        const int r = row0 + 16 * min(g, (rows - 1) >> 4);
        if constexpr (EXPERTS && EPI == 1) {
            const int tok = max(m.slot_tok[r + (lane & 15)], 0);
            B[g] = m.B + (size_t)(tok >> 4) * KT * 1024 + (lane >> 4) * 256 + (tok & 15) * 16;
        } else {
            B[g] = m.B + (size_t)(r >> 4) * KT * 1024 + lane * 16;
        }
    }
    // what the epilogue needs, ahead of the products
    const int n = n0 + (tid & 15);
    const bool in = n < m.N;
    const size_t at_n = (size_t)expert * m.N + min(n, m.N - 1);
    const int64_t s1 = m.sw[at_n], s2 = M == 2 ? m.sw2[at_n] : 0;
    int64_t sb[IT], more[IT];   // more: the base, or the slot's weight
    int tok[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const int r = min((tid + NT * i) >> 4, rows - 1);
        tok[i] = EXPERTS ? m.slot_tok[row0 + r] : 0;
        sb[i] = m.sb[EXPERTS && EPI == 1 ? max(tok[i], 0) : row0 + r];
        more[i] = 0;
        if constexpr (EPI == 2)
            more[i] = m.slot_w[row0 + r];
        if (EPI == 0 && m.base)
            more[i] = m.base[(size_t)(row0 + r) * m.N + min(n, m.N - 1)];
    }
    v4i acc[M][NB] = {};
    for (int k0 = w; k0 < KT; k0 += NW * P) {
        v4i a[M][P], b[NB][P];
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const size_t k = k0 + NW * p;
            if ((int)k >= KT)
                break;
#pragma unroll
            for (int j = 0; j < M; ++j)
                a[j][p] = *(const v4i *)(A[j] + k * 1024);
#pragma unroll
            for (int g = 0; g < NB; ++g)
                b[g][p] = *(const v4i *)(B[g] + k * 1024);
        }
#pragma unroll
        for (int p = 0; p < P; ++p)
            if (k0 + NW * p < KT)
#pragma unroll
                for (int g = 0; g < NB; ++g)
#pragma unroll
                    for (int j = 0; j < M; ++j)
                        acc[j][g] =
                            __builtin_amdgcn_mfma_i32_16x16x64_i8(a[j][p], b[g][p], acc[j][g], 0, 0, 0);
    }
    // lane l, register i: weight row 4 (l / 16) + i, row l % 16
#pragma unroll
    for (int j = 0; j < M; ++j)
#pragma unroll
        for (int g = 0; g < NB; ++g)
            *(v4i *)&red[(j * NB + g) * NW + w][(lane & 15) * 16 + 4 * (lane >> 4)] = acc[j][g];
    lds_barrier();
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const int o = tid + NT * i, g = o >> 8, r = o >> 4;
        if (!in || r >= rows || tok[i] < 0)
            continue;
        int S[2] = {};
#pragma unroll
        for (int j = 0; j < M; ++j)
#pragma unroll
            for (int u = 0; u < NW; ++u)
                S[j] += red[(j * NB + g) * NW + u][o & 255];
        const size_t row = (size_t)row0 + r;
        if constexpr (EPI == 1) {
            m.Y[row * m.N + n] = w8_swiglu(S[0], S[1], sb[i], s1, s2);
        } else {
            const int64_t y = w8_times(S[0], sb[i], s1);
            if constexpr (EPI == 2)
                atomicAdd((unsigned long long *)m.Y + (size_t)tok[i] * m.N + n,
                          (unsigned long long)q48_mul(more[i], y));
            else
                m.Y[row * m.N + n] = (int64_t)((uint64_t)y + (uint64_t)more[i]);
        }
    }
}

// ---- one row ------------------------------------------------------------------

constexpr int ONE_NT = 1024;   // threads of a k_w8_one block

// One row times weights: S = 2^sl of the block's sixteen waves share a tile of 16 weight
// rows, each every S-th of its 64-column tiles; the row stands in all 16 columns of the
// matrix instruction's other operand.  SRC 1: the row from words, 2: rmsnorm'ed, both
// quantised by every block while its first weight tiles are on their way; 0: from codes.
// 32000 x 2048 normed 13.5 us: 65.5 MB at 6 TB/s behind the row's own 4 us (a launch of its
// own for the row would come on top); 2560 x 2048 7.0, nearly all of it the row's chain.
// Rows of 4096 (512 threads of 16 words): 4096 x 4096 normed 11.3, 128256 x 4096 103.  With a
// norm that form spills 53 registers, 56 with SwiGLU.
template <int EPI, bool EXPERTS, int SRC, int NT, int J>
__global__ __launch_bounds__(ONE_NT) void k_w8_one(W8Mul m, const int64_t *__restrict__ X,
                                                  const int64_t *__restrict__ norm_w, int K, int sl)
{
    q48_round_down();
    constexpr int M = EPI == 1 ? 2 : 1, NW = ONE_NT / 64, P = 8 / M;
    __shared__ __align__(16) uint8_t codes[SRC ? 2 * NT * J : 16];
    __shared__ uint64_t red[NW][2], top[NW];
    __shared__ int64_t step;
    __shared__ __align__(16) int sums[M][NW][16];
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int S = 1 << sl, TB = NW >> sl, ks = w & (S - 1);
    int expert = 0, slot = 0, tok = 0;
    int64_t wt = 0;
    if constexpr (EXPERTS) {
        const int4 it = m.items[blockIdx.y];
        expert = it.x;
        slot = it.y;
        if (it.z <= 0)
            return;
        tok = m.slot_tok[slot];
        if constexpr (EPI == 2)
            wt = m.slot_w[slot];
    }
    const int KT = m.KT, NTILE = (m.N + 15) / 16, groups = (NTILE + TB - 1) / TB;
    const size_t ex = (size_t)expert * m.a_stride + lane * 16;
    const uint8_t *A0 = m.A + ex, *A1 = M == 2 ? m.A2 + ex : nullptr;
    auto tile_at = [&](int g) { return (size_t)min(g * TB + (w >> sl), NTILE - 1) * KT; };
    v4i pre[M][P];
    auto load = [&](size_t t, int k0) {
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int k = k0 + p * S;
            if (k >= KT)
                break;
            pre[0][p] = *(const v4i *)(A0 + (t + k) * 1024);
            if constexpr (M == 2)
                pre[1][p] = *(const v4i *)(A1 + (t + k) * 1024);
        }
    };
    int g = blockIdx.x;
    load(tile_at(g), ks);
    int64_t sb;
    const uint8_t *B = nullptr;
    if constexpr (SRC) {
        if (tid < NT) {
            RowWords<NT, 2, J> x;
            x.load(X + (EXPERTS ? (size_t)slot * K : 0), K);
            if constexpr (SRC == 2)
                x.norm(X, norm_w, K, red);
            sb = x.quantise(K, KT, top,
                            [&](int i, uint32_t q) { *(uint16_t *)&codes[i] = (uint16_t)q; });
            if (tid == 0)
                step = sb;
        } else {
            lds_barrier();
            if constexpr (SRC == 2)
                lds_barrier();
        }
        lds_barrier();
        sb = step;
    } else {
        sb = m.sb[tok];
        B = m.B + (size_t)(tok >> 4) * KT * 1024 + (tok & 15) * 16 + (lane >> 4) * 256;
    }
    auto row = [&](int k) {
        if constexpr (SRC)
            return *(const v4i *)&codes[k * 64 + (lane >> 4) * 16];
        else
            return *(const v4i *)(B + (size_t)k * 1024);
    };
    const int64_t *sw = m.sw + (size_t)expert * m.N, *sw2 = m.sw2 + (size_t)expert * m.N;
    for (; g < groups; g += gridDim.x) {
        const size_t t = tile_at(g);
        // what the epilogue needs, ahead of the products
        int64_t s1 = 0, s2 = 0, add = 0;
        const int at = min((g * TB + (tid >> (sl + 4))) * 16 + ((tid >> sl) & 15), m.N - 1);
        if (tid < 256) {
            s1 = sw[at];
            if constexpr (EPI == 1)
                s2 = sw2[at];
            if (EPI == 0 && m.base)
                add = m.base[at];
        }
        v4i acc[M] = {};
        for (int k0 = ks; k0 < KT; k0 += P * S) {
            v4i now[M][P];
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
                for (int j = 0; j < M; ++j)
                    now[j][p] = pre[j][p];
            // the next tiles: of this row block, or of the block's next one
            if (k0 + P * S < KT)
                load(t, k0 + P * S);
            else if (g + (int)gridDim.x < groups)
                load(tile_at(g + gridDim.x), ks);
#pragma unroll
            for (int p = 0; p < P; ++p)
                if (k0 + p * S < KT) {
                    const v4i b = row(k0 + p * S);
#pragma unroll
                    for (int j = 0; j < M; ++j)
                        acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(now[j][p], b, acc[j], 0, 0, 0);
                }
        }
        // every column holds the sums of weight rows 4 (l / 16) + i
        if ((lane & 15) == 0)
#pragma unroll
            for (int j = 0; j < M; ++j)
                *(v4i *)&sums[j][w][4 * (lane >> 4)] = acc[j];
        lds_barrier();
        // lane i of every S: the i-th wave's sum of one weight row
        if (tid < 256) {
            const int i = tid & (S - 1), ch = (tid >> sl) & 15, tl = tid >> (sl + 4);
            int sum[M];
#pragma unroll
            for (int j = 0; j < M; ++j) {
                sum[j] = sums[j][(tl << sl) + i][ch];
                if (sl > 0)
                    sum[j] += q48_dpp32<Q48_DPP_XOR1>(sum[j]);
                if (sl > 1)
                    sum[j] += q48_dpp32<Q48_DPP_XOR2>(sum[j]);
                if (sl > 2)
                    sum[j] += q48_dpp32<Q48_DPP_HALF_MIRROR>(sum[j]);
                if (sl > 3)
                    sum[j] += q48_dpp32<Q48_DPP_MIRROR>(sum[j]);
            }
            const int n = (g * TB + tl) * 16 + ch;
            if (i == 0 && n < m.N) {
                int64_t y;
                if constexpr (EPI == 1)
                    y = w8_swiglu(sum[0], sum[1], sb, s1, s2);
                else
                    y = w8_times(sum[0], sb, s1);
                if constexpr (EPI == 2)
                    atomicAdd((unsigned long long *)m.Y + (size_t)tok * m.N + n,
                              (unsigned long long)q48_mul(wt, y));
                else
                    m.Y[(size_t)slot * m.N + n] = (int64_t)((uint64_t)y + (uint64_t)add);
            }
        }
        if (g + (int)gridDim.x < groups)
            lds_barrier();
    }
}

// ---- many rows ------------------------------------------------------------------

typedef int v16i __attribute__((ext_vector_type(16)));

// s_waitcnt vmcnt(n) with the other counters left alone (gfx9 encoding)
template <int N>
__device__ __forceinline__ void wait_vm()
{
    static_assert(N >= 0 && N < 64, "vmcnt");
    __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
}

// 16 bytes a lane from `from` to the wave's 1 KB at `to`
__device__ __forceinline__ void dma_tile(const uint8_t *from, uint8_t *to)
{
    __builtin_amdgcn_global_load_lds(from, to, 16, 0, 0);
}

constexpr int GT = 128;                  // weight rows (EPI 1: half of each matrix) and rows a block
constexpr int GSTAGE = 2 * GT * 64;      // bytes of a stage: 64 columns of both

// A block 128 weight rows x 128 rows, four waves of 64 x 64.  Tiles of both operands go to a
// ring of three LDS stages by DMA, 1 KB a wave and instruction, two stages ahead; the matrix
// instruction's first operand is the rows, so that a lane holds one weight row and stores of
// a wave are 256 contiguous bytes.  The sums leave the registers through LDS, half of the
// rows at a time, so that one loop of the epilogue's code serves all of them.
// KS 1: three blocks a compute unit; a wave alone on its SIMD issues every other turn at
// most, and the epilogue is as much work as the products.  KS 2, where there is at most a
// block a compute unit: two groups of four waves, each over half of the columns with a ring
// of its own, that share the epilogue.
// 2048 x 2048 x 5632 with a residual 36.5 us (1.29 POP/s, epilogue included): one tile a
// compute unit, so that its residual and results (67 MB) wait for its products; of 66 k cycles
// 23 k are matrix instructions and 12 k vector instructions.  SwiGLU of 2048 x 5632 x 2048 100
// us: vector instructions (28.5 M, four cycles each; 158 an output, 112 of them FP64) and
// matrix instructions (45 k cycles a SIMD) add up to 0.9 of its cycles; they do not overlap on
// one SIMD, whatever the order of the blocks or the waves a block.
template <int EPI, bool EXPERTS, int KS>
__global__ __launch_bounds__(256 * KS, KS == 1 ? 3 : 2) void k_w8_gemm(W8Mul m, int nx, int ny)
{
    q48_round_down();
    constexpr int CH = EPI == 1 ? GT / 2 : GT;   // weight rows of one matrix
    constexpr int WPG = 4;                       // waves of a group
    constexpr int TPW = GSTAGE / 1024 / WPG;     // tiles of it a wave moves
    // apart, so that the compiler sees that a stage's reads do not wait for another's DMA
    __shared__ __align__(16) uint8_t r0[KS * GSTAGE], r1[KS * GSTAGE], r2[KS * GSTAGE];
    __shared__ double sd[GT], wd[EPI == 2 ? GT : 1];
    __shared__ int toks[EXPERTS ? GT : 1];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int q = wave / WPG, w = wave % WPG, wc = w & 1, r_w = (w >> 1) * 64;   // its rows
    // blocks of one die (every eighth) take neighbouring tiles, the rows' fastest
    const int per = (nx * ny + 7) >> 3, at = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || at >= nx * ny)
        return;
    const int bx = at / ny, by = at % ny;
    int expert = 0, row0 = by * GT, rows = m.T - row0;
    if constexpr (EXPERTS) {
        const int4 it = m.items[by];
        expert = it.x;
        row0 = it.y;
        rows = it.z;
        if (rows <= 0)
            return;
    }
    rows = min(rows, GT);
    const int KT = (m.KT + KS - 1) / KS;        // steps of a group; of the last one, its own
    const int kt0 = q * KT, mine_kt = KS == 1 ? KT : min(KT, m.KT - kt0);
    const int n0 = bx * CH, ntile = (m.N + 15) / 16;
    int64_t mine_step = 0;   // in LDS behind the first DMA
    if (tid < GT) {
        const int r = min(tid, rows - 1);
        int64_t step;
        if constexpr (EXPERTS) {
            const int tok = m.slot_tok[row0 + r];
            toks[tid] = tok;
            step = m.sb[EPI == 1 ? max(tok, 0) : row0 + r];
            if constexpr (EPI == 2)
                wd[tid] = (double)m.slot_w[row0 + r] * 0x1p-48;
        } else {
            step = m.sb[row0 + r];
        }
        mine_step = step;
    }
    // row t of the wave's, in sb and base; rows past the block's last: that one
    auto row_of = [&](int t) {
        const int i = min(r_w + t, rows - 1);
        if constexpr (EXPERTS && EPI == 1)
            return max(toks[i], 0);
        else
            return row0 + i;
    };
    // this wave's tiles of a stage, of 8 of the weights and then 8 of the rows
    const uint8_t *src[TPW];
#pragma unroll
    for (int j = 0; j < TPW; ++j) {
        const int a = TPW * w + j;
        if (a < 8) {   // EPI 1: tiles 0 .. 3 of gate, 4 .. 7 of up
            const bool second = EPI == 1 && a >= 4;
            const int t = min((n0 >> 4) + (second ? a - 4 : a), ntile - 1);
            src[j] = (second ? m.A2 : m.A) + (size_t)expert * m.a_stride +
                     ((size_t)t * m.KT + kt0) * 1024 + lane * 16;
        } else {
            const int r = min(16 * (a - 8), (rows - 1) & ~15) + row0;
            if constexpr (EXPERTS && EPI == 1) {
                const int tok = max(m.slot_tok[r + (lane & 15)], 0);
                src[j] = m.B + ((size_t)(tok >> 4) * m.KT + kt0) * 1024 + (lane >> 4) * 256 +
                         (tok & 15) * 16;
            } else {
                src[j] = m.B + ((size_t)(r >> 4) * m.KT + kt0) * 1024 + lane * 16;
            }
        }
    }
    auto dma = [&](int k, uint8_t(&st)[KS * GSTAGE]) {
        uint8_t *to = st + q * GSTAGE + TPW * w * 1024;
        if constexpr (KS > 1)   // (past a shorter group's end: a stage that is not multiplied)
            k = min(k, mine_kt - 1);
#pragma unroll
        for (int j = 0; j < TPW; ++j)
            dma_tile(src[j] + (size_t)k * 1024, to + j * 1024);
    };
    v16i acc[2][2] = {};
    // rows l % 32 of a pair of tiles, columns 16 (l / 32) on
    const int mine = ((lane & 31) >> 4) * 1024 + (lane >> 5) * 256 + (lane & 15) * 16;
    auto step = [&](const uint8_t(&stage)[KS * GSTAGE]) {
        const uint8_t *st = stage + q * GSTAGE + mine;
        v4i a[2][2], b[2][2];   // [pair][half of the columns], of the weights and of the rows
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int f = 0; f < 2; ++f) {
                const int ta = EPI == 1 ? 4 * f + 2 * wc : 4 * wc + 2 * f;
                a[f][h] = *(const v4i *)(st + ta * 1024 + h * 512);
                b[f][h] = *(const v4i *)(st + (8 + r_w / 16 + 2 * f) * 1024 + h * 512);
            }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
                for (int f = 0; f < 2; ++f)
                    acc[f][g] = __builtin_amdgcn_mfma_i32_32x32x32_i8(b[g][h], a[f][h], acc[f][g], 0, 0, 0);
    };
    dma(0, r0);
    if (KT > 1)
        dma(1, r1);
    const int64_t *sw = m.sw + (size_t)expert * m.N, *sw2 = m.sw2 + (size_t)expert * m.N;
    const int n = n0 + (EPI == 1 ? 32 * wc + (lane & 31) : 64 * wc + lane);
    const bool in = n < m.N;
    const int64_t s1 = in ? sw[n] : 0, s2 = in && EPI == 1 ? sw2[n] : 0;
    if (tid < GT)
        sd[tid] = w8_step_double(mine_step);
    int k = 0;
    // Step k: its stage has arrived, and every wave is done with the last one's, which the
    // DMA of k + 2 takes.
    auto turn = [&](const uint8_t(&now)[KS * GSTAGE], uint8_t(&free)[KS * GSTAGE]) {
        wait_vm<TPW>();
        lds_barrier();
        dma(k + 2, free);
        step(now);
        ++k;
    };
    // the last ones
    auto tail = [&](const uint8_t(&now)[KS * GSTAGE], uint8_t(&free)[KS * GSTAGE]) {
        if (k >= KT)
            return;
        wait_vm<0>();
        lds_barrier();
        if (k + 2 < KT)
            dma(k + 2, free);
        if (KS == 1 || k < mine_kt)
            step(now);
        ++k;
    };
    while (k + 4 < KT) {
        turn(r0, r2);
        turn(r1, r0);
        turn(r2, r1);
    }
    tail(r0, r2);
    tail(r1, r0);
    tail(r2, r1);
    tail(r0, r2);
    // of wave i: [pair of weight rows][row][weight row]
    auto sums_of = [&](int i) { return (int *)((i < 2 * KS ? r0 : r1) + i % (2 * KS) * 8192); };
    int *own = sums_of(wave);
    const int *part0 = sums_of(w), *part1 = sums_of(KS > 1 ? WPG + w : w);
    auto sum = [&](int o) { return KS > 1 ? part0[o] + part1[o] : part0[o]; };
    const double d1 = w8_step_double(s1) * 0x1p-48, d2 = w8_step_double(s2) * 0x1p-48;
    // U outputs a turn: chains of FP64 operations side by side
    constexpr int U = EPI == 1 ? 2 : 8, PER = EPI == 1 ? 2 : 1;   // rows of a wave at once
    const int first = EPI == 1 ? lane >> 5 : 0;
    // the base a turn ahead of the sums
    int64_t add[U] = {};
    auto base = [&](int t0) {
        if constexpr (EPI == 0)
            if (m.base && in)
#pragma unroll
                for (int j = 0; j < U; ++j)
                    add[j] = m.base[(size_t)row_of(t0 + j) * m.N + n];
    };
#pragma nounroll
    for (int half = 0; half < 2; ++half) {
        lds_barrier();   // the ring, or the other half's sums, are done with
        // lane l, register i: row 8 (i / 4) + 4 (l / 32) + i % 4, weight row l % 32
        auto put = [&](const v16i(&s)[2][2], int g) {
#pragma unroll
            for (int f = 0; f < 2; ++f)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    own[(f * 32 + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3)) * 32 + (lane & 31)] = s[f][g][i];
        };
        if (half)
            put(acc, 1);
        else
            put(acc, 0);
        // (a group's share of the rows)
        const int begin = 32 * half + 32 / KS * q, last = min(begin + 32 / KS, rows - r_w);
        base(begin);
        if constexpr (KS > 1)
            lds_barrier();
        else
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the wave's own words
#pragma nounroll
        for (int t0 = begin; t0 < last; t0 += U * PER) {
            double y[U], up[EPI == 1 ? U : 1];
            bool ok = true;
            // output j's sum (up's lies 1024 words on)
            auto at_of = [&](int j) {
                const int t = t0 - 32 * half + PER * j + first;   // (past the last: of other rows)
                return t * 32 + (lane & 31) + (EPI == 1 ? 0 : (lane >> 5) * 1024);
            };
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const double sa = sd[r_w + t0 + PER * j + first];
                bool sure;
                y[j] = w8_scaled_double(sum(at_of(j)), sa, d1, sure);
                ok &= sure;
                if constexpr (EPI == 1) {
                    up[j] = w8_scaled_double(sum(1024 + at_of(j)), sa, d2, sure);
                    ok &= sure;
                }
            }
            if constexpr (EPI == 1) {
                double z[U];
                ok &= w8_silu_mul<U>(y, up, z);
#pragma unroll
                for (int j = 0; j < U; ++j)
                    y[j] = z[j];
            }
            if constexpr (EPI == 2)   // fp_mul by the weight, at most 1
#pragma unroll
                for (int j = 0; j < U; ++j)
                    y[j] = __builtin_floor(y[j] * wd[r_w + t0 + j]);
            int64_t v[U];
            if constexpr (EPI == 0) {   // (w8_words' two forms of eight would spill)
#pragma unroll
                for (int j = 0; j < U; ++j)
                    v[j] = (int64_t)y[j];
            } else {
                w8_words<U>(y, v);
            }
            if (__any(!ok))
#pragma nounroll
                for (int j = 0; j < U; ++j) {
                    const int64_t sa = m.sb[row_of(t0 + PER * j + first)];
                    int64_t z = w8_scaled(sum(at_of(j)), sa, s1);
                    if constexpr (EPI == 1)
                        z = q48_mul(q48_silu(z), w8_scaled(sum(1024 + at_of(j)), sa, s2));
                    if constexpr (EPI == 2)
                        z = q48_mul(z, m.slot_w[row_of(t0 + j)]);
#pragma unroll
                    for (int i = 0; i < U; ++i)
                        v[i] = i == j ? z : v[i];
                }
            if constexpr (EPI == 0) {
#pragma unroll
                for (int j = 0; j < U; ++j)
                    v[j] = (int64_t)((uint64_t)v[j] + (uint64_t)add[j]);
                if (t0 + U < last)
                    base(t0 + U);
            }
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const int t = t0 + PER * j + first;
                const size_t row = (size_t)(row0 + r_w + t);
                if (!in || t >= last || (EXPERTS && toks[r_w + t] < 0))
                    continue;
                if constexpr (EPI == 2)
                    atomicAdd((unsigned long long *)m.Y + (size_t)toks[r_w + t] * m.N + n,
                              (unsigned long long)v[j]);
                else
                    m.Y[row * m.N + n] = v[j];
            }
        }
    }
}

int launch_rc(int e) { return e == (int)hipSuccess ? Q48_OK : Q48_EHIP; }

// Y and what a product reads, and the product itself: gate and up, or one matrix.
int w8_product(q48_ctx *c, int64_t *Y, const int64_t *base, const q48_w8 *w, const q48_w8 *w2,
               const int64_t *X, const int64_t *norm_w, int T)
{
    if (!c || !Y || !X || !q48_w8_ok(w) || (w2 && !q48_w8_ok(w2)) || T <= 0 || T > W8_MAX_T ||
        q48_off_words<8>(Y, base, X, norm_w))
        return Q48_EINVAL;
    if (w->count != 1 || (w2 && (w2->count != 1 || w2->N != w->N || w2->K != w->K)))
        return Q48_EINVAL;
    const int N = w->N, K = w->K;
    const size_t out = (size_t)T * N * 8;
    if (q48_share(Y, out, X, (size_t)T * K * 8) || q48_share(Y, out, norm_w, (size_t)K * 8) ||
        (base != Y && q48_share(Y, out, base, out)))
        return Q48_EINVAL;
    for (const q48_w8 *m : {w, w2})
        if (m && (q48_share(Y, out, m->codes, w8_tiles(N, K)) ||
                  q48_share(Y, out, m->step, (size_t)N * 8)))
            return Q48_EINVAL;
    q48_on_device on(c);
    W8Mul m = {};
    m.A = (const uint8_t *)w->codes;
    m.sw = w->step;
    if (w2) {
        m.A2 = (const uint8_t *)w2->codes;
        m.sw2 = w2->step;
    }
    m.N = N;
    m.KT = w8_kt(K);
    m.T = T;
    m.Y = Y;
    m.base = base;
    if (T == 1 && q48_w8_one_ok(K))
        return launch_rc(q48_launch_w8_one(c, m, w2 ? 1 : 0, X, norm_w, K, 0));
    const size_t codes = w8_tiles(T, K);
    int rc = q48_w8_reserve(c, W8_TICKETS + codes + (size_t)T * 8);
    if (rc)
        return rc;
    uint8_t *ws = (uint8_t *)c->w8 + W8_TICKETS;
    W8Rows r = {};
    r.codes = ws;
    r.step = (int64_t *)(ws + codes);
    r.X = X;
    r.norm_w = norm_w;
    r.T = T;
    r.K = K;
    if ((rc = q48_launch_w8_rows(c, r)))
        return launch_rc(rc);
    m.B = r.codes;
    m.sb = r.step;
    return launch_rc(q48_launch_w8_mul(c, m, w2 ? 1 : 0, false, 0));
}

} // namespace

bool q48_w8_ok(const q48_w8 *w)
{
    return w && w->codes && w->step && ((uintptr_t)w->codes & 15) == 0 &&
           ((uintptr_t)w->step & 7) == 0 && w->count > 0 && w->count <= W8_MAX_COUNT &&
           w->N > 0 && w->N <= W8_MAX_N && w->K > 0 && w->K <= W8_MAX_K;
}

int q48_w8_reserve(q48_ctx *c, size_t bytes)
{
    if (q48_foreign_capture(c))
        return Q48_ESTATE;
    if (bytes <= c->w8_bytes)
        return Q48_OK;
    if (c->capturing)
        return Q48_ESTATE;   // workspaces reach their size outside a capture
    if (c->w8) {
        const int rc = q48_release(c, c->w8);
        if (rc)
            return rc;
        c->w8 = nullptr;
        c->w8_bytes = 0;
    }
    const size_t sz = bytes < ((size_t)1 << 20) ? ((size_t)1 << 20) : bytes;
    if (hipMalloc(&c->w8, sz) != hipSuccess) {
        c->w8 = nullptr;
        (void)hipGetLastError();
        return Q48_ENOMEM;
    }
    c->w8_bytes = sz;
    // tickets at its start are zeros between launches
    return launch_rc(q48_launch_zero(c, c->w8, W8_TICKETS));
}

int q48_launch_w8_rows(q48_ctx *c, const W8Rows &r, int blocks)
{
    const dim3 grid(blocks ? blocks : r.T);
    // Waves for a row by what it holds: one up to 512 words (20000 rows of 100 23.6 to 11.1 us,
    // 7000 of 300 11.6 to 7.6), sixteen past 8192, else four (eight are no faster where rows are
    // few either: with a product behind, 26 normed rows of 2048 8.7 / 7.9, 200 of 5632 16.0 /
    // 15.0, not normed 12.4 / 12.4).
#define W8_ROWS(NT, C, J)                                                                      \
    do {                                                                                       \
        if (r.norm_w)                                                                          \
            hipLaunchKernelGGL((k_w8_rows_r<NT, C, J, true>), grid, dim3(NT), 0, c->stream, r);  \
        else                                                                                   \
            hipLaunchKernelGGL((k_w8_rows_r<NT, C, J, false>), grid, dim3(NT), 0, c->stream, r); \
    } while (0)
    if (r.K > 16384)
        hipLaunchKernelGGL(k_w8_rows, grid, dim3(256), 0, c->stream, r);
    else if (r.K > 8192)
        W8_ROWS(1024, 2, 8);
    else if (r.K <= 512)
        W8_ROWS(64, 4, 2);
    else if (r.K <= 1024)
        W8_ROWS(256, 4, 1);
    else if (r.K <= 2048)
        W8_ROWS(256, 4, 2);
    else if (r.K <= 6144)
        W8_ROWS(256, 4, 6);
    else
        W8_ROWS(256, 4, 8);
#undef W8_ROWS
    return (int)hipGetLastError();
}

int q48_launch_w8_one(q48_ctx *c, const W8Mul &m, int epi, const int64_t *X,
                      const int64_t *norm_w, int K, int n_items)
{
    const int nt = (m.N + 15) / 16, per = n_items ? n_items : 1;
    // the most waves a tile with which every block is resident at once
    int sl = 4;
    auto groups_of = [&](int l) { return (nt + (16 >> l) - 1) / (16 >> l); };
    while (sl > 0 && groups_of(sl) * per > c->cu_count)
        --sl;
    const int groups = groups_of(sl), most = c->cu_count;
    const dim3 grid(groups < most ? groups : most, per);
#define W8_ONE(EPI, EX, SRC, NT, J)                                                                  \
    hipLaunchKernelGGL((k_w8_one<EPI, EX, SRC, NT, J>), grid, dim3(ONE_NT), 0, c->stream, m, X, norm_w, \
                       K, sl)
#define W8_ONE_J(EPI, EX, SRC)                                                                   \
    do {                                                                                         \
        if (K <= 2048)                                                                     \
            W8_ONE(EPI, EX, SRC, 256, 4);                                                             \
        else                                                                                     \
            W8_ONE(EPI, EX, SRC, 512, 8);                                                             \
    } while (0)
    if (n_items && epi == 1)
        W8_ONE(1, true, 0, 64, 1);
    else if (n_items)
        W8_ONE_J(2, true, 1);
    else if (epi == 1 && norm_w)
        W8_ONE_J(1, false, 2);
    else if (epi == 1)
        W8_ONE_J(1, false, 1);
    else if (norm_w)
        W8_ONE_J(0, false, 2);
    else
        W8_ONE_J(0, false, 1);
#undef W8_ONE_J
#undef W8_ONE
    return (int)hipGetLastError();
}

int q48_launch_w8_mul(q48_ctx *c, const W8Mul &m, int epi, bool experts, int n_items)
{
    const unsigned nx = (m.N + 15) / 16;
    // Tiles of 128 x 128 where there are outputs to fill the chip with them.  us, k_w8_mul /
    // k_w8_gemm: 2560 x 2048 512 rows 18.6 / 21.7, 768 24.6 / 24.1, 1024 28.6 / 25.7; 2048 x
    // 5632 512 30.9 / 35.3, 1024 49.7 / 40.3; 1031 x 2047 1024 21.9 / 25.2, 2048 33.1 / 29.0;
    // 8000 x 512 256 12.8 / 15.4, 512 19.3 / 16.7; SwiGLU of 5632 x 2048 512 40.3 / 43.8, 768
    // 57.9 / 58.7, 1024 75.4 / 62.7; of 3001 x 700 1024 32.7 / 35.3.  Few rows of many outputs:
    // 128000 x 2048 17 rows 58 / 60, 32 66 / 75, 64 101 / 85; x 4096 17 133 / 118, 64 185 / 134;
    // 64000 x 2048 32 27 / 39, 33 33 / 41, 64 38 / 44, 65 59 / 45; 32000 x 2048 64 22.7 / 24.2, 65
    // 33.1 / 24.4; SwiGLU of 64000 x 2048 64 77 / 94, 96 119 / 95; of 14336 x 4096 256 86 / 64.
    const bool tiles = experts ? m.rows > 64 : (size_t)m.T * m.N >= (epi == 1 ? 4u : 2u) << 20;
    if (tiles) {
        const int ch = epi == 1 ? GT / 2 : GT, gx = (m.N + ch - 1) / ch;
        const int gy = experts ? n_items : (m.T + GT - 1) / GT;
        const dim3 grid((unsigned)((gx * gy + 7) / 8 * 8));
        const bool halves = gx * gy <= c->cu_count && m.KT >= 8;
#define W8_GEMM(EPI, EX, KS)                                                              \
    hipLaunchKernelGGL((k_w8_gemm<EPI, EX, KS>), grid, dim3(256 * KS), 0, c->stream, m, gx, gy)
        if (experts && epi == 1)
            W8_GEMM(1, true, 1);
        else if (experts)
            W8_GEMM(2, true, 1);
        else if (epi == 1)   // (512 blocks and more)
            W8_GEMM(1, false, 1);
        else if (halves)
            W8_GEMM(0, false, 2);
        else
            W8_GEMM(0, false, 1);
#undef W8_GEMM
        return (int)hipGetLastError();
    }
    // Eight waves a block where that is two blocks a compute unit at most.  us, four / eight /
    // sixteen: 26 rows x 2048 x 5632 11.8 / 9.9 / 10.1, 64 14.3 / 12.1 / 12.2; x 2560 x 2048
    // 26 rows 7.4 / 7.1 / 7.3, 256 12.6 / 12.9 / 14.5; SwiGLU of 5632 x 2048 2 rows 7.7 / 7.6
    // / 8.6, 256 24.5 / 24.3 / 24.6.
    const int rows = experts ? m.rows : m.T <= 16 ? 16 : m.T <= 32 ? 32 : 64;
    const int ny = experts ? n_items : (m.T + rows - 1) / rows;
    const bool eight = (size_t)nx * ny <= 2 * (size_t)c->cu_count;
#define W8_MUL(NB, EPI, EX)                                                                      \
    do {                                                                                         \
        if (eight)                                                                               \
            hipLaunchKernelGGL((k_w8_mul<NB, EPI, EX, 8>), dim3(nx, ny), dim3(512), 0, c->stream, m); \
        else                                                                                     \
            hipLaunchKernelGGL((k_w8_mul<NB, EPI, EX, 4>), dim3(nx, ny), dim3(256), 0, c->stream, m); \
    } while (0)
#define W8_MUL_NB(EPI, EX)                                                                       \
    do {                                                                                         \
        if (rows == 16)                                                                          \
            W8_MUL(1, EPI, EX);                                                                  \
        else if (rows == 32)                                                                     \
            W8_MUL(2, EPI, EX);                                                                  \
        else                                                                                     \
            W8_MUL(4, EPI, EX);                                                                  \
    } while (0)
    if (experts && epi == 1)
        W8_MUL_NB(1, true);
    else if (experts)
        W8_MUL_NB(2, true);
    else if (epi == 1)
        W8_MUL_NB(1, false);
    else
        W8_MUL_NB(0, false);
#undef W8_MUL_NB
#undef W8_MUL
    return (int)hipGetLastError();
}

extern "C" {

int q48_w8_bytes(int count, int N, int K, size_t *codes, size_t *steps)
{
    alignas(16) static char some[16];
    const q48_w8 w = {some, (int64_t *)some, count, N, K};
    if (!codes || !steps || !q48_w8_ok(&w))
        return Q48_EINVAL;
    *codes = (size_t)count * w8_tiles(N, K);
    *steps = (size_t)count * N * 8;
    return Q48_OK;
}

static int w8_fill(q48_ctx *c, const q48_w8 *w, int index, const int64_t *W, const int8_t *codes,
                   const int64_t *steps)
{
    if (!c || !q48_w8_ok(w) || index < 0 || index >= w->count)
        return Q48_EINVAL;
    const int N = w->N, K = w->K;
    const size_t bytes = w8_tiles(N, K), n = (size_t)N * K;
    uint8_t *to = (uint8_t *)w->codes + (size_t)index * bytes;
    int64_t *st = w->step + (size_t)index * N;
    auto over = [&](const void *in, size_t size) {
        return q48_share(to, bytes, in, size) || q48_share(st, (size_t)N * 8, in, size);
    };
    if (over(W, n * 8) || over(codes, n) || over(steps, (size_t)N * 8))
        return Q48_EINVAL;
    q48_on_device on(c);
    // a launch holds fewer than 2^32 threads: N may be 2^24
    constexpr int most = 1 << 20;
    if (W) {   // as rows are
        for (int n0 = 0; n0 < N; n0 += most) {
            W8Rows r = {};
            r.codes = to + (size_t)(n0 / 16) * w8_kt(K) * 1024;
            r.step = st + n0;
            r.X = W + (size_t)n0 * K;
            r.T = min(N - n0, most);
            r.K = K;
            if (const int rc = q48_launch_w8_rows(c, r, (r.T + 15) & ~15))
                return launch_rc(rc);
        }
        return Q48_OK;
    }
    hipLaunchKernelGGL(k_w8_put, dim3(min((N + 15) / 16 * 16, most)), dim3(256), 0, c->stream, to,
                       st, codes, steps, N, K);
    return launch_rc((int)hipGetLastError());
}

int q48_w8_pack(q48_ctx *c, const q48_w8 *w, int index, const int64_t *W)
{
    if (!W || q48_off_words<8>(W))
        return Q48_EINVAL;
    return w8_fill(c, w, index, W, nullptr, nullptr);
}

int q48_w8_put(q48_ctx *c, const q48_w8 *w, int index, const int8_t *codes, const int64_t *steps)
{
    if (!codes || !steps || q48_off_words<8>(steps))
        return Q48_EINVAL;
    return w8_fill(c, w, index, nullptr, codes, steps);
}

int q48_w8_values(q48_ctx *c, int64_t *out, const q48_w8 *w, int index)
{
    if (!c || !out || q48_off_words<8>(out) || !q48_w8_ok(w) || index < 0 || index >= w->count)
        return Q48_EINVAL;
    const int N = w->N, K = w->K;
    const size_t bytes = w8_tiles(N, K), n = (size_t)N * K * 8;
    const uint8_t *from = (const uint8_t *)w->codes + (size_t)index * bytes;
    const int64_t *st = w->step + (size_t)index * N;
    if (q48_share(out, n, from, bytes) || q48_share(out, n, st, (size_t)N * 8))
        return Q48_EINVAL;
    q48_on_device on(c);
    hipLaunchKernelGGL(k_w8_values, dim3((N + 7) / 8, (K + 2047) / 2048), dim3(512), 0, c->stream, out, from, st, N, K);
    return launch_rc((int)hipGetLastError());
}

int q48_gemm_w8(q48_ctx *c, int64_t *Y, const int64_t *base, const q48_w8 *w, const int64_t *X,
                const int64_t *norm_w, int T)
{
    return w8_product(c, Y, base, w, nullptr, X, norm_w, T);
}

int q48_gemm_w8_swiglu(q48_ctx *c, int64_t *out, const q48_w8 *gate, const q48_w8 *up,
                       const int64_t *X, const int64_t *norm_w, int T)
{
    if (!up)
        return Q48_EINVAL;
    return w8_product(c, out, nullptr, gate, up, X, norm_w, T);
}

} // extern "C"
