// q48_w8.hip — weights in 8 bits with a step a row, and their product with rows that
// are put into 8 bits with a step a row (include/intllm_hip.h has the integer steps).
#include "q48_w8.hpp"

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

__device__ __forceinline__ size_t w8_at(int row, int col, int KT)
{
    return ((size_t)(row >> 4) * KT + (col >> 6)) * 1024 + ((col & 63) >> 4) * 256 +
           (row & 15) * 16 + (col & 15);
}

// A block a row: sum of squares, largest magnitude, codes, each a pass over the row.
__global__ __launch_bounds__(256) void k_w8_rows(W8Rows a)
{
    q48_round_down();
    __shared__ uint64_t red[4], red_lo[4], red_hi[4];
    __shared__ int64_t r_sh;
    const int t = blockIdx.x, tid = threadIdx.x, K = a.K, KT = (K + 63) / 64;
    if (a.tok && a.tok[t] < 0)
        return;
    const int64_t *x = a.X + (size_t)t * K;
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
    auto at = [&](int i) { return a.norm_w ? q48_mul(q48_mul(x[i], r), a.norm_w[i]) : x[i]; };
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
    if (tid == 0)
        a.step[t] = (int64_t)step;
    for (int i = tid; i < KT * 64; i += 256)
        a.codes[w8_at(t, i, KT)] = i < K && step ? (uint8_t)q48_code<127>(at(i), step, rc) : 0;
}

// A block a row of weights: step and codes, or codes and steps as they come.
__global__ __launch_bounds__(256) void k_w8_pack(uint8_t *__restrict__ codes,
                                                int64_t *__restrict__ steps,
                                                const int64_t *__restrict__ W,
                                                const int8_t *__restrict__ from,
                                                const int64_t *__restrict__ from_step, int N,
                                                int K)
{
    q48_round_down();
    __shared__ uint64_t red[4];
    const int n = blockIdx.x, tid = threadIdx.x, KT = (K + 63) / 64;
    uint64_t m = 0, step = 0;
    double rc = 0;
    if (n < N) {
        if (W) {
            for (int i = tid; i < K; i += 256) {
                const uint64_t g = q48_magnitude(W[(size_t)n * K + i]);
                m = g > m ? g : m;
            }
            step = w8_step(block_umax(m, red), rc);
        } else {
            step = from_step[n] < 0 ? 0 : (uint64_t)from_step[n];
        }
        if (tid == 0)
            steps[n] = (int64_t)step;
    }
    for (int i = tid; i < KT * 64; i += 256) {
        int q = 0;
        if (n < N && i < K)
            q = W ? step ? q48_code<127>(W[(size_t)n * K + i], step, rc) : 0
                  : from[(size_t)n * K + i];
        codes[w8_at(n, i, KT)] = (uint8_t)q;
    }
}

__global__ __launch_bounds__(256) void k_w8_values(int64_t *__restrict__ out,
                                                  const uint8_t *__restrict__ codes,
                                                  const int64_t *__restrict__ steps, int N, int K)
{
    const int n = blockIdx.x, KT = (K + 63) / 64;
    const uint64_t step = (uint64_t)steps[n];
    for (int i = threadIdx.x; i < K; i += 256)
        out[(size_t)n * K + i] = (int64_t)((uint64_t)(int64_t)(int8_t)codes[w8_at(n, i, KT)] * step);
}

// A block 16 weight rows x 16 NB rows: its four waves take every fourth tile of 64
// columns and add up in LDS.
template <int NB, int EPI, bool EXPERTS>
__global__ __launch_bounds__(256) void k_w8_mul(W8Mul m)
{
    q48_round_down();
    constexpr int M = EPI == 1 ? 2 : 1;
    __shared__ __align__(16) int red[M][4][256];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    int expert = 0, row0 = blockIdx.y * 16 * NB, rows = m.T - row0;
    if constexpr (EXPERTS) {
        const int4 it = m.items[blockIdx.y];
        expert = it.x;
        row0 = it.y;
        rows = it.z;
        if (rows <= 0)
            return;
    }
    const int KT = m.KT, n0 = blockIdx.x * 16;
    const size_t tile = (size_t)expert * m.a_stride + (size_t)blockIdx.x * KT * 1024 + lane * 16;
    const uint8_t *A[2] = {m.A + tile, M == 2 ? m.A2 + tile : nullptr};
    const uint8_t *B[NB];
#pragma unroll
    for (int g = 0; g < NB; ++g) {
        const int last = (rows + 15) / 16 - 1;
        const int r = row0 + 16 * (g < last ? g : last);
        if constexpr (EXPERTS && EPI == 1) {
            int tok = m.slot_tok[r + (lane & 15)];
            tok = tok < 0 ? 0 : tok;
            B[g] = m.B + (size_t)(tok >> 4) * KT * 1024 + (lane >> 4) * 256 + (tok & 15) * 16;
        } else {
            B[g] = m.B + (size_t)(r >> 4) * KT * 1024 + lane * 16;
        }
    }
    v4i acc[M][NB] = {};
#pragma unroll 4
    for (int k = w; k < KT; k += 4) {
        v4i a[M], b[NB];
#pragma unroll
        for (int j = 0; j < M; ++j)
            a[j] = *(const v4i *)(A[j] + (size_t)k * 1024);
#pragma unroll
        for (int g = 0; g < NB; ++g)
            b[g] = *(const v4i *)(B[g] + (size_t)k * 1024);
#pragma unroll
        for (int g = 0; g < NB; ++g)
#pragma unroll
            for (int j = 0; j < M; ++j)
                acc[j][g] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[j], b[g], acc[j][g], 0, 0, 0);
    }
    // lane l, register i: weight row 4 (l / 16) + i, row l % 16
    const int n = n0 + (tid & 15);
    const int64_t *sw = m.sw + (size_t)expert * m.N, *sw2 = m.sw2 + (size_t)expert * m.N;
    const bool in = n < m.N;
    const int64_t s1 = in ? sw[n] : 0, s2 = in && M == 2 ? sw2[n] : 0;
#pragma unroll
    for (int g = 0; g < NB; ++g) {
#pragma unroll
        for (int j = 0; j < M; ++j)
            *(v4i *)&red[j][w][(lane & 15) * 16 + 4 * (lane >> 4)] = acc[j][g];
        __syncthreads();
        const int r = 16 * g + (tid >> 4);
        if (in && r < rows) {
            int S[2] = {};
#pragma unroll
            for (int j = 0; j < M; ++j)
                S[j] = red[j][0][tid] + red[j][1][tid] + red[j][2][tid] + red[j][3][tid];
            const size_t row = (size_t)row0 + r;
            const int tok = EXPERTS ? m.slot_tok[row] : 0;
            if (tok >= 0) {
                const int64_t sb = m.sb[EXPERTS && EPI == 1 ? (size_t)tok : row];
                int64_t y = w8_scaled(S[0], sb, s1);
                if constexpr (EPI == 1)
                    y = q48_mul(q48_silu(y), w8_scaled(S[1], sb, s2));
                if constexpr (EPI == 2)
                    atomicAdd((unsigned long long *)m.Y + (size_t)tok * m.N + n,
                              (unsigned long long)q48_mul(m.slot_w[row], y));
                else
                    m.Y[row * m.N + n] =
                        (int64_t)((uint64_t)y +
                                  (EPI == 0 && m.base ? (uint64_t)m.base[row * m.N + n] : 0));
            }
        }
        __syncthreads();
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
    const size_t codes = w8_tiles(T, K);
    int rc = q48_w8_reserve(c, codes + (size_t)T * 8);
    if (rc)
        return rc;
    uint8_t *ws = (uint8_t *)c->w8;
    W8Rows r = {};
    r.codes = ws;
    r.step = (int64_t *)(ws + codes);
    r.X = X;
    r.norm_w = norm_w;
    r.T = T;
    r.K = K;
    if ((rc = q48_launch_w8_rows(c, r)))
        return launch_rc(rc);
    W8Mul m = {};
    m.A = (const uint8_t *)w->codes;
    m.sw = w->step;
    if (w2) {
        m.A2 = (const uint8_t *)w2->codes;
        m.sw2 = w2->step;
    }
    m.N = N;
    m.KT = w8_kt(K);
    m.B = r.codes;
    m.sb = r.step;
    m.T = T;
    m.Y = Y;
    m.base = base;
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
    return Q48_OK;
}

int q48_launch_w8_rows(q48_ctx *c, const W8Rows &r)
{
    hipLaunchKernelGGL(k_w8_rows, dim3(r.T), dim3(256), 0, c->stream, r);
    return (int)hipGetLastError();
}

int q48_launch_w8_mul(q48_ctx *c, const W8Mul &m, int epi, bool experts, int n_items)
{
    const unsigned nx = (m.N + 15) / 16;
#define W8_MUL(NB, EPI, EX)                                                            \
    hipLaunchKernelGGL((k_w8_mul<NB, EPI, EX>), dim3(nx, EX ? n_items : (m.T + 16 * NB - 1) / (16 * NB)), \
                       dim3(256), 0, c->stream, m)
    if (experts) {
        if (epi == 1)
            W8_MUL(1, 1, true);
        else
            W8_MUL(1, 2, true);
    } else if (epi == 1) {
        if (m.T <= 16)
            W8_MUL(1, 1, false);
        else
            W8_MUL(4, 1, false);
    } else if (m.T <= 16) {
        W8_MUL(1, 0, false);
    } else {
        W8_MUL(4, 0, false);
    }
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
    hipLaunchKernelGGL(k_w8_pack, dim3((N + 15) / 16 * 16), dim3(256), 0, c->stream, to, st, W,
                       codes, steps, N, K);
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
    hipLaunchKernelGGL(k_w8_values, dim3(N), dim3(256), 0, c->stream, out, from, st, N, K);
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
