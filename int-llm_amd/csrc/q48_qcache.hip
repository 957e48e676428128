// q48_qcache.hip — the quantised key/value cache: rows quantised as they are
// written (with RoPE, or already rotated), read back, and moved after a tree of
// drafted tokens has been verified (include/intllm_hip.h has the format).
#include "q48_quant.hpp"

namespace {

int launch_rc(int e) { return e == (int)hipSuccess ? Q48_OK : Q48_EHIP; }

// One layer's arrays at row 0, and the sizes a row needs.
struct QcLayer {
    uint8_t *k, *v;
    int64_t *ks, *vs;
    int n_kv;
};

QcLayer qc_layer(const q48_qcache *qc, int layer)
{
    const size_t rows = (size_t)layer * qc->max_seq * qc->n_kv;
    const size_t code = rows * ((size_t)qc->head_dim * qc->bits / 8);
    return {(uint8_t *)qc->k + code, (uint8_t *)qc->v + code, qc->k_step + rows,
            qc->v_step + rows, qc->n_kv};
}

// 16 lanes a head vector, 16 vectors a block, each read and written once; with ROPE the
// query heads too, in place.  Bound by HBM where there are rows: 1999 rows of 8 heads of
// 128 at 4 bits, 35 MB, in 8.4 us (4.2 TB/s; a large copy reaches 4.4); with RoPE 2000 rows
// of 32 heads on 4 of 64, 79 MB of them in cache, in 16.7 us, 512 in 5.6.  One row is a
// launch: 2 us.
template <int BITS, int HD, bool ROPE>
__global__ __launch_bounds__(256) void k_qc_store(QcLayer L, int64_t *K, int64_t *V, size_t ld,
                                                 int64_t *Q, int nq, int p0, size_t vectors,
                                                 const int *__restrict__ d_pos,
                                                 const int64_t *__restrict__ cos_t,
                                                 const int64_t *__restrict__ sin_t, int n_pos)
{
    q48_round_down();
    constexpr int N = HD / 32;   // pairs (i, i + HD / 2) a lane holds
    const size_t idx = (size_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    if (idx >= vectors)   // whole rows of 16 lanes
        return;
    const int l = threadIdx.x & 15, i0 = l * N;
    const int per = nq + 2 * L.n_kv, u = (int)(idx % per), t = (int)(idx / per);
    const bool is_q = u < nq, is_v = u >= nq + L.n_kv;
    const int kh = is_q ? u : (u - nq) % L.n_kv;
    int64_t *x = (is_q ? Q : is_v ? V : K) + (size_t)t * ld + (size_t)kh * HD;
    int64_t lo[N], hi[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        lo[i] = x[i0 + i];
        hi[i] = x[i0 + i + HD / 2];
    }
    if constexpr (ROPE) {
        const int pos = d_pos ? d_pos[t] : p0 + t;
        if (pos < 0 || pos >= n_pos)
            return;
        if (!is_v)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int64_t c = cos_t[(size_t)pos * (HD / 2) + i0 + i];
                const int64_t s = sin_t[(size_t)pos * (HD / 2) + i0 + i];
                q48_rope_pair(lo[i], hi[i], c, s);
                x[i0 + i] = lo[i];
                x[i0 + i + HD / 2] = hi[i];
            }
        if (is_q)
            return;
    }
    const size_t row = (size_t)(p0 + t) * L.n_kv + kh;
    q48_quantise_row<BITS, HD>((is_v ? L.v : L.k) + row * (HD * BITS / 8),
                               (is_v ? L.vs : L.ks) + row, l, lo, hi);
}

// The way back, the same lanes and bytes: 9.2 us (3.8 TB/s).
template <int BITS, int HD>
__global__ __launch_bounds__(256) void k_qc_load(int64_t *__restrict__ K, int64_t *__restrict__ V,
                                                QcLayer L, int p0, size_t ld, size_t vectors)
{
    constexpr int N = HD / 32;
    const size_t idx = (size_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    if (idx >= vectors)
        return;
    const int i0 = (threadIdx.x & 15) * N;
    const int u = (int)(idx % (2 * L.n_kv)), t = (int)(idx / (2 * L.n_kv));
    const bool is_v = u >= L.n_kv;
    const int kh = is_v ? u - L.n_kv : u;
    const size_t row = (size_t)(p0 + t) * L.n_kv + kh;
    const uint8_t *code = (is_v ? L.v : L.k) + row * (HD * BITS / 8);
    const uint64_t step = (uint64_t)(is_v ? L.vs : L.ks)[row];
    int64_t *x = (is_v ? V : K) + (size_t)t * ld + (size_t)kh * HD;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        int a, b;
        if (BITS == 8) {
            a = (int8_t)code[i0 + i];
            b = (int8_t)code[i0 + i + HD / 2];
        } else {
            b = (int8_t)code[i0 + i];
            a = (b << 28) >> 28;
            b >>= 4;
        }
        x[i0 + i] = (int64_t)((uint64_t)(int64_t)a * step);
        x[i0 + i + HD / 2] = (int64_t)((uint64_t)(int64_t)b * step);
    }
}

// Up to four arrays of rows of 8-byte words, [layers][max_seq][words].
struct KeepArrays {
    uint64_t *p[4];
    int words[4];
};

// One thread a word of a row: the n moves in turn, so that a row that is both
// source and target is read before it is written (every later source lies past
// the rows written so far).  The moves of a word wait for one another: a path of a
// drafted tree is a few rows, and all layers move at once (22 layers of 4 heads of 64: 1 to
// 5 rows 3.2 us a call, a launch; 16 rows 4.2).
__global__ __launch_bounds__(256) void k_keep_rows(KeepArrays a, int max_seq, int p0,
                                                  const int *__restrict__ rows, int n)
{
    const int w = blockIdx.x * 256 + threadIdx.x, words = a.words[blockIdx.z];
    if (w >= words)
        return;
    uint64_t *base = a.p[blockIdx.z] + (size_t)blockIdx.y * max_seq * words + w;
    for (int i = 0; i < n; ++i) {
        const int r = rows[i];
        if (r > i && r < max_seq - p0)
            base[(size_t)(p0 + i) * words] = base[(size_t)(p0 + r) * words];
    }
}

} // namespace

bool q48_qcache_ok(const q48_qcache *qc)
{
    return qc && qc->k && qc->v && qc->k_step && qc->v_step && (qc->bits == 8 || qc->bits == 4) &&
           ((uintptr_t)qc->k & 15) == 0 && ((uintptr_t)qc->v & 15) == 0 &&
           ((uintptr_t)qc->k_step & 7) == 0 && ((uintptr_t)qc->v_step & 7) == 0 &&
           qc->layers > 0 && qc->layers <= 65535 && qc->max_seq > 0 && qc->max_seq <= 32767 && qc->n_kv > 0 &&
           qc->n_kv <= 65535 &&
           (qc->head_dim == 32 || qc->head_dim == 64 || qc->head_dim == 128);
}

#define QC_SHAPE(BITS_, HD_, CALL)        \
    do {                                  \
        if ((BITS_) == 8) {               \
            if ((HD_) == 32)              \
                CALL(8, 32);              \
            else if ((HD_) == 64)         \
                CALL(8, 64);              \
            else                          \
                CALL(8, 128);             \
        } else {                          \
            if ((HD_) == 32)              \
                CALL(4, 32);              \
            else if ((HD_) == 64)         \
                CALL(4, 64);              \
            else                          \
                CALL(4, 128);             \
        }                                 \
    } while (0)

int q48_launch_qcache_store(q48_ctx *c, const q48_qcache *qc, int layer, int p0, int T,
                            int64_t *K, int64_t *V, size_t ld, int64_t *Q, int n_heads,
                            const int *d_pos)
{
    const QcLayer L = qc_layer(qc, layer);
    const size_t vectors = (size_t)T * (n_heads + 2 * qc->n_kv);
    const dim3 grid((unsigned)((vectors + 15) / 16));
#define QC_STORE(B, H)                                                                         \
    do {                                                                                       \
        if (n_heads > 0)                                                                       \
            hipLaunchKernelGGL((k_qc_store<B, H, true>), grid, dim3(256), 0, c->stream, L, K,  \
                               V, ld, Q, n_heads, p0, vectors, d_pos, c->rope_cos,             \
                               c->rope_sin, c->rope_max_seq);                                  \
        else                                                                                   \
            hipLaunchKernelGGL((k_qc_store<B, H, false>), grid, dim3(256), 0, c->stream, L, K, \
                               V, ld, Q, 0, p0, vectors, nullptr, nullptr, nullptr, 0);        \
    } while (0)
    QC_SHAPE(qc->bits, qc->head_dim, QC_STORE);
#undef QC_STORE
    return (int)hipGetLastError();
}

extern "C" {

int q48_qcache_bytes(int bits, int layers, int max_seq, int n_kv, int head_dim, size_t *codes,
                     size_t *steps)
{
    alignas(16) static char some[16];
    const q48_qcache qc = {some, some, (int64_t *)some, (int64_t *)some, bits, layers, max_seq,
                           n_kv, head_dim};
    if (!codes || !steps || !q48_qcache_ok(&qc))
        return Q48_EINVAL;
    const size_t rows = (size_t)layers * max_seq * n_kv;
    *codes = rows * ((size_t)head_dim * bits / 8);
    *steps = rows * sizeof(int64_t);
    return Q48_OK;
}

int q48_qcache_store_rows(q48_ctx *c, const q48_qcache *qc, int layer, int p0, int T,
                          const int64_t *K, const int64_t *V, int ld)
{
    if (!c || !K || !V || q48_off_words<8>(K, V) || !q48_qcache_ok(qc) || layer < 0 ||
        layer >= qc->layers || T <= 0 || ld < qc->n_kv * qc->head_dim)
        return Q48_EINVAL;
    if (p0 < 0 || p0 >= qc->max_seq || T > qc->max_seq - p0)
        return Q48_ERANGE;
    q48_on_device on(c);
    return launch_rc(q48_launch_qcache_store(c, qc, layer, p0, T, const_cast<int64_t *>(K),
                                             const_cast<int64_t *>(V), (size_t)ld, nullptr, 0,
                                             nullptr));
}

int q48_qcache_load_rows(q48_ctx *c, int64_t *K, int64_t *V, const q48_qcache *qc, int layer,
                         int p0, int T, int ld)
{
    if (!c || !K || !V || q48_off_words<8>(K, V) || !q48_qcache_ok(qc) || layer < 0 ||
        layer >= qc->layers || T <= 0 || ld < qc->n_kv * qc->head_dim)
        return Q48_EINVAL;
    if (p0 < 0 || p0 >= qc->max_seq || T > qc->max_seq - p0)
        return Q48_ERANGE;
    q48_on_device on(c);
    const QcLayer L = qc_layer(qc, layer);
    const size_t vectors = (size_t)T * 2 * qc->n_kv;
    const dim3 grid((unsigned)((vectors + 15) / 16));
#define QC_LOAD(B, H)                                                                          \
    hipLaunchKernelGGL((k_qc_load<B, H>), grid, dim3(256), 0, c->stream, K, V, L, p0,          \
                       (size_t)ld, vectors)
    QC_SHAPE(qc->bits, qc->head_dim, QC_LOAD);
#undef QC_LOAD
    return launch_rc((int)hipGetLastError());
}

int q48_rope_store_rows_qcache(q48_ctx *c, int64_t *QKV, const q48_qcache *qc, int layer, int p0,
                               int T, const int *d_pos, int n_heads)
{
    if (!c || !QKV || q48_off_words<8>(QKV) || q48_off_words<4>(d_pos) || !q48_qcache_ok(qc) ||
        layer < 0 || layer >= qc->layers || T <= 0 || n_heads <= 0 || n_heads > 1024 ||
        n_heads % qc->n_kv)
        return Q48_EINVAL;
    if (!c->rope_cos || qc->head_dim != c->rope_head_dim || qc->max_seq > c->rope_max_seq)
        return Q48_ESTATE;
    if (p0 < 0 || p0 >= qc->max_seq || T > qc->max_seq - p0)
        return Q48_ERANGE;
    q48_on_device on(c);
    const size_t hd = qc->head_dim;
    int64_t *K = QKV + n_heads * hd, *V = K + qc->n_kv * hd;
    return launch_rc(q48_launch_qcache_store(c, qc, layer, p0, T, K, V,
                                             (size_t)(n_heads + 2 * qc->n_kv) * hd, QKV, n_heads,
                                             d_pos));
}

int q48_cache_keep_rows(q48_ctx *c, int64_t *kcache, int64_t *vcache, int layers, int p0,
                        const int *d_rows, int n, int n_kv, int head_dim, int max_seq)
{
    if (!c || !kcache || !vcache || q48_off_words<8>(kcache, vcache) || !d_rows ||
        q48_off_words<4>(d_rows) || layers <= 0 || layers > 65535 || n <= 0 ||
        n_kv <= 0 || n_kv > 65535 || head_dim <= 0 || head_dim > 256 || max_seq <= 0)
        return Q48_EINVAL;
    if (p0 < 0 || p0 >= max_seq || n > max_seq - p0)
        return Q48_ERANGE;
    q48_on_device on(c);
    const int w = n_kv * head_dim;
    const KeepArrays a = {{(uint64_t *)kcache, (uint64_t *)vcache, nullptr, nullptr}, {w, w, 0, 0}};
    hipLaunchKernelGGL(k_keep_rows, dim3((w + 255) / 256, layers, 2), dim3(256), 0, c->stream, a,
                       max_seq, p0, d_rows, n);
    return launch_rc((int)hipGetLastError());
}

int q48_qcache_keep_rows(q48_ctx *c, const q48_qcache *qc, int p0, const int *d_rows, int n)
{
    if (!c || !d_rows || q48_off_words<4>(d_rows) || !q48_qcache_ok(qc) || n <= 0)
        return Q48_EINVAL;
    if (p0 < 0 || p0 >= qc->max_seq || n > qc->max_seq - p0)
        return Q48_ERANGE;
    q48_on_device on(c);
    const int w = qc->n_kv * (qc->head_dim * qc->bits / 64), s = qc->n_kv;   // 8-byte words
    const KeepArrays a = {{(uint64_t *)qc->k, (uint64_t *)qc->v, (uint64_t *)qc->k_step,
                           (uint64_t *)qc->v_step},
                          {w, w, s, s}};
    hipLaunchKernelGGL(k_keep_rows, dim3(((w > s ? w : s) + 255) / 256, qc->layers, 4), dim3(256),
                       0, c->stream, a, qc->max_seq, p0, d_rows, n);
    return launch_rc((int)hipGetLastError());
}

} // extern "C"
