// q48_rowattn.hip — exact attention over a quantised cache (single tokens, rows)
// and of masked rows over the int64 cache (trees of drafted tokens); the
// arithmetic is the reference's exact attention path (llama_int.c:1502-1529,
// softmax 1060-1072) on the values the cache stands for.
#include "q48_attn.hpp"
#include "q48_quant.hpp"

namespace {

constexpr int RA_MAX_POS = 32767;   // a softmax row's sum stays below 2^63

// The operands of one launch; k, v, ks, vs at the layer's row 0 (int64 words in
// k and v, and no steps, where the cache is not quantised).
struct RaArgs {
    int64_t *out;
    const int64_t *q;        // row t, head h: q + t ldq + h HD
    size_t ldq;
    const uint8_t *k, *v;
    const int64_t *ks, *vs;
    const uint64_t *mask;    // [T][words], or null: causal
    int64_t *ws;
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

// One block a (head, row).
template <int BITS, int HD, bool DEC>
__global__ __launch_bounds__(256) void k_ra_simple(RaArgs a)
{
    q48_round_down();
    __shared__ int64_t qs[HD], red[4], red2[4], part[256];
    const int h = blockIdx.x, t = blockIdx.y, tid = threadIdx.x;
    const int kh = h / (a.n_heads / a.n_kv);
    int p0 = a.p0;
    if (DEC) {
        if (a.d_pos)
            p0 = *a.d_pos;
        if (p0 < 0 || p0 >= a.max_seq)
            return;
    }
    const int S = p0 + (a.mask ? a.T : t + 1);
    const int64_t *q = a.q + (size_t)t * a.ldq + (size_t)h * HD;
    int64_t *sc = a.ws + ((size_t)t * a.n_heads + h) * a.max_seq;
    if (tid < HD / 2) {
        int64_t x0 = q[tid], x1 = q[tid + HD / 2];
        if (DEC && a.cos_t)
            q48_rope_pair(x0, x1, a.cos_t[(size_t)p0 * (HD / 2) + tid],
                          a.sin_t[(size_t)p0 * (HD / 2) + tid]);
        qs[tid] = x0;
        qs[tid + HD / 2] = x1;
    }
    __shared__ __align__(16) uint8_t nk[2][HD];
    __shared__ int64_t nst[2];
    if (DEC && BITS != 64 && tid < 32) {
        constexpr int N = HD / 32;
        const int l = tid & 15, i0 = l * N, isv = tid >> 4;
        const int64_t *x = (isv ? a.v_new : a.k_new) + (size_t)kh * HD;
        int64_t lo[N], hi[N];
        for (int i = 0; i < N; ++i) {
            lo[i] = x[i0 + i];
            hi[i] = x[i0 + i + HD / 2];
            if (a.cos_t && !isv)
                q48_rope_pair(lo[i], hi[i], a.cos_t[(size_t)p0 * (HD / 2) + i0 + i],
                              a.sin_t[(size_t)p0 * (HD / 2) + i0 + i]);
        }
        q48_quantise_row<BITS == 64 ? 8 : BITS, HD>(nk[isv], &nst[isv], l, lo, hi);
        if (h % (a.n_heads / a.n_kv) == 0) {
            const size_t row = (size_t)p0 * a.n_kv + kh;
            q48_quantise_row<BITS == 64 ? 8 : BITS, HD>(
                const_cast<uint8_t *>(isv ? a.v : a.k) + row * (HD * BITS / 8),
                const_cast<int64_t *>(isv ? a.vs : a.ks) + row, l, lo, hi);
        }
    }
    __syncthreads();
    auto sees = [&](int j) {
        return j < p0 || !a.mask ||
               (a.mask[(size_t)t * a.words + ((j - p0) >> 6)] >> ((j - p0) & 63) & 1);
    };
    int64_t mx = INT64_MIN;
    int any = 0;
    for (int j = tid; j < S; j += 256) {
        if (!sees(j))
            continue;
        any = 1;
        q48_u128 dot = 0;
        const size_t row = (size_t)j * a.n_kv + kh;
        for (int d = 0; d < HD; ++d) {
            const int64_t k = DEC && j == p0 ? value_at<BITS, HD>(nk[0], nst, 0, d)
                                             : value_at<BITS, HD>(a.k, a.ks, row, d);
            dot += (q48_u128)q48_smul128(qs[d], k);
        }
        const int64_t s = q48_mul((int64_t)((q48_i128)dot >> 48), a.scale);
        sc[j] = s;
        mx = s > mx ? s : mx;
    }
    any = __syncthreads_or(any);
    mx = block_max64<256>(mx, red);
    int64_t sum = 0;
    for (int j = tid; j < S; j += 256) {
        int64_t e = 0;
        if (sees(j))
            e = q48_safe_exp((int64_t)((uint64_t)sc[j] - (uint64_t)mx));
        sc[j] = e;
        sum = (int64_t)((uint64_t)sum + (uint64_t)e);
    }
    sum = block_sum64<256>(sum, red2);
    for (int j = tid; j < S; j += 256)
        if (sum > 0)
            sc[j] = q48_div(sc[j], sum);
    __syncthreads();
    constexpr int SL = 256 / HD;
    const int d = tid % HD, sl = tid / HD;
    uint64_t o = 0;
    if (any)
        for (int j = sl; j < S; j += SL) {
            const size_t row = (size_t)j * a.n_kv + kh;
            const int64_t v = DEC && j == p0 ? value_at<BITS, HD>(nk[1], nst + 1, 0, d)
                                             : value_at<BITS, HD>(a.v, a.vs, row, d);
            o += (uint64_t)q48_mul(sc[j], v);
        }
    part[tid] = (int64_t)o;
    __syncthreads();
    if (tid < HD) {
        for (int i = 1; i < SL; ++i)
            o += (uint64_t)part[tid + i * HD];
        a.out[((size_t)t * a.n_heads + h) * HD + tid] = (int64_t)o;
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

template <int BITS, bool DEC>
int launch(q48_ctx *c, RaArgs &a, int hd)
{
    int rc = q48_ws_reserve(c, (size_t)a.T * a.n_heads * a.max_seq * 8);
    if (rc)
        return rc;
    a.ws = (int64_t *)c->ws;
    a.scale = score_scale(hd);
    const dim3 grid(a.n_heads, a.T);
    if (hd == 32)
        hipLaunchKernelGGL((k_ra_simple<BITS, 32, DEC>), grid, dim3(256), 0, c->stream, a);
    else if (hd == 64)
        hipLaunchKernelGGL((k_ra_simple<BITS, 64, DEC>), grid, dim3(256), 0, c->stream, a);
    else
        hipLaunchKernelGGL((k_ra_simple<BITS, 128, DEC>), grid, dim3(256), 0, c->stream, a);
    return hipGetLastError() == hipSuccess ? Q48_OK : Q48_EHIP;
}

int decode_qcache(q48_ctx *c, int64_t *out, const int64_t *q, const q48_qcache *qc,
                  const int64_t *k_new, const int64_t *v_new, int layer, int pos, int n_heads,
                  bool rope)
{
    if (!c || !out || !q || !k_new || !v_new || !q48_qcache_ok(qc) || layer < 0 ||
        layer >= qc->layers || n_heads <= 0 || n_heads > 65535 || n_heads % qc->n_kv)
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
        n_heads <= 0 || n_heads > 65535 || n_heads % qc->n_kv)
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
        n_heads > 65535 || n_kv <= 0 || n_heads % n_kv || max_seq <= 0 ||
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
