// q48_logprob.hip — log probabilities of given tokens, the entropy and the most
// probable tokens of rows of logits (q48_logprobs_rows; include/intllm_hip.h has
// the integer steps).
//
// e^-u over the whole range: u = n LN2 + j / 64 + s splits the exponent into a
// shift, a table and a six-step Horner row on s < 2^-6 (s^7 / 5040 < 2^-54), a
// third of fp_exp's squarings and division, and 4 units of 2^-48 from e^-u.
#include "q48_attn.hpp"
#include "q48_expn.hpp"

namespace {

constexpr int64_t LP_LN2 = EXPN_LN2;
constexpr int LP_MAX_TOP = 32;
constexpr int LP_MAX_ROWS = 1 << 30;   // a row's number and a grid's stride add up in 31 bits
constexpr int LP_CAP = 512;   // candidates of a row; past that (ties) the slow selection

// floor(2^54 / (64 + j)), round(2^48 log(1 + j/64)), round(2^48 / (k + 1))
static __constant__ int64_t kRcp[64] = {
    281474976710656LL, 277144592453568LL, 272945431961848LL, 268871619544507LL, 264917625139440LL,
    261078239267854LL, 257348550135456LL, 253723922668760LL, 250199979298360LL, 246772582321671LL,
    243437817695702LL, 240191980126426LL, 237031559335289LL, 233953227395869LL, 230953827044640LL,
    228030360879518LL, 225179981368524LL, 222399981598543LL, 219687786700999LL, 217040945897373LL,
    214457125112880LL, 211934100111552LL, 209469750110255LL, 207062051833126LL, 204709073971386LL,
    202408972016651LL, 200159983438688LL, 197960423181120LL, 195808679450891LL, 193703209779376LL,
    191642537334914LL, 189625247468231LL, 187649984473770LL, 185715448551360LL, 183820392953897LL,
    181963621307898LL, 180143985094819LL, 178360381281999LL, 176611750092960LL, 174897072907592LL,
    173215370283480LL, 171565700090304LL, 169947155749830LL, 168358864574597LL, 166799986198907LL,
    165269711096164LL, 163767259177108LL, 162291878463801LL, 160842843834660LL, 159419455836123LL,
    158021039556859LL, 156646943560712LL, 155296538874844LL, 153969218029760LL, 152664394148152LL,
    151381500079680LL, 150119987579016LL, 148879326524644LL, 147659004176081LL, 146458524467333LL,
    145277407334532LL, 144115188075855LL, 142971416741920LL, 141845657554976LL};
static __constant__ int64_t kLog[64] = {
    0LL, 4364040544128LL, 8661451906573LL, 12894238087534LL, 17064314013873LL, 21173510740946LL,
    25223580280171LL, 29216200084181LL, 33152977218291LL, 37035452244253LL, 40865102839786LL,
    44643347175162LL, 48371547066152LL, 52051010920882LL, 55682996496557LL, 59268713480576LL,
    62809325909300LL, 66305954436582LL, 69759678463100LL, 73171538136644LL, 76542536232600LL,
    79873639923174LL, 83165782443125LL, 86419864659224LL, 89636756550011LL, 92817298601953LL,
    95962303127591LL, 99072555510867LL, 102148815384384LL, 105191817743039LL, 108202273998089LL,
    111180872975452LL, 114128281861729LL, 117045147101217LL, 119932095246910LL, 122789733768302LL,
    125618651818601LL, 128419420963759LL, 131192595875603LL, 133938714991134LL, 136658301139996LL,
    139351862141900LL, 142019891375752LL, 144662868322042LL, 147281259080020LL, 149875516861029LL,
    152446082459311LL, 154993384701515LL, 157517840876039LL, 160019857143290LL, 162499828927881LL,
    164958141293684LL, 167395169302662LL, 169811278358287LL, 172206824534353LL, 174582154889912LL,
    176937607771029LL, 179273513100022LL, 181590192652790LL, 183887960324830LL, 186167122386477LL,
    188427977727901LL, 190670818094329LL, 192895928311988LL};
constexpr int64_t kInvK[8] = {
    281474976710656LL, 140737488355328LL, 93824992236885LL, 70368744177664LL, 56294995342131LL,
    46912496118443LL, 40210710958665LL, 35184372088832LL};

// T_j 2^-48 as doubles, and the logarithm's tables, into LDS
__device__ __forceinline__ void lp_table(double *tab, int64_t *rcps, int64_t *logs, int tid)
{
    if (tid < 45)
        tab[tid] = (double)kExp[tid] * 0x1p-48;
    if (tid < 64) {
        rcps[tid] = kRcp[tid];
        logs[tid] = kLog[tid];
    }
}

// e of each u (include/intllm_hip.h; 0 from LP_LIM on), added to z, and floor(e u
// 2^-48) added to w.  FP64 rounds down, so with M = 2^52 a truncated product of
// integers below 2^49 is one fused operation, fma(a, b 2^-48, M) = M + floor(a b
// 2^-48), and a Horner step two: the next h = (C_k + M) - that, exact.  u = q 2^52 +
// u0 (q <= 2) keeps every double an exact integer where u passes 2^53: r = (q 2^52 -
// n LN2) + u0.  1 / LN2 is rounded down, so n is the quotient or one less.  About 55
// operations and no branch; N terms step by step, since one is a chain of them all.
constexpr uint64_t LP_LIM = 49 * (uint64_t)LP_LN2;   // 2^53.1
template <int N>
__device__ __forceinline__ void lp_terms(const uint64_t (&u)[N], const double *tab, uint64_t &z,
                                         uint64_t &w)
{
    constexpr double ln2 = (double)LP_LN2, inv = 0x1.7154765200000p-48;
    static_assert(inv * ln2 < 1.0 && inv * ln2 > 1.0 - 0x1p-24, "1 / LN2, rounded down");
    bool in[N], more[N];
    uint32_t q[N], n[N];
    double u0[N], top[N], tn[N], r[N], tj[N], s[N], h[N], tt[N];
#define LP_EACH for (int i = 0; i < N; ++i)
#pragma unroll
    LP_EACH
    {
        in[i] = u[i] < LP_LIM;
        const uint32_t hi = in[i] ? (uint32_t)(u[i] >> 32) : 0;
        q[i] = hi >> 20;
        u0[i] = __builtin_bit_cast(double, ((uint64_t)((hi & 0xFFFFFu) | 0x43300000u) << 32) |
                                               (uint32_t)u[i]) -
                0x1p52;
    }
#pragma unroll
    LP_EACH top[i] = __builtin_ldexp((double)q[i], 52);
#pragma unroll
    LP_EACH tn[i] = __builtin_fma(u0[i] + top[i], inv, 0x1p52);
#pragma unroll
    LP_EACH
    {
        n[i] = (uint32_t)__builtin_bit_cast(uint64_t, tn[i]);
        r[i] = __builtin_fma(-(tn[i] - 0x1p52), ln2, top[i]) + u0[i];
    }
#pragma unroll
    LP_EACH
    {
        more[i] = r[i] >= ln2;
        n[i] += more[i];
        r[i] = more[i] ? r[i] - ln2 : r[i];
    }
#pragma unroll
    LP_EACH tj[i] = __builtin_fma(r[i], 0x1p-42, 0x1p52);
#pragma unroll
    LP_EACH
    {
        tt[i] = tab[(uint32_t)__builtin_bit_cast(uint64_t, tj[i]) & 63];
        s[i] = __builtin_fma(tj[i] - 0x1p52, -0x1p-6, r[i] * 0x1p-48);   // s 2^-48
        h[i] = (double)kFactK[6];
    }
#pragma unroll
    for (int k = 5; k >= 0; --k)
#pragma unroll
        LP_EACH h[i] = ((double)kFactK[k] + 0x1p52) - __builtin_fma(s[i], h[i], 0x1p52);
#pragma unroll
    LP_EACH
    {
        const uint64_t e = q48_word_m52(__builtin_fma(tt[i], h[i], 0x1p52)) >> (in[i] ? n[i] : 63);
        const double ed = __builtin_bit_cast(double, e | 0x4330000000000000ull) - 0x1p52;
        z += e;
        // e 2^4 q: e is below 2^27 where q is not 0
        w += q48_word_m52(__builtin_fma(ed, u0[i] * 0x1p-48, 0x1p52)) +
             (uint64_t)(uint32_t)e * (16 * q[i]);
    }
#undef LP_EACH
}

// logZ of Z >= 2^48, and its b; the Horner steps as in lp_terms, around 1.5 2^52 since
// d may be a unit or two below 0
__device__ __forceinline__ int64_t lp_log(q48_u128 Z, int &b, const int64_t *rcps,
                                          const int64_t *logs)
{
    const uint64_t zh = (uint64_t)(Z >> 64), zl = (uint64_t)Z;
    b = (zh ? 128 - __builtin_clzll(zh) : 64 - __builtin_clzll(zl)) - 49;
    const int64_t z = (int64_t)(Z >> b);
    const int j = (int)(z >> 42) - 64;
    const int64_t rcp = rcps[j], l = logs[j];
    const double M = 0x1.8p52, d = (double)(q48_mul(z, rcp) - Q48_ONE) * 0x1p-48;
    double g = (double)kInvK[7];
#pragma unroll
    for (int k = 6; k >= 0; --k)
        g = ((double)kInvK[k] + M) - __builtin_fma(d, g, M);
    const int64_t log1p = __builtin_bit_cast(int64_t, __builtin_fma(d, g, M)) -
                          __builtin_bit_cast(int64_t, M);
    return b * LP_LN2 + l + log1p;
}

__device__ __forceinline__ int64_t lp_value(uint64_t u, int64_t logz)
{
    const uint64_t v = u + (uint64_t)logz;
    return v < u || v > (uint64_t)INT64_MAX ? INT64_MIN : -(int64_t)v;
}

// A value's order as an unsigned word, and its high half: what the selection of
// the most probable tokens compares first.
__device__ __forceinline__ uint32_t lp_high(int64_t x)
{
    return (uint32_t)((uint64_t)x >> 32) ^ 0x80000000u;
}

// A threshold that n of the high halves g[0 .. N - 1] of a wave's lanes (64 N >= n)
// reach, most often no more: from the top, two bits at a time, until n are left.  n of
// the groups whose maxima these are have a value at least that large, so the n largest
// values of the row are among the values whose high halves are not below it.  high: the
// largest of all; the bits above the first in which a maximum but 0 (no value) differs
// from it are taken as they are.  A step is 3 N compares and counts, 140 ns for N = 4:
// all 16 took 2.3 us of a single row's 12.
template <int N>
__device__ __forceinline__ uint32_t lp_threshold(const uint32_t (&g)[N], uint32_t high, int n)
{
    uint32_t low = high;
#pragma unroll
    for (int i = 0; i < N; ++i)
        low = min(low, g[i] ? g[i] : high);
    low = min(low, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)low, Q48_DPP_XOR1, 0xf, 0xf, false));
    low = min(low, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)low, Q48_DPP_XOR2, 0xf, 0xf, false));
    low = min(low, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)low, Q48_DPP_HALF_MIRROR, 0xf, 0xf,
                                                         false));
    low = min(low, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)low, Q48_DPP_MIRROR, 0xf, 0xf,
                                                         false));
    uint32_t differ = 0;
#pragma unroll
    for (int row = 0; row < 64; row += 16)
        differ |= (uint32_t)__builtin_amdgcn_readlane((int)low, row) ^ high;
    int bit = differ ? 31 - __builtin_clz(differ) : 0;
    bit &= ~1;
    auto reach = [&](uint32_t t) {
        int c = 0;
#pragma unroll
        for (int i = 0; i < N; ++i)
            c += __popcll(__ballot(g[i] >= t));
        return c;
    };
    uint32_t t = (high >> bit >> 2) << bit << 2;
    int have = reach(t);
    if (have < n) {   // some of the n groups have no value
        t = 0;
        bit = 30;
    }
    for (; bit >= 0 && have != n; bit -= 2) {
        int count[3];
#pragma unroll
        for (int c = 0; c < 3; ++c)
            count[c] = reach(t | ((uint32_t)(c + 1) << bit));
        const int d = (count[0] >= n) + (count[1] >= n) + (count[2] >= n);
        t |= (uint32_t)d << bit;
        have = d == 3 ? count[2] : d == 2 ? count[1] : d == 1 ? count[0] : have;
    }
    return t;
}

template <bool AGENT>
__device__ __forceinline__ void lp_put(int64_t *cv, int *ci, int at, int64_t y, int i)
{
    if (AGENT) {
        __hip_atomic_store(cv + at, y, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(ci + at, i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    } else {
        cv[at] = y;
        ci[at] = i;
    }
}

// The candidates (high half >= thr) among the values first + k stride < end of the
// threads whose maximum is one, appended to cv and ci: the wave reads such a thread's
// values together, 64 at a time.
template <bool AGENT>
__device__ __forceinline__ void lp_collect(const int64_t *x, int first, int stride, int end,
                                           bool some, uint32_t thr, int64_t *cv, int *ci,
                                           int *count, int cap, int lane)
{
    uint64_t todo = __ballot(some);
    while (todo) {
        const int l = __builtin_ctzll(todo);
        todo &= todo - 1;
        for (int i = __builtin_amdgcn_readlane(first, l) + lane * stride; i < end;
             i += 64 * stride) {
            const int64_t y = x[i];
            if (lp_high(y) >= thr) {
                const int at = atomicAdd(count, 1);
                if (at < cap)
                    lp_put<AGENT>(cv, ci, at, y, i);
            }
        }
    }
}

// The token of a row and its logit, loaded ahead of the sums they are used with.
struct LpToken {
    bool valid;
    int64_t y;
    __device__ __forceinline__ LpToken(const int64_t *x, int V, const int *tokens, bool wanted, int t)
    {
        const int id = wanted ? tokens[t] : -1;
        valid = id >= 0 && id < V;
        y = valid ? x[id] : 0;
    }
};

// The row's log probability and entropy from its sums z and w; returns logZ.  rcps, logs:
// the logarithm's tables.
__device__ __forceinline__ int64_t lp_finish(q48_u128 z, q48_u128 w, int64_t m, LpToken k, int t,
                                             const int64_t *rcps, const int64_t *logs,
                                             int64_t *logp, int64_t *entropy, bool writer)
{
    int b;
    const int64_t logz = lp_log(z, b, rcps, logs);
    if (writer) {
        if (logp)
            logp[t] = k.valid ? lp_value((uint64_t)m - (uint64_t)k.y, logz) : 0;
        if (entropy)
            entropy[t] = logz + q48_div((int64_t)(w >> b), (int64_t)(z >> b));
    }
    return logz;
}


// How many of the candidates cv, ci [0, count) come before the candidate v, id, eight
// at a time (the arrays hold LP_CAP + 8: what lies past count is not counted).
__device__ __forceinline__ int lp_before(const int64_t *cv, const int *ci, int count, int64_t v,
                                         int id)
{
    int rank = 0;
    for (int k = 0; k < count; k += 8)
#pragma unroll
        for (int i = 0; i < 8; ++i)
            rank += (k + i < count) & ((cv[k + i] > v) | ((cv[k + i] == v) & (ci[k + i] < id)));
    return rank;
}

__device__ __forceinline__ void lp_place(int rank, int64_t v, int id, int64_t m, int64_t logz, int t,
                                         int top, int *ids, int64_t *tlp)
{
    if (rank < top) {
        ids[(size_t)t * top + rank] = id;
        tlp[(size_t)t * top + rank] = lp_value((uint64_t)m - (uint64_t)v, logz);
    }
}

// The top values of a row from its candidates.  count <= LP_CAP.
template <int NT>
__device__ __forceinline__ void lp_rank(const int64_t *cv, const int *ci, int count, int64_t m,
                                        int64_t logz, int t, int top, int *ids, int64_t *tlp,
                                        int tid)
{
    for (int i = tid; i < count; i += NT)
        lp_place(lp_before(cv, ci, count, cv[i], ci[i]), cv[i], ci[i], m, logz, t, top, ids, tlp);
}

// The same by top passes over the row, for rows with more candidates: the largest
// value after the last one in the order (value, lowest id).
template <int NT>
__device__ void lp_select(const int64_t *x, int V, int64_t m, int64_t logz, int t, int top,
                          int *ids, int64_t *tlp, int tid, int64_t *bv, int *bi)
{
    int64_t lv = INT64_MAX;
    int li = -1;
    for (int n = 0; n < top; ++n) {
        int64_t v = INT64_MIN;
        int at = INT_MAX;
        for (int i = tid; i < V; i += NT)
            if ((x[i] < lv || (x[i] == lv && i > li)) && (at == INT_MAX || x[i] > v)) {
                v = x[i];
                at = i;
            }
        for (int o = 32; o; o >>= 1) {
            const int64_t ov = __shfl_xor(v, o);
            const int oi = __shfl_xor(at, o);
            if (oi != INT_MAX && (at == INT_MAX || ov > v || (ov == v && oi < at))) {
                v = ov;
                at = oi;
            }
        }
        __syncthreads();
        if ((tid & 63) == 0) {
            bv[tid >> 6] = v;
            bi[tid >> 6] = at;
        }
        __syncthreads();
        v = bv[0];
        at = bi[0];
        for (int i = 1; i < NT / 64; ++i)
            if (bi[i] != INT_MAX && (at == INT_MAX || bv[i] > v || (bv[i] == v && bi[i] < at))) {
                v = bv[i];
                at = bi[i];
            }
        lv = v;
        li = at;
        if (tid == 0) {
            ids[(size_t)t * top + n] = at;
            tlp[(size_t)t * top + n] = lp_value((uint64_t)m - (uint64_t)v, logz);
        }
    }
}

__device__ __forceinline__ void agent_store(uint64_t *p, uint64_t v)
{
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename T>
__device__ __forceinline__ T agent_load(const T *p)
{
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Sums of z and w over a wave, in exact 128 bits, as four words (lanes 0 to 3).
template <bool AGENT>
__device__ __forceinline__ void lp_wave_sums(uint64_t z64, uint64_t w64, uint64_t *s, int lane)
{
    const q48_u128 z = q48_wave_sum128(z64), w = q48_wave_sum128(w64);
    const q48_u128 v = lane & 2 ? w : z;
    const uint64_t word = (uint64_t)(lane & 1 ? v >> 64 : v);
    if (lane < 4) {
        if (AGENT)
            agent_store(s + lane, word);
        else
            s[lane] = word;
    }
}

// A row of logits through a buffer descriptor: loads past its end give 0 and need no
// branch.  (The whole offset goes where the bounds check sees it: not into the scalar
// offset, which it leaves out.)
struct LpRow {
    __amdgpu_buffer_rsrc_t d;
    __device__ __forceinline__ LpRow(const int64_t *x, int V)
        : d(__builtin_amdgcn_make_buffer_rsrc(const_cast<int64_t *>(x), 0, V * 8, 0x00027000))
    {
    }
    __device__ __forceinline__ int64_t at(int i) const
    {
        return __builtin_bit_cast(int64_t, __builtin_amdgcn_raw_buffer_load_b64(d, 8 * i, 0, 0));
    }
};

constexpr int LR_NT = 512;

// Rows of up to 512 R logits, a block a row at a time (row blockIdx.x, + gridDim.x,
// ...): a row stays in registers between the maximum and the exponentials, so it is
// read once, and the next row's loads go out as its registers fall free, under the
// remaining exponentials.  Groups of 4 threads keep their maxima for the threshold,
// which wave 0 finds before its exponentials; the few threads with a candidate read
// their logits again.
// Bound by vector issue: 500 rows of 32000, 16 M terms of about 60 operations, in 51 us
// (2.5 TB/s of logits), 70% of what issue allows; two rows a block, and a row's 4 us of
// maximum, threshold, logarithm and candidates are not covered by another's terms.
template <int R>
__global__ __launch_bounds__(LR_NT) void k_lp_row(const int64_t *__restrict__ X, int T, int V,
                                                 const int *__restrict__ tokens,
                                                 int64_t *__restrict__ logp,
                                                 int64_t *__restrict__ entropy, int top,
                                                 int *__restrict__ ids, int64_t *__restrict__ tlp)
{
    q48_round_down();
    constexpr int NW = LR_NT / 64;
    __shared__ double tab[64];
    __shared__ int64_t red[2][NW];
    __shared__ uint32_t gmax[LR_NT / 4];
    __shared__ uint64_t sums[NW][4];
    __shared__ int64_t cv[LP_CAP + 8], slogz, rcps[64], logs[64];
    __shared__ int ci[LP_CAP + 8];
    __shared__ int count;
    __shared__ uint32_t thr;
    const int tid = threadIdx.x, lane = tid & 63;
    const int whole = V / LR_NT;   // tiles of 512 with every thread in the row
    lp_table(tab, rcps, logs, tid);
    int64_t v[R];
    {
        const LpRow row(X + (size_t)blockIdx.x * V, V);
#pragma unroll
        for (int k = 0; k < R; ++k)
            v[k] = row.at(k * LR_NT + tid);
    }
    int par = 0;
    for (int t = blockIdx.x; t < T; t += gridDim.x, par ^= 1) {
        const int64_t *x = X + (size_t)t * V;
        int64_t m = INT64_MIN;
#pragma unroll
        for (int k = 0; k < R; ++k) {
            int64_t y = v[k];
            if (k >= whole)
                y = k * LR_NT + tid < V ? y : INT64_MIN;
            m = y > m ? y : m;
        }
        const uint32_t mine = lp_high(m);
        if (top) {
            // the maximum of 4 lanes' high halves; 0, below every value, where none has one
            uint32_t g = tid < V ? mine : 0;
            g = max(g, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)g, Q48_DPP_XOR1, 0xf, 0xf,
                                                             false));
            g = max(g, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)g, Q48_DPP_XOR2, 0xf, 0xf,
                                                             false));
            if ((tid & 3) == 0)
                gmax[tid >> 2] = g;
        }
        if (tid == 0)
            count = 0;
        m = block_max64<LR_NT>(m, red[par], false);
        if (top && tid < 64) {
            const uint32_t g[2] = {gmax[tid], gmax[tid + 64]};
            const uint32_t h = lp_threshold<2>(
                g, (uint32_t)__builtin_amdgcn_readfirstlane((int)lp_high(m)), top);
            if (tid == 0)
                thr = h;
        }
        // (a block's last row: a row of no logits, nothing is read)
        const bool again = t + gridDim.x < (unsigned)T;
        const LpRow next(again ? x + (size_t)gridDim.x * V : x, again ? V : 0);
        LpToken token(x, V, tokens, logp != nullptr, t);
        uint64_t z64 = 0, w64 = 0;   // R terms below 2^49 each
#pragma unroll
        for (int k = 0; k < R; k += 4) {
            uint64_t u[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                u[i] = (uint64_t)m - (uint64_t)v[k + i];
                if (k + i >= whole)
                    u[i] = (k + i) * LR_NT + tid < V ? u[i] : LP_LIM;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                v[k + i] = next.at((k + i) * LR_NT + tid);
            lp_terms<4>(u, tab, z64, w64);
            __builtin_amdgcn_sched_barrier(0);   // more terms would not fit the registers
        }
        asm volatile("" : "+v"(token.y));   // (loaded by now: not after the sums)
        lp_wave_sums<false>(z64, w64, sums[tid >> 6], lane);
        __syncthreads();
        if (tid < 64) {
            q48_u128 z = 0, w = 0;
            for (int i = 0; i < NW; ++i) {
                z += ((q48_u128)sums[i][1] << 64) | sums[i][0];
                w += ((q48_u128)sums[i][3] << 64) | sums[i][2];
            }
            const int64_t logz =
                lp_finish(z, w, m, token, t, rcps, logs, logp, entropy, tid == 0);
            if (tid == 0)
                slogz = logz;
        }
        if (!top)
            continue;   // (the next row's first barrier is behind its reads of v alone)
        lp_collect<false>(x, tid, LR_NT, V, tid < V && mine >= thr, thr, cv, ci, &count, LP_CAP, lane);
        __syncthreads();
        if (count <= LP_CAP)
            lp_rank<LR_NT>(cv, ci, count, m, slogz, t, top, ids, tlp, tid);
        else
            lp_select<LR_NT>(x, V, m, slogz, t, top, ids, tlp, tid, red[par],
                             reinterpret_cast<int *>(sums));
        __syncthreads();
    }
}

// ---- a row over many blocks ------------------------------------------------------------
// Two launches of (chunk, row) blocks, at most 64 chunks a row: the chunks' wave
// maxima; then sums and candidates, which go out with agent-coherent stores ahead of
// a ticket, and the row's last block makes its results (no block waits on another).
// One row of 32000 with its 20 most probable tokens: 2 + 8.5 us, all latencies: of the
// second launch 1.0 the maxima, 1.6 the threshold, 0.6 the terms, 1.5 the candidates on
// their way out, 0.5 the ticket, 2.3 the sums of all waves (1.3 to fetch them from other
// dies) and the logarithm.
// A chunk is one stretch of the row: where the largest logits sit in few chunks (a row in
// order, or all but a block of ids masked), more candidates come than LP_CAP and the last
// block passes over the row for each token asked for: 545 us with a top 20, 64 rows of 130000
// 4.4 ms instead of 41 us.

struct LpWork {
    int64_t *gmax;     // [T][4 chunks]: a wave's maximum
    uint64_t *sums;    // [T][4 chunks][4]: a wave's z and w, 128 bits each
    int *count;        // [T][2]: candidates, tickets
    int64_t *cv;       // [T][LP_CAP]
    int *ci;           // [T][LP_CAP]
    int chunks, ch;    // ch: values a chunk, a multiple of 256
};

__global__ __launch_bounds__(256) void k_lp_max(const int64_t *__restrict__ X, int V, LpWork p)
{
    const int t = blockIdx.y, c = blockIdx.x, tid = threadIdx.x;
    const int64_t *x = X + (size_t)t * V;
    const int end = min(V, (c + 1) * p.ch);
    int64_t m = INT64_MIN;
#pragma unroll 4
    for (int i = c * p.ch + tid; i < end; i += 256)
        m = x[i] > m ? x[i] : m;
    m = q48_wave_max64(m);
    if ((tid & 63) == 0)
        p.gmax[(size_t)t * 4 * p.chunks + 4 * c + (tid >> 6)] = m;
    if (c == 0 && tid < 2)
        p.count[2 * t + tid] = 0;
}

__global__ __launch_bounds__(256) void k_lp_sum(const int64_t *__restrict__ X, int V,
                                               const int *__restrict__ tokens,
                                               int64_t *__restrict__ logp,
                                               int64_t *__restrict__ entropy, int top,
                                               int *__restrict__ ids, int64_t *__restrict__ tlp,
                                               LpWork p)
{
    q48_round_down();
    __shared__ double tab[64];
    __shared__ int64_t cv[LP_CAP + 8], bv[4], slogz, rcps[64], logs[64];
    __shared__ int ci[LP_CAP + 8], bi[4];
    __shared__ uint32_t thr;
    __shared__ int last;
    const int t = blockIdx.y, c = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const int64_t *x = X + (size_t)t * V;
    const int end = min(V, (c + 1) * p.ch), groups = 4 * p.chunks;
    int64_t g[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int k = lane + 64 * i;
        g[i] = k < groups ? p.gmax[(size_t)t * groups + k] : INT64_MIN;
    }
    lp_table(tab, rcps, logs, tid);
    LpToken token(x, V, tokens, logp != nullptr, t);
    int64_t m = g[0];
#pragma unroll
    for (int i = 1; i < 4; ++i)
        m = g[i] > m ? g[i] : m;
    m = q48_wave_max64(m);
    __syncthreads();   // the table
    if (top && tid < 64) {
        // waves past the row's end have no value: they count as below every other
        uint32_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int k = lane + 64 * i;
            h[i] = k < groups && (k >> 2) * p.ch + 64 * (k & 3) < V ? lp_high(g[i]) : 0;
        }
        const uint32_t n = lp_threshold<4>(
            h, (uint32_t)__builtin_amdgcn_readfirstlane((int)lp_high(m)), top);
        if (tid == 0)
            thr = n;
    }
    uint64_t z64 = 0, w64 = 0;
    int64_t mine = INT64_MIN;
    int i = c * p.ch + tid;
    for (; i + 256 < end; i += 512) {
        const int64_t v[2] = {x[i], x[i + 256]};
        mine = v[0] > mine ? v[0] : mine;
        mine = v[1] > mine ? v[1] : mine;
        const uint64_t u[2] = {(uint64_t)m - (uint64_t)v[0], (uint64_t)m - (uint64_t)v[1]};
        lp_terms<2>(u, tab, z64, w64);
    }
    if (i < end) {
        mine = x[i] > mine ? x[i] : mine;
        const uint64_t u[1] = {(uint64_t)m - (uint64_t)x[i]};
        lp_terms<1>(u, tab, z64, w64);
    }
    uint64_t *sums = p.sums + (size_t)t * groups * 4;
    asm volatile("" : "+v"(token.y));   // (loaded by now: not after the sums)
    lp_wave_sums<true>(z64, w64, sums + 4 * (4 * c + (tid >> 6)), lane);
    if (top) {
        __syncthreads();   // the threshold
        const int first = c * p.ch + tid;
        lp_collect<true>(x, first, 256, end, first < end && lp_high(mine) >= thr, thr,
                         p.cv + (size_t)t * LP_CAP, p.ci + (size_t)t * LP_CAP, p.count + 2 * t,
                         LP_CAP, lane);
    }
    // every wave's stores are out before the block's ticket
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid == 0)
        last = __hip_atomic_fetch_add(p.count + 2 * t + 1, 1, __ATOMIC_RELAXED,
                                      __HIP_MEMORY_SCOPE_AGENT) == p.chunks - 1;
    __syncthreads();
    if (!last)
        return;

    // the row's last block.  Wave 0: the row's sums; the others: its candidates, which
    // wave 1 ranks meanwhile where it holds them all
    const int count = top ? agent_load(p.count + 2 * t) : 0;
    const bool few = count <= 64;
    int64_t v = 0;
    int id = 0, rank = LP_MAX_TOP;
    if (tid < 64) {
        q48_u128 z = 0, w = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (lane + 64 * k < groups) {
                const uint64_t *s = sums + 4 * (lane + 64 * k);
                z += ((q48_u128)agent_load(s + 1) << 64) | agent_load(s);
                w += ((q48_u128)agent_load(s + 3) << 64) | agent_load(s + 2);
            }
        z = q48_wave_sum128(z);
        w = q48_wave_sum128(w);
        const int64_t logz = lp_finish(z, w, m, token, t, rcps, logs, logp, entropy, tid == 0);
        if (tid == 0)
            slogz = logz;
    } else if (!few) {
        for (int k = tid - 64; k < min(count, LP_CAP); k += 192) {
            cv[k] = agent_load(p.cv + (size_t)t * LP_CAP + k);
            ci[k] = agent_load(p.ci + (size_t)t * LP_CAP + k);
        }
    } else if (tid < 128) {
        if (lane < count) {
            v = agent_load(p.cv + (size_t)t * LP_CAP + lane);
            id = agent_load(p.ci + (size_t)t * LP_CAP + lane);
            cv[lane] = v;
            ci[lane] = id;
        }
        // the wave's own writes before its reads
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (lane < count)
            rank = lp_before(cv, ci, count, v, id);
    }
    if (!top)
        return;
    __syncthreads();
    if (few)
        lp_place(rank, v, id, m, slogz, t, top, ids, tlp);
    else if (count <= LP_CAP)
        lp_rank<256>(cv, ci, count, m, slogz, t, top, ids, tlp, tid);
    else
        lp_select<256>(x, V, m, slogz, t, top, ids, tlp, tid, bv, bi);
}

// whether two arrays (or a null one) have bytes in common
bool lp_share(const void *a, size_t na, const void *b, size_t nb)
{
    return a && b && na && (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}

} // namespace

extern "C" {

int q48_logprobs_rows(q48_ctx *c, const int64_t *logits, int T, int vocab, const int *d_tokens,
                      int64_t *logp, int64_t *entropy, int top_n, int *top_ids, int64_t *top_logp)
{
    if (!c || !logits || T <= 0 || T > LP_MAX_ROWS || vocab <= 0 || vocab > (1 << 22) || top_n < 0 ||
        top_n > LP_MAX_TOP || top_n > vocab || (logp && !d_tokens) ||
        (top_n > 0 && (!top_ids || !top_logp)) || (!logp && !entropy && top_n == 0) ||
        q48_off_words<8>(logits, logp, entropy, top_logp) || q48_off_words<4>(d_tokens, top_ids))
        return Q48_EINVAL;
    const size_t n = T, nt = n * top_n;
    auto over = [&](const void *in, size_t bytes) {   // an output that shares words with it
        return lp_share(logp, 8 * n, in, bytes) || lp_share(entropy, 8 * n, in, bytes) ||
               lp_share(top_logp, 8 * nt, in, bytes);
    };
    // (one id a row may replace the row's token: it is read first)
    const bool same = top_n == 1 && top_ids == d_tokens;
    if (over(logits, 8 * n * vocab) || lp_share(top_ids, 4 * nt, logits, 8 * n * vocab) ||
        (logp && (over(d_tokens, 4 * n) || (!same && lp_share(top_ids, 4 * nt, d_tokens, 4 * n)))))
        return Q48_EINVAL;
    q48_on_device on(c);
    // A block a row where the row fits its registers and there are rows for most compute
    // units; else a row over many blocks.  us, a block a row / many: one row of 8000 9.7
    // / 9.8, 16 10.4 / 11.6; 64 rows of 16000 16.0 / 15.6, of 32000 25.6 / 17.9; 128 of
    // 16000 16.2 / 21.8, of 32000 26.3 / 26.7; 256 of 32000 31.4 / 47.6.
    if (vocab <= 8192 || (vocab <= 16384 && T >= 64) || (vocab <= 32768 && T >= 128)) {
#define LP_ROW(R, PER)                                                                         \
    hipLaunchKernelGGL(k_lp_row<R>, dim3(T < PER * c->cu_count ? T : PER * c->cu_count),       \
                       dim3(LR_NT), 0, c->stream, logits, T, vocab, d_tokens, logp, entropy,   \
                       top_n, top_ids, top_logp)
        // (the second number: blocks a compute unit's registers hold)
        if (vocab <= 4096)
            LP_ROW(8, 2);
        else if (vocab <= 8192)
            LP_ROW(16, 2);
        else if (vocab <= 16384)
            LP_ROW(32, 1);
        else
            LP_ROW(64, 1);
#undef LP_ROW
        return hipGetLastError() == hipSuccess ? Q48_OK : Q48_EHIP;
    }
    LpWork p = {};
    // Chunks a row: 16, and up to 64 of long rows that are few: a row's blocks take turns
    // at its counters.  us with 9 / 16 / 32 / 64: one row of 32000 12.1 / 11.0 / 11.1 /
    // 10.9, 16 rows 13.8 / 12.6 / 14.9 / 21.6, 64 18.9 / 17.9 / 23.5 / 37.8; of 130000 one
    // 20.7 / 15.8 / 12.2 / 11.5, 16 22.6 / 20.5 / 18.4 / 24.2, 64 42.8 / 36.0 / 41.1 / 51.8.
    // (Chunks of whole 256s leave at least 8 past 8192 logits: 32 wave maxima, which a
    // threshold for 32 tokens needs.)
    int want = vocab > 65536 ? 2 * c->cu_count / T : 16;
    want = want < 16 ? 16 : want > 64 ? 64 : want;
    p.ch = ((vocab + want - 1) / want + 255) & ~255;
    p.chunks = (vocab + p.ch - 1) / p.ch;
    size_t o = 0;
    auto take = [&](size_t bytes) {
        const size_t at = o;
        o += (bytes + 255) & ~(size_t)255;
        return at;
    };
    // rows of one launch: a grid's y, and a bounded workspace
    const int rows = T < 32768 ? T : 32768;
    const size_t o_g = take((size_t)rows * 4 * p.chunks * 8);
    const size_t o_s = take((size_t)rows * 4 * p.chunks * 32), o_n = take((size_t)rows * 8);
    const size_t o_v = take((size_t)rows * LP_CAP * 8), o_i = take((size_t)rows * LP_CAP * 4);
    const int rc = q48_ws_reserve(c, o);
    if (rc)
        return rc;
    uint8_t *ws = (uint8_t *)c->ws;
    p.gmax = (int64_t *)(ws + o_g);
    p.sums = (uint64_t *)(ws + o_s);
    p.count = (int *)(ws + o_n);
    p.cv = (int64_t *)(ws + o_v);
    p.ci = (int *)(ws + o_i);
    for (int t0 = 0; t0 < T; t0 += rows) {
        const int n = rows < T - t0 ? rows : T - t0;
        const int64_t *x = logits + (size_t)t0 * vocab;
        hipLaunchKernelGGL(k_lp_max, dim3(p.chunks, n), dim3(256), 0, c->stream, x, vocab, p);
        hipLaunchKernelGGL(k_lp_sum, dim3(p.chunks, n), dim3(256), 0, c->stream, x, vocab,
                           d_tokens ? d_tokens + t0 : nullptr, logp ? logp + t0 : nullptr,
                           entropy ? entropy + t0 : nullptr, top_n,
                           top_ids ? top_ids + (size_t)t0 * top_n : nullptr,
                           top_logp ? top_logp + (size_t)t0 * top_n : nullptr, p);
    }
    return hipGetLastError() == hipSuccess ? Q48_OK : Q48_EHIP;
}

} // extern "C"
