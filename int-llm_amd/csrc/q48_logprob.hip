// q48_logprob.hip — log probabilities of given tokens, the entropy and the most
// probable tokens of rows of logits (q48_logprobs_rows; include/intllm_hip.h has
// the integer steps).
//
// e^-u over the whole range: u = n LN2 + j / 64 + s splits the exponent into a
// shift, a table and a six-step Horner row on s < 2^-6 (s^7 / 5040 < 2^-54), a
// third of fp_exp's squarings and division, and 4 units of 2^-48 from e^-u.
#include "q48_attn.hpp"

namespace {

constexpr int64_t LP_LN2 = 195103586505167LL;   // fp_log's ln 2 (fp_math.h:752-773)
constexpr int LP_MAX_TOP = 32;

// round(2^48 e^(-j/64)), round(2^48 / k!), floor(2^54 / (64 + j)),
// round(2^48 log(1 + j/64)), round(2^48 / (k + 1))
static __constant__ int64_t kExp[45] = {
    281474976710656LL, 277111111677821LL, 272814902101423LL, 268585299080830LL, 264421269977109LL,
    260321798160909LL, 256285882764256LL, 252312538436196LL, 248400795102225LL, 244549697727451LL,
    240758306083425LL, 237025694518590LL, 233350951732284LL, 229733180552255LL, 226171497715615LL,
    222665033653200LL, 219212932277264LL, 215814350772475LL, 212468459390137LL, 209174441245618LL,
    205931492118908LL, 202738820258272LL, 199595646186949LL, 196501202512843LL, 193454733741172LL,
    190455496090014LL, 187502757308717LL, 184595796499121LL, 181733903939560LL, 178916380911580LL,
    176142539529353LL, 173411702571733LL, 170723203316912LL, 168076385379650LL, 165470602551013LL,
    162905218640611LL, 160379607321268LL, 157893151976115LL, 155445245548039LL, 153035290391475LL,
    150662698126495LL, 148326889495156LL, 146027294220076LL, 143763350865205LL, 141534506698753LL};
static __constant__ int64_t kFact[7] = {
    281474976710656LL, 281474976710656LL, 140737488355328LL, 46912496118443LL, 11728124029611LL,
    2345624805922LL, 390937467654LL};
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
static __constant__ int64_t kInv[8] = {
    281474976710656LL, 140737488355328LL, 93824992236885LL, 70368744177664LL, 56294995342131LL,
    46912496118443LL, 40210710958665LL, 35184372088832LL};

// e_i of u (include/intllm_hip.h)
__device__ __forceinline__ int64_t lp_exp(uint64_t u)
{
    const uint64_t n = u / LP_LN2;
    if (n >= 49)
        return 0;
    const int64_t r = (int64_t)(u - n * LP_LN2), s = r & (((int64_t)1 << 42) - 1);
    int64_t h = kFact[6];
#pragma unroll
    for (int k = 5; k >= 0; --k)
        h = kFact[k] - q48_mul(s, h);
    return q48_mul(kExp[r >> 42], h) >> n;
}

// logZ of Z >= 2^48, and its b
__device__ int64_t lp_log(q48_u128 Z, int &b)
{
    const uint64_t zh = (uint64_t)(Z >> 64), zl = (uint64_t)Z;
    b = (zh ? 128 - __builtin_clzll(zh) : 64 - __builtin_clzll(zl)) - 49;
    const int64_t z = (int64_t)(Z >> b);
    const int j = (int)(z >> 42) - 64;
    const int64_t d = q48_mul(z, kRcp[j]) - Q48_ONE;
    int64_t g = kInv[7];
#pragma unroll
    for (int k = 6; k >= 0; --k)
        g = kInv[k] - q48_mul(d, g);
    return b * LP_LN2 + kLog[j] + q48_mul(d, g);
}

__device__ __forceinline__ int64_t lp_value(uint64_t u, int64_t logz)
{
    const uint64_t v = u + (uint64_t)logz;
    return v < u || v > (uint64_t)INT64_MAX ? INT64_MIN : -(int64_t)v;
}

__global__ __launch_bounds__(256) void k_lp_simple(const int64_t *__restrict__ X, int V,
                                                  const int *__restrict__ tokens,
                                                  int64_t *__restrict__ logp,
                                                  int64_t *__restrict__ entropy, int top,
                                                  int *__restrict__ ids,
                                                  int64_t *__restrict__ tlp)
{
    q48_round_down();
    __shared__ int64_t red[4], bv[4];
    __shared__ uint64_t sums[4][4];
    __shared__ int bi[4];
    const int t = blockIdx.x, tid = threadIdx.x;
    const int64_t *x = X + (size_t)t * V;
    int64_t m = INT64_MIN;
    for (int i = tid; i < V; i += 256)
        m = x[i] > m ? x[i] : m;
    m = block_max64<256>(m, red);
    q48_u128 z = 0, w = 0;
    for (int i = tid; i < V; i += 256) {
        const uint64_t u = (uint64_t)m - (uint64_t)x[i];
        const int64_t e = lp_exp(u);
        if (e) {
            z += (uint64_t)e;
            w += (uint64_t)q48_mul(e, (int64_t)u);
        }
    }
    z = q48_wave_sum128(z);
    w = q48_wave_sum128(w);
    if ((tid & 63) == 0) {
        sums[tid >> 6][0] = (uint64_t)z;
        sums[tid >> 6][1] = (uint64_t)(z >> 64);
        sums[tid >> 6][2] = (uint64_t)w;
        sums[tid >> 6][3] = (uint64_t)(w >> 64);
    }
    __syncthreads();
    z = w = 0;
    for (int i = 0; i < 4; ++i) {
        z += ((q48_u128)sums[i][1] << 64) | sums[i][0];
        w += ((q48_u128)sums[i][3] << 64) | sums[i][2];
    }
    int b;
    const int64_t logz = lp_log(z, b);
    if (tid == 0) {
        if (logp) {
            const int id = tokens[t];
            logp[t] = id >= 0 && id < V ? lp_value((uint64_t)m - (uint64_t)x[id], logz) : 0;
        }
        if (entropy)
            entropy[t] = logz + q48_div((int64_t)(w >> b), (int64_t)(z >> b));
    }
    int64_t lv = INT64_MAX;
    int li = -1;
    for (int n = 0; n < top; ++n) {
        int64_t v = INT64_MIN;
        int at = INT_MAX;
        for (int i = tid; i < V; i += 256)
            if ((x[i] < lv || (x[i] == lv && i > li)) &&
                (at == INT_MAX || x[i] > v)) {
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
        for (int i = 1; i < 4; ++i)
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

} // namespace

extern "C" {

int q48_logprobs_rows(q48_ctx *c, const int64_t *logits, int T, int vocab, const int *d_tokens,
                      int64_t *logp, int64_t *entropy, int top_n, int *top_ids, int64_t *top_logp)
{
    if (!c || !logits || T <= 0 || vocab <= 0 || vocab > (1 << 22) || top_n < 0 ||
        top_n > LP_MAX_TOP || top_n > vocab || (logp && !d_tokens) ||
        (top_n > 0 && (!top_ids || !top_logp)) || (!logp && !entropy && top_n == 0))
        return Q48_EINVAL;
    q48_on_device on(c);
    hipLaunchKernelGGL(k_lp_simple, dim3(T), dim3(256), 0, c->stream, logits, vocab, d_tokens, logp,
                       entropy, top_n, top_ids, top_logp);
    return hipGetLastError() == hipSuccess ? Q48_OK : Q48_EHIP;
}

} // extern "C"
