// q48_expn.hpp — e^-u of Q16.48 words over the whole range: u = n LN2 + j / 64 + s
// splits the exponent into a shift, a table and a six-step Horner row on s < 2^-6.
// Included by the HIP sources of libintllm_hip only.
#pragma once

#include "q48_device.hpp"

namespace {

constexpr int64_t EXPN_LN2 = 195103586505167LL;   // fp_log's ln 2 (fp_math.h:752-773)

// round(2^48 e^(-j/64)), round(2^48 / k!)
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
constexpr int64_t kFactK[7] = {
    281474976710656LL, 281474976710656LL, 140737488355328LL, 46912496118443LL, 11728124029611LL,
    2345624805922LL, 390937467654LL};

// floor(floor(T_j h 2^-48) 2^-n) of one u, for the few exponentials of a row of expert
// logits (q48_logprob.hip's lp_terms has the form for many).  FP64 rounds down
// (q48_round_down): a truncated product of integers below 2^49 is one fused operation,
// fma(a, b 2^-48, 2^52) = 2^52 + floor(a b / 2^48).
__device__ __forceinline__ int64_t q48_expn(uint64_t u)
{
    constexpr uint64_t L = (uint64_t)EXPN_LN2;
    const bool in = u < 49 * L;
    const uint64_t v = in ? u : 0;
    // the quotient or one less: both factors are rounded down
    uint32_t n = (uint32_t)((double)(v >> 8) * (0x1.7154765200000p-48 * 256));
    uint64_t r = v - n * L;
    if (r >= L) {
        r -= L;
        ++n;
    }
    const double s = (double)(int64_t)(r & (((uint64_t)1 << 42) - 1)) * 0x1p-48;
    double h = (double)kFactK[6];
#pragma unroll
    for (int k = 5; k >= 0; --k)
        h = ((double)kFactK[k] + 0x1p52) - __builtin_fma(s, h, 0x1p52);
    const double e = __builtin_fma((double)kExp[r >> 42] * 0x1p-48, h, 0x1p52);
    return in ? (int64_t)(q48_word_m52(e) >> n) : 0;
}

} // namespace
