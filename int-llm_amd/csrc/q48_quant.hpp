// q48_quant.hpp — a head vector as the quantised cache holds it, for the kernels
// that write the cache.  Included by the HIP sources of libintllm_hip only.
#pragma once

#include "q48_internal.h"

namespace {

// rope_apply's rotation of one pair (llama_int.c:997-1008)
__device__ __forceinline__ void q48_rope_pair(int64_t &x0, int64_t &x1, int64_t c, int64_t s)
{
    const int64_t y0 = (int64_t)((uint64_t)q48_mul(x0, c) - (uint64_t)q48_mul(x1, s));
    const int64_t y1 = (int64_t)((uint64_t)q48_mul(x1, c) + (uint64_t)q48_mul(x0, s));
    x0 = y0;
    x1 = y1;
}

__device__ __forceinline__ uint64_t q48_magnitude(int64_t x)
{
    return x < 0 ? (uint64_t)0 - (uint64_t)x : (uint64_t)x;
}

// maximum over the 16 lanes of a row (all active), unsigned
__device__ __forceinline__ uint64_t q48_row16_umax(uint64_t v)
{
    uint64_t o = q48_dpp64<Q48_DPP_XOR1>(v);
    v = o > v ? o : v;
    o = q48_dpp64<Q48_DPP_XOR2>(v);
    v = o > v ? o : v;
    o = q48_dpp64<Q48_DPP_HALF_MIRROR>(v);
    v = o > v ? o : v;
    o = q48_dpp64<Q48_DPP_MIRROR>(v);
    return o > v ? o : v;
}

// sign(x) min(Q, floor((|x| + floor(step / 2)) / step)); r = 1 / step in FP64,
// within a few units of 2^-50: the estimate of a quotient of at most Q + 1 is
// off by less than one, and the remainder settles it.
template <int Q>
__device__ __forceinline__ int q48_code(int64_t x, uint64_t step, double r)
{
    const uint64_t n = q48_magnitude(x) + (step >> 1);
    int q = (int)((double)n * r);
    const int64_t rem = (int64_t)(n - (uint64_t)(uint32_t)q * step);
    q += rem < 0 ? -1 : rem >= (int64_t)step ? 1 : 0;
    q = q < Q ? q : Q;
    return x < 0 ? -q : q;
}

// The 16 lanes of a row quantise one head vector: lane l holds the dims i = l N +
// (0 .. N - 1) in lo and i + HD / 2 in hi, N = HD / 32.  Codes to dst, step to
// *st (lane 0).  16 lanes a vector: a maximum is four DPP steps, and the pairs of
// a byte (4 bits) or of a rotation are one lane's.
template <int BITS, int HD>
__device__ __forceinline__ void q48_quantise_row(uint8_t *dst, int64_t *st, int l,
                                                 const int64_t (&lo)[HD / 32],
                                                 const int64_t (&hi)[HD / 32])
{
    constexpr int N = HD / 32, Q = BITS == 8 ? 127 : 7;
    uint64_t a = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint64_t p = q48_magnitude(lo[i]), q = q48_magnitude(hi[i]);
        a = p > a ? p : a;
        a = q > a ? q : a;
    }
    a = q48_row16_umax(a);
    uint64_t step = (a + (Q - 1)) / Q;
    constexpr uint64_t cap = (uint64_t)INT64_MAX / Q;
    step = step < cap ? step : cap;
    const double d = (double)step;
    double r = __builtin_amdgcn_rcp(d);
    r = __builtin_fma(r, __builtin_fma(-d, r, 1.0), r);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int p = step ? q48_code<Q>(lo[i], step, r) : 0;
        const int q = step ? q48_code<Q>(hi[i], step, r) : 0;
        if (BITS == 8) {
            dst[l * N + i] = (uint8_t)p;
            dst[l * N + i + HD / 2] = (uint8_t)q;
        } else {
            dst[l * N + i] = (uint8_t)((p & 15) | (q << 4));
        }
    }
    if (l == 0)
        *st = (int64_t)step;
}

} // namespace
