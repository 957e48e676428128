// q48_moe.hip — a mixture-of-experts layer over weights in 8 bits (q48_moe_w8;
// include/intllm_hip.h has the integer steps).
//
// Rows normed and put into 8 bits, the router's logits, the choice; then the chosen
// (token, expert) pairs as slots sorted by expert, each expert's from a multiple of 16
// on, so that the products run over 16 slots of one expert at a time; gate and up with
// SwiGLU, its rows into 8 bits, and down, added to the tokens' rows.  The adds are of
// integers mod 2^64: their order changes nothing.
#include "q48_expn.hpp"
#include "q48_w8.hpp"

namespace {

constexpr int MOE_MAX_TOP = 64;

// Words that other blocks of the launch read behind a ticket: coherent stores and loads.
template <class V>
__device__ __forceinline__ void out_to_all(V *p, V v)
{
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <class V>
__device__ __forceinline__ V from_all(const V *p)
{
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// A wave chooses a token's experts: lane l holds the logits of experts l + 64 i in v, and
// gets the l-th choice and its weight (l < top).  top times the largest logit not yet
// taken, of equal ones the lowest expert.
template <int PER>
__device__ __forceinline__ void moe_choose(const int64_t (&v)[PER], int E, int top, bool renorm,
                                           int &id, int64_t &weight)
{
    const int lane = threadIdx.x & 63;
    uint32_t left = 0;   // bit i: expert lane + 64 i, not taken
#pragma unroll
    for (int i = 0; i < PER; ++i)
        left |= lane + 64 * i < E ? 1u << i : 0u;
    int64_t m = 0, mine = 0;
    id = 0;
    for (int j = 0; j < top; ++j) {
        int64_t best = INT64_MIN;
        int at = E;   // none left: past every expert
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (((left >> i) & 1) && (at == E || v[i] > best)) {
                best = v[i];
                at = lane + 64 * i;
            }
        const int64_t most = q48_wave_max64(best);
        uint64_t who = __ballot(at < E && best == most);
        int won;
        if constexpr (PER == 1) {
            won = (int)__builtin_ctzll(who);
        } else {
            won = E;   // the lowest expert of the lanes that hold it
            while (who) {
                const int o = __builtin_amdgcn_readlane(at, (int)__builtin_ctzll(who));
                won = o < won ? o : won;
                who &= who - 1;
            }
        }
        if (at == won)
            left &= ~(1u << (won >> 6));
        if (j == 0)
            m = most;
        if (lane == j) {
            mine = most;
            id = won;
        }
    }
    const int64_t e = q48_expn((uint64_t)m - (uint64_t)mine);
    int64_t sum = lane < top ? e : 0;
    if (!renorm) {
        sum = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            sum += lane + 64 * i < E ? q48_expn((uint64_t)m - (uint64_t)v[i]) : 0;
    }
    sum = q48_wave_sum64(sum);
    weight = q48_div(e, sum);
}

// The pairs counted by expert, each expert's first slot, the items of `rows` slots, and every
// pair into its slot: one block of NT threads.  A launch of its own: 4096 pairs of 8 experts
// 9 us, 16384 of 64 33.
struct MoeSlots {
    int4 *items;
    int *tok;
    int64_t *w;
    int slots, n_items, rows;
};
template <int NT>
__device__ __forceinline__ void moe_slots(const MoeSlots &s, const int *chosen,
                                          const int64_t *weight, int pairs, int top, int E)
{
    __shared__ int count[W8_MAX_COUNT], first[W8_MAX_COUNT], item[W8_MAX_COUNT];
    const int tid = threadIdx.x, lane = tid & 63;
    // a thread's first pair, fetched once
    const int e0 = tid < pairs ? from_all(chosen + tid) : 0;
    const int64_t w0 = tid < pairs ? from_all(weight + tid) : 0;
    for (int i = tid; i < E; i += NT)
        count[i] = 0;
    for (int i = tid; i < s.slots; i += NT)
        s.tok[i] = -1;
    for (int i = tid; i < s.n_items; i += NT)
        s.items[i] = make_int4(0, 0, 0, 0);
    __syncthreads();
    for (int i = tid; i < pairs; i += NT) {
        const int e = i == tid ? e0 : from_all(chosen + i);
        atomicAdd(&count[e], 1);
    }
    __syncthreads();
    if (tid < 64) {   // slots (in sixteens) and items before each expert: sums over a wave
        int slots = 0, items = 0;
        for (int b = 0; b < E; b += 64) {
            const int c = b + lane < E ? count[b + lane] : 0;
            const int n = (c + 15) & ~15, k = (c + s.rows - 1) / s.rows;
            int sn = n, sk = k;
            for (int d = 1; d < 64; d <<= 1) {
                const int on = __shfl_up(sn, d), ok = __shfl_up(sk, d);
                sn += lane >= d ? on : 0;
                sk += lane >= d ? ok : 0;
            }
            if (b + lane < E) {
                first[b + lane] = slots + sn - n;
                item[b + lane] = items + sk - k;
            }
            slots += __builtin_amdgcn_readlane(sn, 63);
            items += __builtin_amdgcn_readlane(sk, 63);
        }
    }
    __syncthreads();
    for (int e = tid; e < E; e += NT) {
        const int n = count[e];
        for (int i = 0; i < n; i += s.rows)
            s.items[item[e] + i / s.rows] = make_int4(e, first[e] + i, min(s.rows, n - i), 0);
        count[e] = first[e];
    }
    __syncthreads();
    for (int i = tid; i < pairs; i += NT) {
        const int at = atomicAdd(&count[i == tid ? e0 : from_all(chosen + i)], 1);
        s.tok[at] = i / top;
        s.w[at] = i == tid ? w0 : from_all(weight + i);
    }
}

// A wave a token.
template <int PER>
__global__ __launch_bounds__(256) void k_moe_choose(const int64_t *__restrict__ logits, int T,
                                                   int E, int top, int renorm,
                                                   int *__restrict__ chosen,
                                                   int64_t *__restrict__ weight)
{
    q48_round_down();
    const int lane = threadIdx.x & 63, t = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= T)
        return;
    int64_t v[PER], w;
    int id;
#pragma unroll
    for (int i = 0; i < PER; ++i)
        v[i] = lane + 64 * i < E ? logits[(size_t)t * E + lane + 64 * i] : 0;
    moe_choose<PER>(v, E, top, renorm != 0, id, w);
    if (lane < top) {
        chosen[(size_t)t * top + lane] = id;
        weight[(size_t)t * top + lane] = w;
    }
}

__global__ __launch_bounds__(1024) void k_moe_slots(const int *__restrict__ chosen,
                                                   const int64_t *__restrict__ weight, int pairs,
                                                   int top, int E, MoeSlots s)
{
    moe_slots<1024>(s, chosen, weight, pairs, top, E);
}

// Everything before the experts in one launch, for few tokens: block (g, t) norms row t
// and makes the logits of experts g per + 0 .. per - 1; one block more a token its codes.
// The last block of a token to finish chooses, the last of those makes the slots (tickets;
// no block waits for another).  It is a chain of latencies: a token and 8 experts of 2048
// 9.3 us (the separate launches' kernels 18), 26 tokens and 64 experts 20.5 (45), 200 tokens
// and 15 of 1000 16.3 (30).  Two blocks a unit leave 64 registers a thread: of normed rows up
// to 2048 that form spills 32, and is faster for it (one block a unit: 27.9 for 20.7).
constexpr int ROUTE_PER = 16;    // experts a block at most
constexpr int ROUTE_T = 1024;    // tokens at most
struct MoeRoute {
    W8Rows rows;
    const int64_t *router;
    int64_t *logits;
    int E, per, sl, p2, top, renorm;   // p2: 2^p2 >= E, at least 64
    int one;                     // T = 1 and k_w8_one behind it: every choice an item of one slot
    int *chosen;
    int64_t *weight;
    int *ticket;                 // [0]: tokens, [1 + t]: blocks of token t; zeros between launches
    MoeSlots s;
};
template <int NT, int J, bool NORM>
__global__ __launch_bounds__(1024, J == 8 ? 4 : 8) void k_moe_route(MoeRoute a)
{
    q48_round_down();
    constexpr int NW = 16;
    extern __shared__ __align__(16) int64_t xs[];   // the row, normed; then logits and ranks
    __shared__ uint64_t red[NT / 64][2], peak[NT / 64], part[NW][2];
    __shared__ int last;
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int t = blockIdx.y, K = a.rows.K, T = a.rows.T, E = a.E, G = gridDim.x - 1;
    const int e0 = blockIdx.x * a.per, n = min(a.per, E - e0);
    if (tid < NT) {
        RowWords<NT, 2, J> x;
        x.load(a.rows.X + (size_t)t * K, K);
        if constexpr (NORM)
            x.norm(a.rows.X + (size_t)t * K, a.rows.norm_w, K, red);
        if ((int)blockIdx.x == G) {
            const int KT = (K + 63) / 64;
            const int64_t step = x.quantise(K, KT, peak, [&](int i, uint32_t q) {
                *(uint16_t *)(a.rows.codes + w8_at(t, i, KT)) = (uint16_t)q;
            });
            if (tid == 0)
                a.rows.step[t] = step;
            return;
        }
#pragma unroll
        for (int j = 0; j < J; ++j)
            if (x.at(j) < K) {
                xs[x.at(j)] = x.word(j, 0);
                xs[x.at(j) + 1] = x.word(j, 1);
            }
    } else {
        if constexpr (NORM)
            lds_barrier();
        if ((int)blockIdx.x == G) {
            if (a.rows.out)
                for (int i = tid - NT; i < K; i += 1024 - NT)
                    a.rows.out[(size_t)t * K + i] = a.rows.base ? a.rows.base[(size_t)t * K + i] : 0;
            lds_barrier();
            return;
        }
    }
    lds_barrier();
    // S = 2^sl waves an expert, each its share of the row.  Words below 2^54 as halves of 27
    // bits: four multiply-adds into three sums without a carry (the four products of a
    // signed 64 x 64 multiplication with its carries and signs take twice as long); a share
    // with larger words again in 128 bits.
    const int sl = a.sl, S = 1 << sl, e = w >> sl, seg = ((K + S - 1) >> sl);
    q48_u128 sum = 0;
    if (e < n) {
        const int from = (w & (S - 1)) * seg, to = min(from + seg, K);
        const int64_t *r = a.router + (size_t)(e0 + e) * K;
        int64_t hh = 0, hl = 0, ll = 0;
        uint32_t big = 0;
        for (int i = from + lane; i < to; i += 64 * 8) {
            int64_t v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u)
                v[u] = i + 64 * u < to ? r[i + 64 * u] : 0;
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (i - lane + 64 * u < to) {
                    const int64_t x = xs[min(i + 64 * u, K - 1)];
                    const int xh = (int)(x >> 27), xl = (int)((uint32_t)x & 0x7ffffffu);
                    const int vh = (int)(v[u] >> 27), vl = (int)((uint32_t)v[u] & 0x7ffffffu);
                    const int xt = (int)(x >> 32), vt = (int)(v[u] >> 32);
                    big |= (uint32_t)(xt ^ (xt >> 31)) | (uint32_t)(vt ^ (vt >> 31));
                    hh += (int64_t)xh * vh;
                    hl += (int64_t)xh * vl;
                    hl += (int64_t)xl * vh;
                    ll += (int64_t)xl * vl;
                }
        }
        sum = ((q48_u128)(q48_i128)hh << 54) + ((q48_u128)(q48_i128)hl << 27) + (uint64_t)ll;
        if (__any(big >= 1u << 22)) {
            sum = 0;
            for (int i = from + lane; i < to; i += 64)
                sum += (q48_u128)q48_smul128(xs[i], r[i]);
        }
        sum = q48_wave_sum128(sum);
    }
    if (lane == 0) {
        part[w][0] = (uint64_t)sum;
        part[w][1] = (uint64_t)(sum >> 64);
    }
    lds_barrier();   // (the row is done with)
    int64_t *lg = xs;
    int *rank = (int *)(xs + E);
    int64_t mine_l = 0;
    if (tid < n) {
        sum = 0;
        for (int i = 0; i < S; ++i)
            sum += ((q48_u128)part[(tid << sl) + i][1] << 64) | part[(tid << sl) + i][0];
        mine_l = (int64_t)(uint64_t)(sum >> 48);
    }
    if (G > 1) {
        if (tid < n) {
            out_to_all(a.logits + (size_t)t * E + e0 + tid, mine_l);
            __builtin_amdgcn_s_waitcnt(0);   // out before the ticket (n <= 16: one wave's stores)
        }
        if (tid == 0) {
            const int at = __hip_atomic_fetch_add(a.ticket + 1 + t, 1, __ATOMIC_RELAXED,
                                                  __HIP_MEMORY_SCOPE_AGENT);
            last = at == G - 1;
            if (at == G - 1)
                out_to_all(a.ticket + 1 + t, 0);
        }
        __syncthreads();
        if (!last)
            return;
        if (tid < E)
            mine_l = from_all(a.logits + (size_t)t * E + tid);
    }
    // The token's choice by all threads: an expert's rank is the number of larger logits
    // and of equal ones before it, counted by 1024 / P threads an expert (P: experts to a
    // power of two), and each chosen expert makes its own weight.
    {
        __shared__ int64_t most;
        __shared__ uint64_t z;
        const int P = 1 << a.p2, ex = tid & (P - 1), parts = 1024 >> a.p2, part_ = tid >> a.p2;
        if (tid < E) {
            lg[tid] = mine_l;
            rank[tid] = 0;
        }
        if (tid == 0)
            z = 0;
        lds_barrier();
        const int64_t mine = lg[min(ex, E - 1)];
        int before = 0;
        for (int i = part_; i < E; i += parts)
            before += lg[i] > mine || (lg[i] == mine && i < ex) ? 1 : 0;
        if (ex < E && before)
            atomicAdd(&rank[ex], before);
        lds_barrier();
        const int my = tid < E ? rank[tid] : E;
        if (my == 0)
            most = mine;
        lds_barrier();
        int64_t ew = 0;
        if (my < (a.renorm ? a.top : E)) {
            ew = q48_expn((uint64_t)most - (uint64_t)mine);
            atomicAdd((unsigned long long *)&z, (unsigned long long)ew);
        }
        lds_barrier();
        if (my < a.top) {
            const int64_t wt = q48_div(ew, (int64_t)z);
            out_to_all(a.chosen + (size_t)t * a.top + my, tid);
            out_to_all(a.weight + (size_t)t * a.top + my, wt);
            if (a.one) {
                a.s.items[my] = make_int4(tid, 16 * my, 1, 0);
                a.s.tok[16 * my] = 0;
                a.s.w[16 * my] = wt;
            }
        }
    }
    if (a.one)
        return;
    __builtin_amdgcn_s_waitcnt(0);   // every wave's stores are out before the ticket
    __syncthreads();
    if (tid == 0) {
        const int at = __hip_atomic_fetch_add(a.ticket, 1, __ATOMIC_RELAXED,
                                              __HIP_MEMORY_SCOPE_AGENT);
        last = at == T - 1;
        if (at == T - 1)
            out_to_all(a.ticket, 0);
    }
    __syncthreads();
    if (last)
        moe_slots<1024>(a.s, a.chosen, a.weight, T * a.top, a.top, E);
}

int launch_rc(int e) { return e == (int)hipSuccess ? Q48_OK : Q48_EHIP; }

// slots that n pairs of at most E experts can take, in sixteens
size_t slots_of(size_t pairs, int E)
{
    return (pairs + 15 * (pairs < (size_t)E ? pairs : (size_t)E) + 15) & ~(size_t)15;
}

// Experts a block of k_moe_route, 0 for the separate launches (a row of words in LDS): the
// fewest with which every block, the codes' among them, is resident at once, or 16 and up to
// three rounds of blocks (two of them a compute unit for rows of up to 2048).  us for a whole
// layer, one launch / separate: 8 experts, 64 tokens 32 / 68, 512 86 / 111, 700 113 / 130; 16,
// 700 131 / 136, 1024 185 / 174; 64, 128 tokens 71 / 88, 256 123 / 127, 400 161 / 150; 128 of
// rows of 1024, 128 tokens 62 / 74, 256 90 / 77; 8 of rows of 4096, 512 133 / 141, 700 171 / 160.
int route_per(const q48_ctx *c, int T, int E, int dim)
{
    if (dim > 6144 || T > ROUTE_T)
        return 0;
    const int most = (dim <= 2048 ? 2 : 1) * c->cu_count, G = most / T > 1 ? most / T - 1 : 1;
    const int per = (E + G - 1) / G < ROUTE_PER ? (E + G - 1) / G : ROUTE_PER;
    const int blocks = T * ((E + per - 1) / per + 1);
    return blocks <= (dim <= 2048 ? 6 : 4) * c->cu_count ? per : 0;
}

int launch_route(q48_ctx *c, const MoeRoute &a)
{
    const dim3 grid((a.E + a.per - 1) / a.per + 1, a.rows.T);
    const size_t lds = max(8 * ((a.rows.K + 1) & ~1), 12 * a.E);
#define ROUTE(NT, J, NORM)                                                                   \
    hipLaunchKernelGGL((k_moe_route<NT, J, NORM>), grid, dim3(1024), lds, c->stream, a)
    if (a.rows.K <= 2048 && a.rows.norm_w)
        ROUTE(256, 4, true);
    else if (a.rows.K <= 2048)
        ROUTE(256, 4, false);
    else if (a.rows.norm_w)
        ROUTE(512, 8, true);
    else
        ROUTE(512, 8, false);
#undef ROUTE
    return (int)hipGetLastError();
}

// items of `rows` slots that they can take
size_t items_of(size_t pairs, int E, int rows)
{
    return pairs / rows + (pairs < (size_t)E ? pairs : (size_t)E);
}

} // namespace

extern "C" {

int q48_moe_w8(q48_ctx *c, int64_t *out, const int64_t *base, const q48_moe *moe,
               const int64_t *X, const int64_t *norm_w, int T, int *chosen, int64_t *weight)
{
    if (!c || !out || !X || !moe || !moe->router || T <= 0 || T > W8_MAX_T ||
        !q48_w8_ok(&moe->gate) || !q48_w8_ok(&moe->up) || !q48_w8_ok(&moe->down) ||
        q48_off_words<8>(out, base, X, norm_w, weight, moe->router) || q48_off_words<4>(chosen))
        return Q48_EINVAL;
    const q48_w8 &g = moe->gate, &u = moe->up, &d = moe->down;
    const int E = g.count, dim = g.K, ffn = g.N, top = moe->top_k;
    if (u.count != E || d.count != E || u.K != dim || u.N != ffn || d.K != ffn || d.N != dim ||
        top <= 0 || top > E || top > MOE_MAX_TOP)
        return Q48_EINVAL;
    const size_t row = (size_t)dim * 8, all = (size_t)T * row;
    // out may be X itself where that is the base too: the adds come after X was read
    const void *ins[] = {norm_w, moe->router, g.codes, g.step, u.codes, u.step, d.codes, d.step};
    const size_t sizes[] = {row, (size_t)E * row, (size_t)E * w8_tiles(ffn, dim),
                            (size_t)E * ffn * 8, (size_t)E * w8_tiles(ffn, dim),
                            (size_t)E * ffn * 8, (size_t)E * w8_tiles(dim, ffn),
                            (size_t)E * dim * 8};
    const size_t np = (size_t)T * top;
    for (int i = 0; i < 8; ++i)
        if (q48_share(out, all, ins[i], sizes[i]) || q48_share(chosen, np * 4, ins[i], sizes[i]) ||
            q48_share(weight, np * 8, ins[i], sizes[i]))
            return Q48_EINVAL;
    if ((out == X ? base != out : q48_share(out, all, X, all)) ||
        (base != out && q48_share(out, all, base, all)))
        return Q48_EINVAL;
    for (const void *v : {(const void *)out, (const void *)X, (const void *)base})
        if (q48_share(chosen, np * 4, v, all) || q48_share(weight, np * 8, v, all))
            return Q48_EINVAL;
    if (q48_share(chosen, np * 4, weight, np * 8))
        return Q48_EINVAL;
    q48_on_device on(c);
    static_assert(sizeof(int) * (1 + ROUTE_T) <= W8_TICKETS, "tickets");
    size_t o = W8_TICKETS;
    auto take = [&](size_t bytes) {
        const size_t at = o;
        o += (bytes + 255) & ~(size_t)255;
        return at;
    };
    // Tokens of one pass: 2^19 pairs and half a GiB of their hidden words at most, and a GiB
    // with the slots that fill up each expert's sixteens (16 slots a pair while there are no
    // more pairs than experts: a token's 64 pairs of the longest rows are a GiB).
    size_t Tc = ((size_t)1 << 30) / ((size_t)16 * top * ffn);
    Tc = Tc < ((size_t)1 << 19) / top ? Tc : ((size_t)1 << 19) / top;
    const size_t most = ((size_t)1 << 30) / ((size_t)8 * ffn);   // slots
    const size_t fit = (most / 16 <= (size_t)E ? most / 16 : most - 15 * (size_t)E - 15) / top;
    Tc = Tc < fit ? Tc : fit;
    Tc = Tc < 1 ? 1 : Tc < (size_t)T ? Tc : (size_t)T;
    const size_t slots = slots_of(Tc * top, E), n_items = items_of(Tc * top, E, 16);
    const size_t o_x = take(w8_tiles((int)Tc, dim)), o_xs = take(Tc * 8);
    const size_t o_xn = take(norm_w ? Tc * row : 0), o_l = take(Tc * E * 8);
    const size_t o_c = take(Tc * top * 4), o_w = take(Tc * top * 8);
    const size_t o_i = take(n_items * sizeof(int4)), o_t = take(slots * 4), o_sw = take(slots * 8);
    const size_t o_h = take(slots * ffn * 8), o_hc = take(w8_tiles((int)slots, ffn));
    const size_t o_hs = take(slots * 8);
    int rc = q48_w8_reserve(c, o);
    if (rc)
        return rc;
    uint8_t *ws = (uint8_t *)c->w8;
    for (size_t t0 = 0; t0 < (size_t)T; t0 += Tc) {
        const int n = (int)(Tc < T - t0 ? Tc : T - t0);
        const int sl = (int)slots_of((size_t)n * top, E);
        // Slots an item, by an expert's average: weights are read once an item.  128, in
        // k_w8_gemm, where that leaves blocks for most of the chip in down's launch too.
        // us, 32 / 64 / 128 slots: 8 experts of 2048 x 5632, 64 pairs each 162 / 163 / 162,
        // 128 287 / 285 / 253, 512 815 / 766 / 499; 64 of 2048 x 1024, 16 pairs 175 / 192 /
        // 183 (16 slots: 172), 32 223 / 226 / 215, 256 894 / 855 / 635; 8 of 1024 x 2816, 64
        // pairs 57 / 60 / 99, 256 165 / 163 / 177, 512 266 / 257 / 238.
        const size_t pairs = (size_t)n * top, mean = pairs / E;
        const size_t blocks = (pairs / 128 + E / 2) * ((dim + 127) / 128);   // of down, expected
        const int rows = mean <= 16                                                  ? 16
                         : mean >= 32 && blocks >= (size_t)c->cu_count * 3 / 4 ? 128
                         : mean <= 32                                          ? 32
                                                                               : 64;
        const int it = (int)items_of((size_t)n * top, E, rows);
        W8Rows r = {};
        r.codes = ws + o_x;
        r.step = (int64_t *)(ws + o_xs);
        r.X = X + t0 * dim;
        r.norm_w = norm_w;
        r.xn = norm_w ? (int64_t *)(ws + o_xn) : nullptr;
        if (base != out) {
            r.out = out + t0 * dim;
            r.base = base ? base + t0 * dim : nullptr;
        }
        r.T = n;
        r.K = dim;
        int *ch = chosen ? chosen + t0 * top : (int *)(ws + o_c);
        int64_t *wt = weight ? weight + t0 * top : (int64_t *)(ws + o_w);
        int64_t *lg = (int64_t *)(ws + o_l);
        int4 *items = (int4 *)(ws + o_i);
        int *tok = (int *)(ws + o_t);
        int64_t *sw = (int64_t *)(ws + o_sw);
        const MoeSlots s = {items, tok, sw, sl, it, rows};
        const bool one = n == 1 && q48_w8_one_ok(ffn);   // every item a slot
        const int per = route_per(c, n, E, dim);
        if (per) {
            int spl = 4;
            while ((per << spl) > 16)
                --spl;
            int p2 = 6;
            while ((1 << p2) < E)
                ++p2;
            const MoeRoute a = {r, moe->router, lg, E, per, spl, p2, top, moe->renorm, one, ch,
                                wt, (int *)ws, s};
            rc = launch_route(c, a);
        } else {
            if ((rc = q48_launch_w8_rows(c, r)))
                return launch_rc(rc);
            const int64_t *xr = norm_w ? r.xn : r.X;
            rc = n == 1 ? launch_rc(q48_launch_gemv(c, lg, moe->router, xr, E, dim))
                        : q48_launch_gemm_i8(c, lg, moe->router, xr, n, E, dim, Q48_GEMM_AUTO,
                                             nullptr);
            if (rc)
                return rc < 0 ? rc : launch_rc(rc);
#define MOE_CHOOSE(PER)                                                                        \
    hipLaunchKernelGGL(k_moe_choose<PER>, dim3((n + 3) / 4), dim3(256), 0, c->stream, lg, n, E, \
                       top, moe->renorm, ch, wt)
            if (E <= 64)
                MOE_CHOOSE(1);
            else if (E <= 128)
                MOE_CHOOSE(2);
            else
                MOE_CHOOSE(16);
#undef MOE_CHOOSE
            hipLaunchKernelGGL(k_moe_slots, dim3(1), dim3(1024), 0, c->stream, ch, wt, n * top, top,
                               E, s);
            rc = (int)hipGetLastError();
        }
        if (rc)
            return launch_rc(rc);
        W8Mul m = {};
        m.A = (const uint8_t *)g.codes;
        m.A2 = (const uint8_t *)u.codes;
        m.sw = g.step;
        m.sw2 = u.step;
        m.a_stride = w8_tiles(ffn, dim);
        m.N = ffn;
        m.KT = w8_kt(dim);
        m.B = r.codes;
        m.sb = r.step;
        m.T = n;
        m.rows = rows;
        m.Y = (int64_t *)(ws + o_h);
        m.items = items;
        m.slot_tok = tok;
        m.slot_w = sw;
        if ((rc = one ? q48_launch_w8_one(c, m, 1, nullptr, nullptr, dim, top)
                      : q48_launch_w8_mul(c, m, 1, true, it)))
            return launch_rc(rc);
        W8Rows h = {};
        h.codes = ws + o_hc;
        h.step = (int64_t *)(ws + o_hs);
        h.X = m.Y;
        h.tok = tok;
        h.T = sl;
        h.K = ffn;
        if (!one && (rc = q48_launch_w8_rows(c, h)))
            return launch_rc(rc);
        m.A = (const uint8_t *)d.codes;
        m.A2 = nullptr;
        m.sw = d.step;
        m.sw2 = nullptr;
        m.a_stride = w8_tiles(dim, ffn);
        m.N = dim;
        m.KT = w8_kt(ffn);
        m.B = h.codes;
        m.sb = h.step;
        m.Y = out + t0 * dim;
        if ((rc = one ? q48_launch_w8_one(c, m, 2, h.X, nullptr, ffn, top)
                      : q48_launch_w8_mul(c, m, 2, true, it)))
            return launch_rc(rc);
    }
    return Q48_OK;
}

} // extern "C"
