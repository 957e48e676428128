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

// A wave a token: k times the largest logit not yet taken, the lowest expert of equal
// ones; then the weights.
__global__ __launch_bounds__(256) void k_moe_choose(const int64_t *__restrict__ logits, int T,
                                                   int E, int top, int renorm,
                                                   int *__restrict__ chosen,
                                                   int64_t *__restrict__ weight)
{
    q48_round_down();
    const int lane = threadIdx.x & 63, t = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= T)
        return;
    const int64_t *l = logits + (size_t)t * E;
    uint32_t taken = 0;   // bit i: expert lane + 64 i
    int64_t m = 0, sum = 0, mine = 0;
    int my_id = 0;
    for (int j = 0; j < top; ++j) {
        int64_t best = INT64_MIN;
        int id = E;   // none left: past every id
        for (int i = 0; lane + 64 * i < E; ++i) {
            const int64_t v = l[lane + 64 * i];
            if (!((taken >> i) & 1) && (id == E || v > best)) {
                best = v;
                id = lane + 64 * i;
            }
        }
        const int64_t at = q48_wave_max64(best);
        const int won = (int)-q48_wave_max64(best == at && id < E ? -(int64_t)id : -(int64_t)E);
        if (id == won)
            taken |= 1u << (won >> 6);
        if (j == 0)
            m = at;
        const int64_t e = q48_expn((uint64_t)m - (uint64_t)at);
        if (renorm)
            sum += e;
        if (lane == j) {
            mine = e;
            my_id = won;
        }
    }
    if (!renorm) {
        for (int i = lane; i < E; i += 64)
            sum += q48_expn((uint64_t)m - (uint64_t)l[i]);
        sum = q48_wave_sum64(sum);
    }
    if (lane < top) {
        chosen[(size_t)t * top + lane] = my_id;
        weight[(size_t)t * top + lane] = q48_div(mine, sum);
    }
}

// One block: the pairs counted by expert, each expert's first slot, the items of 16
// slots, and every pair into its slot.
__global__ __launch_bounds__(1024) void k_moe_slots(const int *__restrict__ chosen,
                                                   const int64_t *__restrict__ weight, int pairs,
                                                   int top, int E, int slots, int n_items,
                                                   int4 *__restrict__ items,
                                                   int *__restrict__ slot_tok,
                                                   int64_t *__restrict__ slot_w)
{
    __shared__ int count[W8_MAX_COUNT], first[W8_MAX_COUNT + 1];
    const int tid = threadIdx.x;
    count[tid] = 0;
    for (int i = tid; i < slots; i += 1024)
        slot_tok[i] = -1;
    for (int i = tid; i < n_items; i += 1024)
        items[i] = make_int4(0, 0, 0, 0);
    __syncthreads();
    for (int i = tid; i < pairs; i += 1024)
        atomicAdd(&count[chosen[i]], 1);
    __syncthreads();
    if (tid == 0) {
        int s = 0;
        for (int e = 0; e < E; ++e) {
            first[e] = s;
            s += (count[e] + 15) & ~15;
        }
        first[E] = s;
    }
    __syncthreads();
    if (tid < E)
        for (int s = 0; s < count[tid]; s += 16)
            items[(first[tid] + s) >> 4] =
                make_int4(tid, first[tid] + s, min(16, count[tid] - s), 0);
    __syncthreads();
    if (tid < E)
        count[tid] = 0;
    __syncthreads();
    for (int i = tid; i < pairs; i += 1024) {
        const int e = chosen[i], s = first[e] + atomicAdd(&count[e], 1);
        slot_tok[s] = i / top;
        slot_w[s] = weight[i];
    }
}

int launch_rc(int e) { return e == (int)hipSuccess ? Q48_OK : Q48_EHIP; }

// slots that n pairs of at most E experts can take, in sixteens
size_t moe_slots(size_t pairs, int E)
{
    return (pairs + 15 * (pairs < (size_t)E ? pairs : (size_t)E) + 15) & ~(size_t)15;
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
    size_t o = 0;
    auto take = [&](size_t bytes) {
        const size_t at = o;
        o += (bytes + 255) & ~(size_t)255;
        return at;
    };
    // tokens of one pass: a GiB of hidden words and 2^19 pairs at most
    size_t Tc = ((size_t)1 << 30) / ((size_t)16 * top * ffn);
    Tc = Tc < ((size_t)1 << 19) / top ? Tc : ((size_t)1 << 19) / top;
    Tc = Tc < 16 ? 16 : Tc < (size_t)T ? Tc : (size_t)T;
    const size_t slots = moe_slots(Tc * top, E), n_items = slots / 16;
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
        const int sl = (int)moe_slots((size_t)n * top, E), it = sl / 16;
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
        if ((rc = q48_launch_w8_rows(c, r)))
            return launch_rc(rc);
        const int64_t *xr = norm_w ? r.xn : r.X;
        int64_t *lg = (int64_t *)(ws + o_l);
        rc = n == 1 ? launch_rc(q48_launch_gemv(c, lg, moe->router, xr, E, dim))
                    : q48_launch_gemm_i8(c, lg, moe->router, xr, n, E, dim, Q48_GEMM_AUTO, nullptr);
        if (rc)
            return rc < 0 ? rc : launch_rc(rc);
        int *ch = chosen ? chosen + t0 * top : (int *)(ws + o_c);
        int64_t *wt = weight ? weight + t0 * top : (int64_t *)(ws + o_w);
        hipLaunchKernelGGL(k_moe_choose, dim3((n + 3) / 4), dim3(256), 0, c->stream, lg, n, E, top,
                           moe->renorm, ch, wt);
        int4 *items = (int4 *)(ws + o_i);
        int *tok = (int *)(ws + o_t);
        int64_t *sw = (int64_t *)(ws + o_sw);
        hipLaunchKernelGGL(k_moe_slots, dim3(1), dim3(1024), 0, c->stream, ch, wt, n * top, top, E,
                           sl, it, items, tok, sw);
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
        m.Y = (int64_t *)(ws + o_h);
        m.items = items;
        m.slot_tok = tok;
        m.slot_w = sw;
        if ((rc = q48_launch_w8_mul(c, m, 1, true, it)))
            return launch_rc(rc);
        W8Rows h = {};
        h.codes = ws + o_hc;
        h.step = (int64_t *)(ws + o_hs);
        h.X = m.Y;
        h.tok = tok;
        h.T = sl;
        h.K = ffn;
        if ((rc = q48_launch_w8_rows(c, h)))
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
        if ((rc = q48_launch_w8_mul(c, m, 2, true, it)))
            return launch_rc(rc);
    }
    return Q48_OK;
}

} // extern "C"
