"""The serving operators around the Q16.48 forward pass, and their plain forms.

A quantised key/value cache (written and read back), attention over it, attention
of a tree of drafted tokens, and log probabilities of given tokens.  Every result
is an integer (Q16.48 words, codes, token ids) defined by integer steps, so a
kernel has to give the plain form's words.  `run` computes them with elementary
torch operations, or with `own` through the entry points of include/intllm_hip.h
by way of the ctypes bindings in int-llm_amd/intllm.

Values are Q16.48: the integer v stands for v / 2^48.
"""
import math
import os
import sys
from decimal import Decimal, getcontext

import numpy as np
import torch

own = False

ONE = 1 << 48
LN2 = 195103586505167       # round(2^48 ln 2)
DEV = "cuda:0"
LEVELS = {8: 127, 4: 7}     # the largest code of a quantised cache

# n_heads, n_kv_heads, head_dim of the TinyLlama shape
LLAMA = dict(nh=32, nkv=4, hd=64)


def listed():
    return [
        # one decoded token's key and value into a layer's cache and back: launches are all of it
        dict(name="cache_token_q8", kind="cache", bits=8, nkv=4, hd=64, T=1, p0=700, max_seq=2048),
        # a long prompt's rows, ragged, at 4 bits
        dict(name="cache_prompt_q4", kind="cache", bits=4, nkv=8, hd=128, T=1999, p0=3,
             max_seq=2048),
        # one decoded token in a chat-sized context
        dict(name="decode_q8_short", kind="decode", bits=8, **LLAMA, pos=120, max_seq=2048),
        # the same at 4 bits with 128-wide heads, a few thousand positions
        dict(name="decode_q4_mid", kind="decode", bits=4, nh=32, nkv=8, hd=128, pos=2060,
             max_seq=4096),
        # and over a very long cache
        dict(name="decode_q8_long", kind="decode", bits=8, **LLAMA, pos=16000, max_seq=16384),
        # a later chunk of a long prompt over a quantised cache
        dict(name="prompt_q8", kind="rows", bits=8, **LLAMA, T=384, p0=512, tree=False,
             max_seq=2048),
        # verifying a tree of drafted tokens over a quantised cache
        dict(name="tree_q8", kind="rows", bits=8, **LLAMA, T=26, p0=2047, tree=True,
             max_seq=4096),
        # a few drafted tokens of the tiny model, int64 cache
        dict(name="tree_tiny", kind="rows", bits=64, nh=8, nkv=2, hd=32, T=7, p0=40, tree=True,
             max_seq=256),
        # a wide tree over a long int64 cache
        dict(name="tree_long", kind="rows", bits=64, **LLAMA, T=48, p0=4000, tree=True,
             max_seq=4096),
        # one decoded token's log probability with the twenty best alternatives
        dict(name="logprobs_token", kind="logprobs", T=1, V=32000, top=20),
        # scoring a prompt
        dict(name="logprobs_prompt", kind="logprobs", T=500, V=32000, top=5),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["cache", "decode", "decode", "rows", "rows", "rows", "logprobs",
                       "logprobs"])
    if kind == "logprobs":
        V = _logint(rng, 300, 130000)
        return dict(kind=kind, T=_logint(rng, 1, min(512, (1 << 24) // V)), V=V,
                    top=rng.choice([0, 1, 5, 20, 32]))
    hd = rng.choice([32, 64, 64, 128])
    nkv = rng.choice([1, 2, 4, 8])
    if kind == "cache":
        T = _logint(rng, 1, 2048)
        p0 = rng.randrange(0, 1000)
        return dict(kind=kind, bits=rng.choice([8, 4]), nkv=nkv, hd=hd, T=T, p0=p0,
                    max_seq=T + p0 + rng.randrange(0, 100))
    nh = nkv * rng.choice([1, 2, 4, 7, 8])
    if kind == "decode":
        pos = _logint(rng, 1, 16000) - 1
        return dict(kind=kind, bits=rng.choice([8, 4]), nh=min(nh, 32) // nkv * nkv, nkv=nkv,
                    hd=hd, pos=pos, max_seq=pos + 1 + rng.randrange(0, 300))
    nh = min(nh, 32) // nkv * nkv
    tree = rng.random() < 0.6
    p0 = rng.choice([0, _logint(rng, 1, 4000)])
    # row x position x dim x head products at most those of tree_long
    room = 48 * 4048 * 32 * 64 // (nh * hd)
    T = _logint(rng, 1, 64 if tree else 512)
    while T * (p0 + T) > room:
        T -= 1
    return dict(kind=kind, bits=rng.choice([8, 4, 64]), nh=nh, nkv=nkv, hd=hd, T=T, p0=p0,
                tree=tree, max_seq=p0 + T + rng.randrange(0, 64))


# ---- inputs --------------------------------------------------------------------

_context = None


def _ctx():
    """A program's one context, on the stream that its torch operations use: calls take
    their turn among them."""
    global _context
    if _context is None:
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                           "int-llm_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import intllm
        _context = intllm.Context(0, stream=torch.cuda.current_stream(DEV).cuda_stream)
    return _context


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) & ((1 << 62) - 1))


def _acts(g, *shape, sigma=1.0):
    """Activations: every fraction bit in use."""
    return (torch.randn(shape, generator=g, device=DEV, dtype=torch.float64) * (sigma * ONE)).to(
        torch.int64)


def _tree_mask(T, seed, p0):
    """The ancestors (and itself) of every node of a random draft tree, one bit
    a node; a batch's padding rows at the end attend to nothing drafted."""
    rng = np.random.RandomState((int(seed) ^ 77) & 0x7FFFFFFF)
    sees = np.zeros((T, T), dtype=bool)
    for t in range(T):
        if t:
            parent = rng.randint(max(-1, t - 6), t)
            if parent >= 0:
                sees[t] = sees[parent]
        sees[t, t] = True
    if T > 4:
        sees[T - 1] = False
    return sees


def _words(sees):
    """A [T][T] table of truth values as [T][ceil(T / 64)] 64-bit masks."""
    T = sees.shape[0]
    W = (T + 63) // 64
    bits = np.zeros((T, 64 * W), dtype=np.uint8)
    bits[:, :T] = sees
    return np.packbits(bits, axis=1, bitorder="little").view("<i8").reshape(T, W)


def prepare(case, seed):
    kind, g = case["kind"], _gen(seed)
    s = dict(case=case)
    if kind == "logprobs":
        T, V = case["T"], case["V"]
        s["logits"] = _acts(g, T, V, sigma=2.5)
        peak = torch.randint(0, V, (T, 4), generator=g, device=DEV)
        s["logits"].scatter_add_(1, peak, _acts(g, T, 4, sigma=8.0))
        s["tokens"] = torch.randint(0, V, (T,), generator=g, device=DEV, dtype=torch.int32)
        if T > 3:
            s["tokens"][T // 2] = -1          # a padded row scores no token
        s["logp"], s["entropy"] = _zeros(T), _zeros(T)
        s["top_logp"] = _zeros(T, case["top"])
        s["top_ids"] = torch.zeros(T, case["top"], dtype=torch.int32, device=DEV)
        return s
    nkv, hd, bits, max_seq = case["nkv"], case["hd"], case["bits"], case["max_seq"]
    if kind == "cache":
        T = case["T"]
        s["K"], s["V"] = _acts(g, T, nkv, hd), _acts(g, T, nkv, hd, sigma=0.3)
        s["K"][:, :, 0] *= 6                  # one channel far above the others
        s["V"][T // 2, 0] = 0                 # and a head of zeros
        s["Kout"], s["Vout"] = _zeros(T, nkv, hd), _zeros(T, nkv, hd)
        s.update(_empty_cache(case))
        return s
    nh, T = case["nh"], case.get("T", 1)
    rows = case["pos"] if kind == "decode" else case["p0"] + T
    K, V = _acts(g, max_seq, nkv, hd), _acts(g, max_seq, nkv, hd)
    K[rows:], V[rows:] = 0, 0
    if bits == 64:
        s["kc"], s["vc"] = K, V
    else:
        s.update(_empty_cache(case))
        for x, codes, steps in ((K, "k", "k_step"), (V, "v", "v_step")):
            c, st = _quantise(x, bits)
            s[codes].copy_(_pack(c, bits))
            s[steps].copy_(st)
    if kind == "decode":
        s["q"] = _acts(g, nh, hd, sigma=1.5)
        s["k_new"], s["v_new"] = _acts(g, nkv, hd), _acts(g, nkv, hd)
        s["out"] = _zeros(nh, hd)
    else:
        s["QKV"] = _acts(g, T, nh + 2 * nkv, hd, sigma=1.5)
        s["out"] = _zeros(T, nh, hd)
        s["mask"] = None
        if case["tree"]:
            s["mask"] = torch.from_numpy(_words(_tree_mask(T, seed, case["p0"]))).to(DEV)
    return s


def _zeros(*shape):
    return torch.zeros(shape, dtype=torch.int64, device=DEV)


def _empty_cache(case):
    """A layer's quantised cache: codes and steps of its keys and values."""
    nkv, hd, max_seq = case["nkv"], case["hd"], case["max_seq"]
    code = lambda: torch.zeros(max_seq, nkv, hd * case["bits"] // 8, dtype=torch.int8,  # noqa: E731
                               device=DEV)
    return dict(k=code(), v=code(), k_step=_zeros(max_seq, nkv), v_step=_zeros(max_seq, nkv))


# ---- one pass --------------------------------------------------------------------

def run(s):
    case = s["case"]
    if own:
        return _own(s, case)
    return {"cache": _cache, "decode": _decode, "rows": _rows, "logprobs": _logprobs}[
        case["kind"]](s, case)


def _handles(s, case):
    """What a program keeps with its buffers: their addresses, and the cache's description."""
    p = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
    cache = None
    if case.get("bits", 64) != 64:
        cache = _ctx().qcache(p["k"], p["v"], p["k_step"], p["v_step"], case["bits"], 1,
                              case["max_seq"], case["nkv"], case["hd"])
    return p, cache


def _own(s, case):
    if "handles" not in s:
        s["handles"] = _handles(s, case)
    ctx, kind, (p, cache) = _ctx(), case["kind"], s["handles"]
    if kind == "logprobs":
        ctx.logprobs_rows(p["logits"], case["T"], case["V"], p["tokens"], p["logp"], p["entropy"],
                          case["top"], p["top_ids"], p["top_logp"])
        return [s["logp"], s["entropy"], s["top_ids"], s["top_logp"]]
    if kind == "cache":
        ctx.qcache_store_rows(cache, 0, case["p0"], case["T"], p["K"], p["V"],
                              case["nkv"] * case["hd"])
        ctx.qcache_load_rows(p["Kout"], p["Vout"], cache, 0, case["p0"], case["T"],
                             case["nkv"] * case["hd"])
        return [s["Kout"], s["Vout"], s["k_step"], s["v_step"]]
    if kind == "decode":
        ctx.attn_decode_qcache(p["out"], p["q"], cache, p["k_new"], p["v_new"], 0, case["pos"],
                               case["nh"])
        return [s["out"], s["k"], s["v"], s["k_step"], s["v_step"]]
    mask = p.get("mask")
    if case["bits"] == 64:
        ctx.attn_tree(p["out"], p["QKV"], p["kc"], p["vc"], 0, case["p0"], case["T"], case["nh"],
                      case["nkv"], case["hd"], case["max_seq"], mask)
    else:
        ctx.attn_rows_qcache(p["out"], p["QKV"], cache, 0, case["p0"], case["T"], case["nh"],
                             mask)
    return s["out"]


# ---- the plain forms ---------------------------------------------------------------

def _mul(a, b):
    """floor(a b / 2^48) for |a|, |b| < 2^61 (mod 2^64): halves of 24 bits."""
    ah, al, bh, bl = a >> 24, a & 0xFFFFFF, b >> 24, b & 0xFFFFFF
    return ah * bh + ((ah * bl + al * bh + ((al * bl) >> 24)) >> 24)


def _div(e, d):
    """floor(2^48 e / d) for 0 <= e < 16 d, d < 2^62: an estimate in float64,
    then the remainder in wrapping int64."""
    q = (e.double() * (float(ONE) / d.double())).to(torch.int64)
    for _ in range(2):
        r = (e << 48) - q * d
        q = q + (r >= d).to(torch.int64) - (r < 0).to(torch.int64)
    return q


def _exp(x):
    """fp_safe_exp of x <= 0: 14 squarings of 1 + |x| / 2^14 and a reciprocal;
    0 below -10."""
    m = (-x).clamp(max=10 * ONE)
    r = ONE + (m >> 14)
    for _ in range(14):
        r = _mul(r, r)
    q = (float(2.0 ** 96) / r.double()).to(torch.int64)
    rem = -(q * r)                            # 2^96 - q r, mod 2^64
    q = q + (rem >= r).to(torch.int64) - (rem < 0).to(torch.int64)
    return torch.where(x < -10 * ONE, torch.zeros_like(q), q)


def _dots(q, k):
    """(sum_d q[h][t][d] k[h][j][d]) >> 48 mod 2^64: products of 16-bit limbs in
    float64 (sums below 2^53, so exact), carried up in int64."""
    limbs = lambda v: [((v >> (16 * i)) & 0xFFFF).double() for i in range(3)] + [  # noqa: E731
        (v >> 48).double()]
    a, b = limbs(q), [w.transpose(1, 2).contiguous() for w in limbs(k)]
    out, acc = 0, 0
    for d in range(7):
        acc = acc + sum(torch.matmul(a[i], b[d - i]).to(torch.int64)
                        for i in range(4) if 0 <= d - i <= 3)
        if d >= 3:
            out = out + ((acc & 0xFFFF) << (16 * (d - 3)))
        acc = acc >> 16
    return out


def _attend(q, K, V, sees):
    """q [T][nh][hd] over K, V [S][nkv][hd] where sees [T][S]: [T][nh][hd]."""
    T, nh, hd = q.shape
    S, nkv, _ = K.shape
    G = nh // nkv
    scale = math.isqrt((1 << 96) // hd)       # floor(2^48 / sqrt(hd)): fp_inv_sqrt's value
    qk = q.reshape(T, nkv, G, hd).permute(1, 0, 2, 3).reshape(nkv, T * G, hd)
    s = _mul(_dots(qk, K.permute(1, 0, 2)), torch.full((), scale, device=DEV, dtype=torch.int64))
    s = s.reshape(nkv, T, G, S)
    see = sees[None, :, None, :]
    top = torch.where(see, s, torch.full_like(s, -(1 << 62))).amax(-1, keepdim=True)
    e = torch.where(see, _exp(torch.where(see, s - top, torch.zeros_like(s))), torch.zeros_like(s))
    z = e.sum(-1, keepdim=True)
    p = _div(e, z.clamp(min=1))
    v = V.permute(1, 0, 2)[:, None, None]     # nkv, 1, 1, S, hd
    o = _mul(p[..., None], v).sum(-2)         # nkv, T, G, hd
    return o.permute(1, 0, 2, 3).reshape(T, nh, hd)


def _quantise(x, bits):
    """Codes and steps of every head vector x[..., hd]."""
    Q = LEVELS[bits]
    top = x.abs().amax(-1)
    step = (top + (Q - 1)) // Q
    half, by = (step >> 1)[..., None], step.clamp(min=1)[..., None]
    code = ((x.abs() + half) // by).clamp(max=Q) * x.sign()
    return code, step


def _pack(code, bits):
    """Codes as the cache holds them: bytes, or at 4 bits dim b and dim b + hd/2
    in the low and high half of byte b."""
    if bits == 8:
        return code.to(torch.int8)
    h = code.shape[-1] // 2
    b = (code[..., :h] & 15) | ((code[..., h:] & 15) << 4)
    return torch.where(b > 127, b - 256, b).to(torch.int8)


def _unpack(packed, steps, bits):
    """The values a cache's codes and steps stand for."""
    c = packed.to(torch.int64)
    if bits == 4:
        c = torch.cat([((c & 15) ^ 8) - 8, c >> 4], -1)
    return c * steps[..., None]


def _cache(s, case):
    rows = slice(case["p0"], case["p0"] + case["T"])
    out = []
    for x, codes, steps in (("K", "k", "k_step"), ("V", "v", "v_step")):
        c, st = _quantise(s[x], case["bits"])
        s[codes][rows], s[steps][rows] = _pack(c, case["bits"]), st
        out.append(_unpack(s[codes][rows], s[steps][rows], case["bits"]))
    return [*out, s["k_step"], s["v_step"]]


def _values(s, case, n):
    if case["bits"] == 64:
        return s["kc"][:n], s["vc"][:n]
    return (_unpack(s["k"][:n], s["k_step"][:n], case["bits"]),
            _unpack(s["v"][:n], s["v_step"][:n], case["bits"]))


def _decode(s, case):
    pos = case["pos"]
    for x, codes, steps in (("k_new", "k", "k_step"), ("v_new", "v", "v_step")):
        c, st = _quantise(s[x], case["bits"])
        s[codes][pos], s[steps][pos] = _pack(c, case["bits"]), st
    K, V = _values(s, case, pos + 1)
    sees = torch.ones(1, pos + 1, dtype=torch.bool, device=DEV)
    return [_attend(s["q"][None], K, V, sees)[0], s["k"], s["v"], s["k_step"], s["v_step"]]


def _rows(s, case):
    T, p0 = case["T"], case["p0"]
    K, V = _values(s, case, p0 + T)
    j = torch.arange(T, device=DEV)
    if case["tree"]:
        new = (s["mask"][:, j >> 6] >> (j & 63)) & 1 > 0
    else:
        new = j[None, :] <= j[:, None]
    sees = torch.cat([torch.ones(T, p0, dtype=torch.bool, device=DEV), new], 1)
    return _attend(s["QKV"][:, :case["nh"]], K, V, sees)


def _tables():
    """T_j = round(2^48 e^(-j/64)), C_k = round(2^48 / k!), R_j = floor(2^48 64 / (64 + j)),
    L_j = round(2^48 log(1 + j/64)), D_k = round(2^48 / k)."""
    getcontext().prec = 50
    r = lambda x: int((x * ONE).to_integral_value())  # noqa: E731
    return ([r((Decimal(-j) / 64).exp()) for j in range(45)],
            [r(1 / Decimal(math.factorial(k))) for k in range(7)],
            [ONE * 64 // (64 + j) for j in range(64)],
            [r((1 + Decimal(j) / 64).ln()) for j in range(64)],
            [r(1 / Decimal(k)) for k in range(1, 9)])


_T, _C, _R, _L, _D = _tables()


def _expn(u):
    """e^-u for u >= 0: u = n LN2 + j / 64 + s, 2^-n T_j e^-s."""
    n = torch.div(u, LN2, rounding_mode="floor")
    r = u - n * LN2
    s = r & ((1 << 42) - 1)
    h = torch.full_like(s, _C[6])
    for c in _C[5::-1]:
        h = c - _mul(s, h)
    t = torch.tensor(_T, device=DEV, dtype=torch.int64)[r >> 42]
    return torch.where(n < 49, _mul(t, h) >> n.clamp(max=62), torch.zeros_like(u))


def _log_sum(z):
    """(log(z / 2^48), b): z >> b in [1, 2), log = b LN2 + L_j + log1p of what is left.
    z < 2^66, as (high, low) words of 48 bits."""
    hi, lo = z
    b = sum((hi >= (1 << k)).to(torch.int64) for k in range(1, 31))    # bitlen(z) - 49
    m = _shift(z, b)
    j = (m - ONE) >> 42
    table = lambda v: torch.tensor(v, device=DEV, dtype=torch.int64)[j]  # noqa: E731
    d = _mul(m, table(_R)) - ONE
    g = torch.full_like(d, _D[7])
    for c in _D[6::-1]:
        g = c - _mul(d, g)
    return b * LN2 + table(_L) + _mul(d, g), b


def _shift(z, b):
    """(high 2^48 + low) >> b"""
    hi, lo = z
    return (hi << (48 - b)) + (lo >> b)


def _sum48(x):
    """Sum over the last axis of values below 2^49, as (high, low) words of 48 bits."""
    lo, hi = (x & 0xFFFFFF).sum(-1), (x >> 24).sum(-1)
    hi = hi + (lo >> 24)
    return hi >> 24, ((hi & 0xFFFFFF) << 24) | (lo & 0xFFFFFF)


def _logprobs(s, case):
    x, top = s["logits"], case["top"]
    u = x.amax(-1, keepdim=True) - x
    e = _expn(u)
    z = _sum48(e)
    logz, b = _log_sum(z)
    eu = _sum48(_mul(e, u.clamp(max=64 * ONE)))
    ent = logz + _div(_shift(eu, b), _shift(z, b))
    t = s["tokens"].to(torch.int64)
    at = u.gather(1, t.clamp(min=0)[:, None])[:, 0]
    logp = torch.where(t >= 0, -(at + logz), torch.zeros_like(at))
    order = torch.sort(u, dim=-1, stable=True)
    ids = order.indices[:, :top]
    return [logp, ent, ids.to(torch.int32), -(order.values[:, :top] + logz[:, None])]


# ---- what a pass cannot do without ---------------------------------------------------

def work(case):
    """flops: two for each multiply-add of a score or a value, ten for a log
    probability's exponential, however the kernels make them."""
    kind = case["kind"]
    if kind == "logprobs":
        T, V = case["T"], case["V"]
        return {"bytes": 8 * T * V + T * (20 + 12 * case["top"]), "flops": 10 * T * V}
    nkv, hd = case["nkv"], case["hd"]
    row = nkv * (hd * case["bits"] // 8 + (8 if case["bits"] != 64 else 0))   # a key row's bytes
    if kind == "cache":
        T = case["T"]
        return {"bytes": 2 * T * (2 * 8 * nkv * hd + 2 * row), "flops": 4 * T * nkv * hd}
    nh = case["nh"]
    if kind == "decode":
        S = case["pos"] + 1
        return {"bytes": 2 * S * row + 16 * (nh + nkv) * hd, "flops": 4 * S * nh * hd}
    T, p0 = case["T"], case["p0"]
    pairs = T * p0 + T * (T + 1) // 2
    return {"bytes": 2 * (p0 + T) * row + 16 * T * nh * hd, "flops": 4 * pairs * nh * hd}


# ---- the definitions, in whole numbers of any length -----------------------------------

def _big(t):
    return t.cpu().numpy().astype(object)


def _big_quantise(x, bits):
    """Codes and steps, x an array of Python integers [..., hd]."""
    Q = LEVELS[bits]
    step = -(-abs(x).max(-1) // Q)
    by = np.where(step > 0, step, 1)[..., None]
    mag = np.minimum((abs(x) + step[..., None] // 2) // by, Q)
    return np.where(x < 0, -mag, mag) * (step > 0)[..., None], step


def _big_exp(x):
    r = np.minimum(-x, 10 * ONE) // (1 << 14) + ONE
    for _ in range(14):
        r = r * r // ONE
    return np.where(x < -10 * ONE, 0, (1 << 96) // r)


def _big_attend(q, K, V, sees):
    T, nh, hd = q.shape
    S, nkv, _ = K.shape
    scale = math.isqrt((1 << 96) // hd)
    out = np.zeros((T, nh, hd), dtype=object)
    for t in range(T):
        at = np.nonzero(sees[t])[0]
        for h in range(nh if at.size else 0):
            kh = h // (nh // nkv)
            sc = (K[at, kh] @ q[t, h] // ONE) * scale // ONE
            e = _big_exp(sc - sc.max())
            p = e * ONE // e.sum()
            out[t, h] = (p[:, None] * V[at, kh] // ONE).sum(0)
    return out


def _big_logprobs(x, tokens, top):
    T, V = x.shape
    logp, ent = np.zeros(T, dtype=object), np.zeros(T, dtype=object)
    ids, tops = np.zeros((T, top), dtype=np.int32), np.zeros((T, top), dtype=object)
    E, F, R, L, D = (np.array(v, dtype=object) for v in (_T, _C, _R, _L, _D))
    for t in range(T):
        u = x[t].max() - x[t]
        n, r = u // LN2, u % LN2
        s = r % (1 << 42)
        h = F[6]
        for k in range(5, -1, -1):
            h = F[k] - s * h // ONE
        e = (E[(r // (1 << 42)).astype(np.int64)] * h // ONE) // 2 ** np.minimum(n, 200)
        z = int(e.sum())
        b = z.bit_length() - 49
        m = z >> b
        j = (m - ONE) >> 42
        d = (m * R[j] >> 48) - ONE
        g = D[7]
        for k in range(6, -1, -1):
            g = D[k] - (d * g >> 48)
        logz = b * LN2 + L[j] + (d * g >> 48)
        logp[t] = -(u[tokens[t]] + logz) if tokens[t] >= 0 else 0
        ent[t] = logz + ((int((e * u // ONE).sum()) >> b) << 48) // m
        ids[t] = np.lexsort((np.arange(V), u))[:top]
        tops[t] = -(u[ids[t]] + logz)
    return [logp, ent, ids, tops]


def exact(case, seed):
    """The same outputs from the definitions, in Python's integers."""
    kind = case["kind"]
    if kind == "logprobs":
        if case["T"] * case["V"] > 500_000:
            return None
        s = prepare(case, seed)
        out = _big_logprobs(_big(s["logits"]), s["tokens"].cpu().numpy(), case["top"])
        return [v.astype(np.int64) if v.dtype == object else v for v in out]
    nkv, hd, bits = case["nkv"], case["hd"], case["bits"]
    if kind == "cache":
        if case["T"] * nkv * hd > 4_000_000:
            return None
        s = prepare(case, seed)
        values, steps = [], []
        for x in ("K", "V"):
            c, st = _big_quantise(_big(s[x]), bits)
            values.append((c * st[..., None]).astype(np.int64))
            whole = np.zeros((case["max_seq"], nkv), dtype=np.int64)
            whole[case["p0"]:case["p0"] + case["T"]] = st.astype(np.int64)
            steps.append(whole)
        return [*values, *steps]
    rows = case["pos"] + 1 if kind == "decode" else case["p0"] + case["T"]
    if case.get("T", 1) * rows * case["nh"] * hd > 12_000_000:
        return None
    s = prepare(case, seed)
    if bits == 64:
        K, V = _big(s["kc"][:rows]), _big(s["vc"][:rows])
    else:
        K, V = [], []
        for vals, codes, steps in ((K, "k", "k_step"), (V, "v", "v_step")):
            c, st = _big(s[codes][:rows]), _big(s[steps][:rows])
            if bits == 4:
                low = c % 16
                c = np.concatenate([low - 16 * (low > 7), c // 16], -1)
            vals.append(c * st[..., None])
        K, V = K[0], V[0]
    if kind == "rows":
        T, p0 = case["T"], case["p0"]
        new = _tree_mask(T, seed, p0) if case["tree"] else np.tri(T, dtype=bool)
        sees = np.concatenate([np.ones((T, p0), dtype=bool), new], 1)
        return _big_attend(_big(s["QKV"][:, :case["nh"]]), K, V, sees).astype(np.int64)
    for vals, x in ((K, "k_new"), (V, "v_new")):
        c, st = _big_quantise(_big(s[x]), bits)
        vals[case["pos"]] = c * st[..., None]
    out = _big_attend(_big(s["q"])[None], K, V, np.ones((1, rows), dtype=bool))[0]
    return [out.astype(np.int64), None, None, None, None]
