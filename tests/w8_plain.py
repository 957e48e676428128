"""Plain forms of the ops over weights in 8 bits and of the mixture-of-experts layer for
the tests: Python integers of any length, and the CPU oracle's rmsnorm and SiLU.
Nothing in the product imports this module.
"""
from __future__ import annotations

import numpy as np

import oracle_lib as O
import serve_plain as P

ONE = P.ONE
M64 = 1 << 64


def wrap(a):
    """Integers of any length as 64-bit words."""
    return np.asarray((np.asarray(a, dtype=object) + (1 << 63)) % M64 - (1 << 63)).astype(np.int64)


def rmsnorm(x, w):
    x, w = np.ascontiguousarray(x), np.ascontiguousarray(w)
    out = np.empty_like(x)
    for t in range(x.shape[0]):
        O.load().q48o_rmsnorm(out[t].ctypes.data, x[t].ctypes.data, w.ctypes.data, x.shape[1])
    return out


def silu_mul(g, u):
    g, u = np.ascontiguousarray(g), np.ascontiguousarray(u)
    out = np.empty_like(g)
    O.load().q48o_silu_mul(out.ctypes.data, g.ctypes.data, u.ctypes.data, g.size)
    return out


def quantise(x):
    """Codes and steps of rows of words [.., K] (the quantised cache's rule at 8 bits)."""
    return P.quantise(x, 8)


def values(codes, steps):
    return wrap(codes.astype(object) * steps.astype(object)[..., None])


def tiles(codes):
    """The bytes of a matrix's codes [N][K] as the library lays them out."""
    N, K = codes.shape
    NT, KT = (N + 15) // 16, (K + 63) // 64
    full = np.zeros((16 * NT, 64 * KT), dtype=np.int8)
    full[:N, :K] = codes
    return full.reshape(NT, 16, KT, 4, 16).transpose(0, 2, 3, 1, 4).reshape(-1).copy()


def times(codes, steps, w, w_steps):
    """floor(S sa sw / 2^48) as integers of any length: codes [T][K], w [N][K]."""
    S = codes.astype(np.int64) @ w.astype(np.int64).T
    return S.astype(object) * steps.astype(object)[:, None] * w_steps.astype(object)[None] >> 48


def product(X, norm_w, w, w_steps, base=None):
    x = X if norm_w is None else rmsnorm(X, norm_w)
    y = times(*quantise(x), w, w_steps)
    return wrap(y if base is None else y + base.astype(object))


def swiglu(X, norm_w, gate, up):
    """gate, up: (codes, steps)"""
    x = X if norm_w is None else rmsnorm(X, norm_w)
    c, s = quantise(x)
    return silu_mul(wrap(times(c, s, *gate)), wrap(times(c, s, *up)))


def choose(logits, top, renorm):
    """Chosen experts and weights of one row of logits."""
    l = [int(v) for v in logits]
    m = max(l)
    ids = sorted(range(len(l)), key=lambda i: (-l[i], i))
    e = {i: P.expn(m - l[i]) for i in ids}
    z = sum(e[i] for i in (ids[:top] if renorm else ids))
    return ids[:top], [(e[i] << 48) // z for i in ids[:top]]


def logits(x, router):
    """matmul_vec of every row."""
    return wrap(x.astype(object) @ router.astype(object).T >> 48)


def moe(X, norm_w, router, gate, up, down, top, renorm, base=None):
    """gate, up, down: (codes [E][N][K], steps [E][N]); out, chosen, weight."""
    x = X if norm_w is None else rmsnorm(X, norm_w)
    lg = logits(x, router)
    T = X.shape[0]
    out = np.zeros(X.shape, dtype=object) if base is None else base.astype(object)
    chosen = np.zeros((T, top), dtype=np.int32)
    weight = np.zeros((T, top), dtype=np.int64)
    cache = {}
    for t in range(T):
        chosen[t], weight[t] = choose(lg[t], top, renorm)
    for e in np.unique(chosen):
        at = np.nonzero((chosen == e).any(1))[0]
        h = swiglu(x[at], None, (gate[0][e], gate[1][e]), (up[0][e], up[1][e]))
        y = product(h, None, down[0][e], down[1][e])
        for i, t in enumerate(at):
            cache[t, int(e)] = y[i]
    for t in range(T):
        for e, w in zip(chosen[t], weight[t]):
            out[t] = out[t] + (int(w) * cache[t, int(e)].astype(object) >> 48)
    return wrap(out), chosen, weight
