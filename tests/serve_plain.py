"""Plain forms of the serving operators (quantised cache, attention under a mask,
log probabilities) for the tests: Python integers of any length, and the CPU
oracle's exact attention over the rows a query attends to.  Nothing in the product
imports this module.
"""
from __future__ import annotations

from decimal import Decimal, getcontext
from functools import lru_cache
from math import factorial

import numpy as np

import oracle_lib as O

ONE = 1 << 48
LN2 = 195103586505167
LEVELS = {8: 127, 4: 7}
I64_MAX = (1 << 63) - 1


def quantise(x, bits):
    """codes (int64 array) and steps of the head vectors x[..., hd] (int64)."""
    Q = LEVELS[bits]
    big = np.asarray(x).astype(object)
    a = abs(big).max(-1)
    step = np.minimum(-(-a // Q), I64_MAX // Q)
    by = np.where(step > 0, step, 1)[..., None]
    mag = np.minimum((abs(big) + step[..., None] // 2) // by, Q)
    code = np.where(big < 0, -mag, mag) * (step[..., None] > 0)
    return code.astype(np.int64), step.astype(np.int64)


def values(code, step):
    return (code.astype(object) * step.astype(object)[..., None]).astype(np.int64)


def pack(code, bits):
    """The bytes of codes[..., hd]."""
    if bits == 8:
        return code.astype(np.int8).view(np.uint8)
    h = code.shape[-1] // 2
    return ((code[..., :h] & 15) | ((code[..., h:] & 15) << 4)).astype(np.uint8)


def unpack(b, bits):
    if bits == 8:
        return b.view(np.int8).astype(np.int64)
    lo, hi = (b & 15).astype(np.int64), (b >> 4).astype(np.int64)
    return np.concatenate([(lo ^ 8) - 8, (hi ^ 8) - 8], -1)


def attend(q, K, V, sees):
    """q [T][nh][hd] over K, V [S][nkv][hd] where sees [T][S]: the oracle's exact
    attention over the rows each query sees, in order; zeros for none."""
    T, nh, hd = q.shape
    nkv = K.shape[1]
    out = np.zeros((T, nh, hd), dtype=np.int64)
    for t in range(T):
        at = np.nonzero(sees[t])[0]
        if not at.size:
            continue
        k, v = np.ascontiguousarray(K[at]), np.ascontiguousarray(V[at])
        qt, kn, vn = np.ascontiguousarray(q[t]), k[-1].copy(), v[-1].copy()
        o = np.zeros((nh, hd), dtype=np.int64)
        O.load().q48o_attn_decode(o.ctypes.data, qt.ctypes.data, k.ctypes.data, v.ctypes.data,
                                  kn.ctypes.data, vn.ctypes.data, 0, at.size - 1, nh, nkv, hd,
                                  at.size)
        out[t] = o
    return out


def mask_words(sees):
    """[T][n] truth values as [T][ceil(n / 64)] words."""
    T, n = sees.shape
    W = (n + 63) // 64
    bits = np.zeros((T, 64 * W), dtype=np.uint8)
    bits[:, :n] = sees
    return np.ascontiguousarray(np.packbits(bits, axis=1, bitorder="little").view("<i8"))


def tree(rng, T, pad=0):
    """Ancestors (and itself) of every node of a random tree of T nodes, parents
    before children; the last `pad` rows see nothing.  Also the nodes' parents."""
    sees = np.zeros((T, T), dtype=bool)
    parent = [-1]
    sees[0, 0] = True
    for t in range(1, T):
        p = int(rng.integers(max(-1, t - 5), t))
        parent.append(p)
        if p >= 0:
            sees[t] = sees[p]
        sees[t, t] = True
    if pad:
        sees[T - pad:] = False
    return sees, parent


def rope(x, cos_t, sin_t, pos):
    """rope_apply of head vectors x[..., hd] at pos."""
    v = np.ascontiguousarray(x).copy()
    flat = v.reshape(-1, v.shape[-1])
    for i in range(flat.shape[0]):
        O.load().q48o_rope_apply(cos_t.ctypes.data, sin_t.ctypes.data, v.shape[-1] // 2,
                                 flat[i].ctypes.data, pos)
    return v


def rope_tables(hd, max_seq, theta=10000):
    c = np.empty((max_seq, hd // 2), dtype=np.int64)
    s = np.empty_like(c)
    O.load().q48o_rope_tables(c.ctypes.data, s.ctypes.data, hd, max_seq, theta)
    return c, s


@lru_cache(None)
def tables():
    getcontext().prec = 60
    r = lambda x: int((x * ONE).to_integral_value())  # noqa: E731
    return ([r((Decimal(-j) / 64).exp()) for j in range(45)],
            [r(1 / Decimal(factorial(k))) for k in range(7)],
            [(1 << 54) // (64 + j) for j in range(64)],
            [r((1 + Decimal(j) / 64).ln()) for j in range(64)],
            [r(1 / Decimal(k)) for k in range(1, 9)])


def expn(u):
    """e_i of one u (a Python integer)."""
    T, C, _, _, _ = tables()
    n, r = divmod(u, LN2)
    j, s = divmod(r, 1 << 42)
    h = C[6]
    for k in range(5, -1, -1):
        h = C[k] - (s * h >> 48)
    return (T[j] * h >> 48) >> min(n, 200)


def logsum(Z):
    _, _, R, L, D = tables()
    b = Z.bit_length() - 49
    z = Z >> b
    i = (z >> 42) - 64
    d = (z * R[i] >> 48) - ONE
    g = D[7]
    for k in range(6, -1, -1):
        g = D[k] - (d * g >> 48)
    return b * LN2 + L[i] + (d * g >> 48), b


def logprobs(x, tokens, top):
    """logp, entropy, ids, their log probabilities of rows x [T][V] (int64)."""
    T, V = x.shape
    logp, ent = [], []
    ids, tlp = np.zeros((T, top), dtype=np.int32), np.zeros((T, top), dtype=np.int64)
    seen = {}
    for t in range(T):
        row = [int(v) for v in x[t]]
        m = max(row)
        e = []
        for v in row:
            u = m - v
            if u not in seen:
                seen[u] = expn(u)
            e.append(seen[u])
        logz, b = logsum(sum(e))
        at = lambda i: max(-(m - row[i] + logz), -(1 << 63))  # noqa: E731
        tok = int(tokens[t])
        logp.append(at(tok) if 0 <= tok < V else 0)
        w = sum(a * (m - v) >> 48 for a, v in zip(e, row))
        ent.append(logz + ((w >> b) << 48) // (sum(e) >> b))
        best = sorted(range(V), key=lambda i: (-row[i], i))[:top]
        ids[t] = best
        tlp[t] = [at(i) for i in best]
    return np.array(logp, dtype=np.int64), np.array(ent, dtype=np.int64), ids, tlp
