"""A small model with 8-bit projections and mixture-of-experts layers, as a program runs it:
a prompt in one pass and the same tokens one at a time give the same words, and the
plain form's.
"""
import ctypes as C

import numpy as np
import pytest

import intllm
import serve_plain as P
import w8_plain as W
from test_gpu_w8 import loaded, own, weights, words  # noqa: F401

pytestmark = pytest.mark.gpu

DIM, NH, NKV, HD, L, E, TOP, FFN, VOCAB, MAX_SEQ = 256, 8, 2, 32, 2, 6, 2, 96, 300, 64
QKV = (NH + 2 * NKV) * HD
_V, _I = C.c_void_p, C.c_int


def raw(name, *types):
    f = getattr(intllm.hip_lib(), name)
    f.argtypes, f.restype = [_V, *types], C.c_int
    return lambda ctx, *a: intllm.check(name, f(ctx.h, *a))


attn_prefill = raw("q48_attn_prefill", _V, _V, _V, _V, _I, _I, _I, _I, _I, _I, _I)
rope_store_rows = raw("q48_rope_store_rows", _V, _V, _V, _I, _I, _I, _I, _I, _I, _I)


class Model:
    def __init__(self, ctx, rng):
        self.ctx = ctx
        norm = lambda: W.ONE + words(rng, DIM, sigma=0.1)  # noqa: E731
        self.host = []
        self.layers = []
        for _ in range(L):
            h = dict(an=norm(), fn=norm(), qkv=weights(rng, QKV, DIM, sigma=0.06),
                     o=weights(rng, DIM, DIM, sigma=0.06), router=words(rng, E, DIM, sigma=0.1),
                     gate=weights(rng, E, FFN, DIM, sigma=0.06), up=weights(rng, E, FFN, DIM, sigma=0.06),
                     down=weights(rng, E, DIM, FFN, sigma=0.1))
            d = {k: ctx.to_device(v) for k, v in h.items() if not isinstance(v, tuple)}
            d.update({k: loaded(ctx, *v) for k, v in h.items() if isinstance(v, tuple)})
            d["moe"] = ctx.moe(d["router"].ptr, d["gate"], d["up"], d["down"], TOP, True)
            self.host.append(h)
            self.layers.append(d)
        self.norm, self.head = norm(), weights(rng, VOCAB, DIM, sigma=0.06)
        self.dnorm, self.dhead = ctx.to_device(self.norm), loaded(ctx, *self.head)
        n = L * MAX_SEQ * NKV * HD
        self.kc, self.vc = ctx.to_device(np.zeros(n)), ctx.to_device(np.zeros(n))

    def forward(self, x, p0):
        """Logits of rows x at positions p0 on."""
        c, T = self.ctx, x.shape[0]
        h = c.to_device(x)
        qkv, att, lg = c.buffer(T * QKV), c.buffer(T * DIM), c.buffer(T * VOCAB)
        for i, d in enumerate(self.layers):
            c.gemm_w8(qkv.ptr, None, d["qkv"], h.ptr, d["an"].ptr, T)
            rope_store_rows(c, qkv.ptr, self.kc.ptr, self.vc.ptr, i, p0, T, NH, NKV, HD, MAX_SEQ)
            attn_prefill(c, att.ptr, qkv.ptr, self.kc.ptr, self.vc.ptr, i, p0, T, NH, NKV, HD, MAX_SEQ)
            c.gemm_w8(h.ptr, h.ptr, d["o"], att.ptr, None, T)
            c.moe_w8(h.ptr, h.ptr, d["moe"], h.ptr, d["fn"].ptr, T)
        c.gemm_w8(lg.ptr, None, self.dhead, h.ptr, self.dnorm.ptr, T)
        return lg.download().reshape(T, VOCAB)

    def plain(self, x):
        cos, sin = P.rope_tables(HD, MAX_SEQ)
        T = x.shape[0]
        for d in self.host:
            q = W.product(x, d["an"], *d["qkv"]).reshape(T, NH + 2 * NKV, HD)
            rot = np.stack([P.rope(q[t, :NH + NKV], cos, sin, t) for t in range(T)])
            att = P.attend(rot[:, :NH], rot[:, NH:], q[:, NH + NKV:], np.tri(T, dtype=bool))
            x = W.product(att.reshape(T, DIM), None, *d["o"], base=x)
            x = W.moe(x, d["fn"], d["router"], d["gate"], d["up"], d["down"], TOP, True, x)[0]
        return W.product(x, self.norm, *self.head)


def test_a_prompt_in_one_pass_and_token_by_token(own):  # noqa: F811
    rng = np.random.default_rng(12)
    intllm.check("rope", intllm.hip_lib().q48_rope_init(own.h, HD, MAX_SEQ, 10000))
    m = Model(own, rng)
    x = words(rng, 21, DIM)
    whole = m.forward(x, 0)
    assert (whole == m.plain(x)).all()
    one = np.concatenate([m.forward(x[t:t + 1], t) for t in range(21)])
    assert (one == whole).all()
    parts = np.concatenate([m.forward(x[:5], 0), m.forward(x[5:20], 5), m.forward(x[20:], 20)])
    assert (parts == whole).all()
