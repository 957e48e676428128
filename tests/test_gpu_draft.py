"""The serving operators together, as a program that drafts and verifies uses them:
a prompt into the cache, a tree of drafted tokens in one pass, the accepted path's
rows kept, log probabilities of what was drafted, and decoding on.

With the int64 cache every logits row equals the C host's forward call by call; with
a quantised cache the tree's rows equal decoding its paths token by token over the
same cache.
"""
import ctypes as C

import numpy as np
import pytest

import intllm
import serve_plain as P

pytestmark = pytest.mark.gpu

DIM, NH, NKV, HD, L, FFN, VOCAB, MAX_SEQ = 256, 8, 2, 32, 2, 688, 512, 256
KVD = NKV * HD
_V, _I = C.c_void_p, C.c_int


def raw(name, *types):
    f = getattr(intllm.hip_lib(), name)
    f.argtypes, f.restype = [_V, *types], C.c_int
    return lambda ctx, *a: intllm.check(name, f(ctx.h, *a))


norm_rows = raw("q48_rmsnorm_rows", _V, _V, _V, _I, _I)
silu_rows = raw("q48_silu_mul_rows", _V, _V, _I, _I)
embed_rows = raw("q48_embed_rows", _V, _V, _V, _I, _I)


def ints(ctx, a):
    a = np.asarray(a, dtype=np.int32).ravel()
    return ctx.to_device(np.concatenate([a, np.zeros(a.size % 2, np.int32)]).view(np.int64))


class Tiny:
    """A two-layer Llama's weights on the device, and its forward over T rows."""

    def __init__(self, ctx, bits, rng):
        self.ctx, self.bits, self.host_weights = ctx, bits, {}
        w = lambda name, n, m, mean=0.0, s=0.05: self._weight(rng, name, n, m, mean, s)  # noqa: E731
        self.embed = w("model.embed_tokens.weight", VOCAB, DIM, s=1.0)
        self.norm = w("model.norm.weight", 1, DIM, 1.0)
        self.head = w("lm_head.weight", VOCAB, DIM)
        self.layers = []
        for i in range(L):
            p = f"model.layers.{i}."
            an = w(p + "input_layernorm.weight", 1, DIM, 1.0)
            fn = w(p + "post_attention_layernorm.weight", 1, DIM, 1.0)
            qkv = self._stack(rng, [(p + "self_attn.q_proj.weight", DIM),
                                    (p + "self_attn.k_proj.weight", KVD),
                                    (p + "self_attn.v_proj.weight", KVD)], DIM)
            wo = w(p + "self_attn.o_proj.weight", DIM, DIM)
            gu = self._stack(rng, [(p + "mlp.gate_proj.weight", FFN),
                                   (p + "mlp.up_proj.weight", FFN)], DIM)
            wd = w(p + "mlp.down_proj.weight", DIM, FFN)
            self.layers.append((an, qkv, wo, fn, gu, wd))
        if bits == 64:
            self.kc, self.vc = (ctx.to_device(np.zeros(L * MAX_SEQ * KVD, np.int64))
                                for _ in range(2))
        else:
            self.cache = ctx.new_qcache(bits, L, MAX_SEQ, NKV, HD)
        self.buf = {k: ctx.buffer(64 * n) for k, n in
                    dict(h=DIM, n=DIM, qkv=DIM + 2 * KVD, att=DIM, o=DIM, gu=2 * FFN, f=FFN,
                         d=DIM, lg=VOCAB).items()}

    def _make(self, rng, name, n, m, mean, s):
        x = ((mean + rng.standard_normal((n, m)) * s) * P.ONE).astype(np.int64)
        self.host_weights[name] = x
        return x

    def _weight(self, rng, name, n, m, mean, s):
        return self.ctx.to_device(self._make(rng, name, n, m, mean, s))

    def _stack(self, rng, parts, m):
        return self.ctx.to_device(np.concatenate(
            [self._make(rng, name, n, m, 0.0, 0.05) for name, n in parts]))

    def forward(self, tokens, p0, where=None, sees=None, decode=False):
        """Logits of rows stored at p0 .. (RoPE positions `where`, mask `sees`); decode:
        one row through the single-token entry point."""
        ctx, T = self.ctx, len(tokens)
        b = {k: v.ptr for k, v in self.buf.items()}
        mask = ctx.to_device(P.mask_words(sees)) if sees is not None else None
        pos = ints(ctx, where) if where is not None else None
        tok = ints(ctx, tokens)
        m, d = (x.ptr if x else None for x in (mask, pos))
        embed_rows(ctx, b["h"], self.embed.ptr, tok.ptr, T, DIM)
        for i, (an, wqkv, wo, fn, wgu, wd) in enumerate(self.layers):
            norm_rows(ctx, b["n"], b["h"], an.ptr, T, DIM)
            ctx.gemm(b["qkv"], wqkv.ptr, b["n"], T, DIM + 2 * KVD, DIM)
            if self.bits == 64:
                at = pos if pos else ints(ctx, np.arange(p0, p0 + T))
                ctx.rope_store_rows_at(b["qkv"], self.kc.ptr, self.vc.ptr, i, p0, T, at.ptr, NH,
                                       NKV, HD, MAX_SEQ)
                ctx.attn_tree(b["att"], b["qkv"], self.kc.ptr, self.vc.ptr, i, p0, T, NH, NKV, HD,
                              MAX_SEQ, m)
            elif decode:
                ctx.attn_decode_rope_qcache(b["att"], b["qkv"], self.cache, b["qkv"] + 8 * DIM,
                                            b["qkv"] + 8 * (DIM + KVD), i, p0, NH)
            else:
                ctx.rope_store_rows_qcache(b["qkv"], self.cache, i, p0, T, NH, d)
                ctx.attn_rows_qcache(b["att"], b["qkv"], self.cache, i, p0, T, NH, m)
            ctx.gemm(b["o"], wo.ptr, b["att"], T, DIM, DIM)
            ctx.add(b["h"], b["o"], T * DIM)
            norm_rows(ctx, b["n"], b["h"], fn.ptr, T, DIM)
            ctx.gemm(b["gu"], wgu.ptr, b["n"], T, 2 * FFN, DIM)
            silu_rows(ctx, b["f"], b["gu"], T, FFN)
            ctx.gemm(b["d"], wd.ptr, b["f"], T, DIM, FFN)
            ctx.add(b["h"], b["d"], T * DIM)
        norm_rows(ctx, b["n"], b["h"], self.norm.ptr, T, DIM)
        ctx.gemm(b["lg"], self.head.ptr, b["n"], T, VOCAB, DIM)
        return self.buf["lg"].download(T * VOCAB).reshape(T, VOCAB)

    def keep(self, p0, rows):
        d = ints(self.ctx, rows)
        if self.bits == 64:
            self.ctx.cache_keep_rows(self.kc.ptr, self.vc.ptr, L, p0, d.ptr, len(rows), NKV, HD,
                                     MAX_SEQ)
        else:
            self.ctx.qcache_keep_rows(self.cache, p0, d.ptr, len(rows))

    def score(self, tokens, top):
        """Log probabilities of the rows' tokens from the logits on the device."""
        T, ctx = len(tokens), self.ctx
        tk = ints(ctx, tokens)
        lp, en, tlp = ctx.buffer(T), ctx.buffer(T), ctx.buffer(T * top)
        ids = ctx.buffer((T * top + 1) // 2)
        ctx.logprobs_rows(self.buf["lg"].ptr, T, VOCAB, tk.ptr, lp.ptr, en.ptr, top, ids.ptr,
                          tlp.ptr)
        return (lp.download(), en.download(),
                ids.download().view(np.int32)[:T * top].reshape(T, top),
                tlp.download().reshape(T, top))


def draft(rng, greedy, T):
    """A tree of T drafted tokens whose path `greedy` (node 0 its first token) is the
    right one: tokens, parents, who sees whom, depths, the right path's nodes."""
    tokens, parent, path = [greedy[0]], [-1], [0]
    right = 1
    while len(tokens) < T:
        if right < len(greedy) and rng.random() < 0.5:
            tokens.append(greedy[right])
            parent.append(path[-1])
            path.append(len(tokens) - 1)
            right += 1
        else:
            tokens.append(int(rng.integers(3, VOCAB)))
            parent.append(int(rng.integers(0, len(parent))))
    sees = np.eye(T, dtype=bool)
    depth = np.zeros(T, dtype=np.int32)
    for t in range(1, T):
        sees[t] |= sees[parent[t]]
        depth[t] = depth[parent[t]] + 1
    return tokens, parent, sees, depth, path


@pytest.mark.parametrize("bits", [64, 8, 4])
@pytest.mark.parametrize("prompt,T", [(16, 12), (90, 40)])
def test_draft_and_verify(ctx, bits, prompt, T):
    rng = np.random.default_rng(prompt + bits)
    with intllm.Context(0) as c:
        c.rope_init(HD, MAX_SEQ, 10000)
        model = Tiny(c, bits, np.random.default_rng(7))
        words = rng.integers(3, VOCAB, prompt).tolist()
        logits = np.concatenate([model.forward(words[i:i + 64], i) for i in range(0, prompt, 64)])
        host = None
        if bits == 64:
            host = intllm.HostModel(c, intllm.Config(DIM, NH, NKV, HD, L, FFN, VOCAB, MAX_SEQ,
                                                     10000))
            for name, x in model.host_weights.items():
                host.upload(name, x)
            step = lambda tok, pos: host.forward(tok, pos, VOCAB, choose=False)[1]  # noqa: E731
            assert all((step(w, i) == logits[i]).all() for i, w in enumerate(words))
        else:
            other = Tiny(c, bits, np.random.default_rng(7))
            for i, w in enumerate(words):      # the prompt token by token: the same cache
                assert (other.forward([w], i, decode=True)[0] == logits[i]).all()
            step = lambda tok, pos: other.forward([tok], pos, decode=True)[0]  # noqa: E731
        # greedy decoding, call by call
        greedy, want = [int(np.argmax(logits[-1]))], []
        for i in range(6):
            want.append(step(greedy[-1], prompt + i))
            greedy.append(int(np.argmax(want[-1])))
        # the same tokens in one pass over a tree
        tokens, parent, sees, depth, path = draft(rng, greedy[:6], T)
        got = model.forward(tokens, prompt, prompt + depth, sees)
        for i, node in enumerate(path):
            assert (got[node] == want[i]).all()
        # what the verifier reads: each node's most probable token, its child's log probability
        child = np.full(T, -1)
        for t in range(T - 1, 0, -1):
            child[parent[t]] = tokens[t]
        lp, en, ids, tlp = model.score(child, 4)
        w = P.logprobs(got, child, 4)
        assert (lp == w[0]).all() and (en == w[1]).all()
        assert (ids == w[2]).all() and (tlp == w[3]).all()
        accepted = [0]
        while True:
            nxt = [t for t in range(T) if parent[t] == accepted[-1] and
                   tokens[t] == ids[accepted[-1], 0]]
            if not nxt:
                break
            accepted.append(nxt[0])
        assert [tokens[t] for t in accepted] == greedy[:len(accepted)]
        assert len(accepted) >= len(path)
        # the accepted rows move together and decoding goes on
        model.keep(prompt, accepted)
        n = len(accepted)
        tok = int(ids[accepted[-1], 0])
        for i in range(3):
            pos = prompt + n + i
            a = model.forward([tok], pos, decode=bits != 64)[0]
            b = step(tok, pos) if n + i >= 6 else (want[n + i] if n + i < 6 else None)
            assert (a == b).all()
            tok = int(np.argmax(a))
        if host:
            host.free()
