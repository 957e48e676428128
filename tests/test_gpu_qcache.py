"""The quantised key/value cache on the GPU: what is written and read back, and
attention over it, word for word against the plain forms.
"""
import ctypes as C

import numpy as np
import pytest

import intllm
import serve_plain as P

pytestmark = pytest.mark.gpu
I64 = np.iinfo(np.int64)


def acts(rng, *shape, sigma=1.0):
    return (rng.standard_normal(shape) * (sigma * P.ONE)).astype(np.int64)


class Cache:
    """A quantised cache on the device, its codes and steps for the tests to see."""

    def __init__(self, ctx, bits, layers, max_seq, nkv, hd):
        self.ctx, self.bits, self.shape = ctx, bits, (layers, max_seq, nkv)
        codes, steps = intllm.qcache_bytes(bits, layers, max_seq, nkv, hd)
        self.row = hd * bits // 8
        self.bufs = [intllm.Buffer(ctx, n // 8) for n in (codes, codes, steps, steps)]
        rng = np.random.default_rng(9)     # what a cache held before: any bytes
        for b in self.bufs:
            b.upload(rng.integers(I64.min, I64.max, b.n))
        self.c = ctx.qcache(*(b.ptr for b in self.bufs), bits, layers, max_seq, nkv, hd)

    def read(self):
        """k, v bytes [layers][max_seq][nkv][row] and steps [layers][max_seq][nkv]"""
        k, v, ks, vs = (b.download() for b in self.bufs)
        s = self.shape
        return (k.view(np.uint8).reshape(*s, self.row), v.view(np.uint8).reshape(*s, self.row),
                ks.reshape(s), vs.reshape(s))

    def fill(self, layer, K, V):
        """Rows [0, n) of a layer from values, quantised by the plain form; their values."""
        k, v, ks, vs = self.read()
        out = []
        for x, codes, steps in ((K, k, ks), (V, v, vs)):
            c, st = P.quantise(x, self.bits)
            codes[layer, :len(x)], steps[layer, :len(x)] = P.pack(c, self.bits), st
            out.append(P.values(c, st))
        for b, x in zip(self.bufs, (k, v, ks, vs)):
            b.upload(np.ascontiguousarray(x).view(np.int64).ravel())
        return out

    def free(self):
        for b in self.bufs:
            b.free()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("nkv,hd,T,p0,pad", [(1, 32, 1, 0, 0), (4, 64, 1, 17, 0), (3, 64, 37, 5, 0),
                                             (2, 128, 70, 0, 24), (8, 32, 129, 2, 1),
                                             (7, 128, 5, 100, 640)])
def test_store_and_load(ctx, bits, nkv, hd, T, p0, pad):
    rng = np.random.default_rng(bits * 1000 + T)
    max_seq, ld = p0 + T + 3, nkv * hd + pad
    K, V = acts(rng, T, ld), acts(rng, T, ld, sigma=0.02)
    K[0, 0], V[T // 2, 1] = I64.min, I64.max
    if T > 4:
        K[3], V[2] = 0, 0
        K[4] = rng.integers(-20, 20, ld)
    cache = Cache(ctx, bits, 2, max_seq, nkv, hd)
    before = cache.read()
    dk, dv = ctx.to_device(K), ctx.to_device(V)
    ctx.qcache_store_rows(cache.c, 1, p0, T, dk.ptr, dv.ptr, ld)
    after = cache.read()
    back = [ctx.to_device(np.full(T * ld, 77, np.int64)) for _ in range(2)]
    ctx.qcache_load_rows(back[0].ptr, back[1].ptr, cache.c, 1, p0, T, ld)
    for i, x in enumerate((K, V)):
        c, st = P.quantise(x[:, :nkv * hd].reshape(T, nkv, hd), bits)
        for got, old, want in ((after[i], before[i], P.pack(c, bits)),
                               (after[i + 2], before[i + 2], st)):
            exp = old.copy()
            exp[1, p0:p0 + T] = want           # and no other row
            assert (got == exp).all()
        got = back[i].download().reshape(T, ld)
        assert (got[:, :nkv * hd].reshape(T, nkv, hd) == P.values(c, st)).all()
        assert (got[:, nkv * hd:] == 77).all()
    cache.free()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 32), (4, 4, 64), (6, 2, 128)])
def test_rope_store(ctx, bits, nh, nkv, hd):
    rng = np.random.default_rng(11)
    T, p0, max_seq = 9, 4, 32
    ctx.rope_init(hd, max_seq, 10000)
    cos_t, sin_t = P.rope_tables(hd, max_seq)
    x = acts(rng, T, nh + 2 * nkv, hd)
    where = np.array([4, 5, 5, 6, -1, 31, 32, 0, 7], dtype=np.int32)
    d_where = ctx.to_device(np.concatenate([where, [0]]).astype(np.int32).view(np.int64))
    for at, ptr in ((range(p0, p0 + T), None), (where, d_where.ptr)):
        cache = Cache(ctx, bits, 1, max_seq, nkv, hd)
        before = cache.read()
        d = ctx.to_device(x)
        ctx.rope_store_rows_qcache(d.ptr, cache.c, 0, p0, T, nh, ptr)
        got, after = d.download().reshape(x.shape), cache.read()
        for t, pos in enumerate(at):
            if not 0 <= pos < max_seq:
                assert (got[t] == x[t]).all()
                assert all((a[0, p0 + t] == b[0, p0 + t]).all() for a, b in zip(after, before))
                continue
            r = P.rope(x[t, :nh + nkv], cos_t, sin_t, int(pos))
            assert (got[t, :nh + nkv] == r).all() and (got[t, nh + nkv:] == x[t, nh + nkv:]).all()
            for i, y in enumerate((r[nh:], x[t, nh + nkv:])):
                c, st = P.quantise(y, bits)
                assert (after[i][0, p0 + t] == P.pack(c, bits)).all()
                assert (after[i + 2][0, p0 + t] == st).all()
        cache.free()


SHAPES = [(1, 1, 64), (8, 2, 32), (32, 4, 64), (7, 1, 128), (8, 8, 64), (28, 4, 32), (6, 3, 128),
          (16, 1, 64), (40, 2, 64)]


def decode_case(ctx, bits, nh, nkv, hd, pos, max_seq, rng, rope=False, layer=0, layers=1,
                sigma=1.0, edit=None):
    """One decoded token against the plain form: its output and its row of the cache."""
    cache = Cache(ctx, bits, layers, max_seq, nkv, hd)
    K, V = acts(rng, pos + 1, nkv, hd, sigma=sigma), acts(rng, pos + 1, nkv, hd, sigma=sigma)
    q = acts(rng, nh, hd, sigma=1.5)
    if edit:
        edit(q, K, V)
    kv, vv = cache.fill(layer, K, V)
    kn, vn = acts(rng, nkv, hd), acts(rng, nkv, hd)
    qr, kr = q, kn
    if rope:
        ctx.rope_init(hd, max_seq, 10000)
        cos_t, sin_t = P.rope_tables(hd, max_seq)
        qr, kr = P.rope(q, cos_t, sin_t, pos), P.rope(kn, cos_t, sin_t, pos)
    want_row = [P.quantise(kr, bits), P.quantise(vn, bits)]
    kv[pos], vv[pos] = (P.values(*w) for w in want_row)
    want = P.attend(qr[None], kv, vv, np.ones((1, pos + 1), bool))[0]
    before = cache.read()
    bufs = [ctx.to_device(a) for a in (q, kn, vn)]
    out = ctx.to_device(np.full(nh * hd, 5, np.int64))
    f = ctx.attn_decode_rope_qcache if rope else ctx.attn_decode_qcache
    f(out.ptr, bufs[0].ptr, cache.c, bufs[1].ptr, bufs[2].ptr, layer, pos, nh)
    got, after = out.download().reshape(nh, hd), cache.read()
    assert (got == want).all(), np.argwhere(got != want)[:5]
    for i, (c, st) in enumerate(want_row):
        for b, a, w in ((before[i], after[i], P.pack(c, bits)), (before[i + 2], after[i + 2], st)):
            b[layer, pos] = w
            assert (a == b).all()
    assert all((b.download() == a.ravel()).all() for b, a in zip(bufs, (q, kn, vn)))
    cache.free()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("nh,nkv,hd", SHAPES)
@pytest.mark.parametrize("pos", [0, 1, 15, 16, 63, 64, 130, 517])
def test_decode(ctx, bits, nh, nkv, hd, pos):
    decode_case(ctx, bits, nh, nkv, hd, pos, pos + 1 + pos % 3,
                np.random.default_rng(pos * 10 + bits))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("nh,nkv,hd,pos", [(32, 4, 64, 2500), (8, 8, 128, 4100), (8, 1, 32, 9000),
                                           (4, 2, 64, 20011), (2, 1, 64, 32766)])
def test_decode_long(ctx, bits, nh, nkv, hd, pos):
    decode_case(ctx, bits, nh, nkv, hd, pos, min(32767, pos + 40), np.random.default_rng(pos))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("pos", [3, 200, 5000])
def test_decode_rope_in_a_later_layer(ctx, bits, pos):
    decode_case(ctx, bits, 8, 2, 64, pos, pos + 5, np.random.default_rng(7), rope=True, layer=2,
                layers=3)


def big_values(q, K, V):
    V[len(V) // 2] *= 300            # |v| past 2^51


def huge_scores(q, K, V):
    q[0] = I64.max                   # dot products that wrap
    K[::3] = I64.min


def tiny(q, K, V):
    q[:] >>= 45
    K[:] >>= 44
    V[:] >>= 46


def one_peak(q, K, V):
    K[len(K) // 3] = np.sign(q[0]) * (8 * P.ONE)


def zeros(q, K, V):
    K[:], V[:] = 0, 0


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("edit", [big_values, huge_scores, tiny, one_peak, zeros])
@pytest.mark.parametrize("pos", [40, 700, 4500])
def test_decode_of_unusual_values(ctx, bits, edit, pos):
    decode_case(ctx, bits, 8, 2, 64, pos, pos + 1, np.random.default_rng(pos), edit=edit)


def rows_case(ctx, bits, nh, nkv, hd, T, p0, max_seq, sees, rng, edit=None, junk=False):
    K, V = acts(rng, p0 + T, nkv, hd), acts(rng, p0 + T, nkv, hd)
    qkv = acts(rng, T, nh + 2 * nkv, hd, sigma=1.5)
    if edit:
        edit(qkv[0], K, V)
    mask = None
    see = np.concatenate([np.ones((T, p0), bool), np.tri(T, dtype=bool) if sees is None else sees],
                         1)
    if sees is not None:
        w = P.mask_words(sees)
        if junk and T % 64:                  # bits from T on say nothing
            w[:, -1] |= np.int64(-1) << np.int64(T % 64)
        mask = ctx.to_device(w).ptr
    out = ctx.to_device(np.full(T * nh * hd, 5, np.int64))
    d = ctx.to_device(qkv)
    if bits == 64:
        kc, vc = np.zeros((2, max_seq, nkv, hd), np.int64), np.zeros((2, max_seq, nkv, hd), np.int64)
        kc[:], vc[:] = I64.max // 3, I64.min // 3   # rows past the last, and the other layer
        kc[1, :p0 + T], vc[1, :p0 + T] = K, V
        dk, dv = ctx.to_device(kc), ctx.to_device(vc)
        ctx.attn_tree(out.ptr, d.ptr, dk.ptr, dv.ptr, 1, p0, T, nh, nkv, hd, max_seq, mask)
        want = P.attend(qkv[:, :nh], K, V, see)
    else:
        cache = Cache(ctx, bits, 2, max_seq, nkv, hd)
        kv, vv = cache.fill(1, K, V)
        ctx.attn_rows_qcache(out.ptr, d.ptr, cache.c, 1, p0, T, nh, mask)
        want = P.attend(qkv[:, :nh], kv, vv, see)
    got = out.download().reshape(T, nh, hd)
    assert (got == want).all(), np.argwhere(got != want)[:5]
    assert (d.download() == qkv.ravel()).all()
    if bits != 64:
        cache.free()


@pytest.mark.parametrize("bits", [8, 4, 64])
@pytest.mark.parametrize("nh,nkv,hd", SHAPES)
@pytest.mark.parametrize("T,p0", [(1, 0), (3, 0), (17, 30), (5, 700)])
def test_rows_causal(ctx, bits, nh, nkv, hd, T, p0):
    rows_case(ctx, bits, nh, nkv, hd, T, p0, p0 + T + 2, None, np.random.default_rng(T + p0))


@pytest.mark.parametrize("bits", [8, 4, 64])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 32), (32, 4, 64), (7, 1, 128), (4, 4, 64)])
@pytest.mark.parametrize("T,p0,pad", [(2, 0, 1), (16, 0, 3), (33, 100, 2), (65, 7, 1), (130, 0, 5)])
def test_rows_tree(ctx, bits, nh, nkv, hd, T, p0, pad):
    rng = np.random.default_rng(T)
    sees, _ = P.tree(rng, T, pad)
    rows_case(ctx, bits, nh, nkv, hd, T, p0, p0 + T, sees, rng, junk=True)


@pytest.mark.parametrize("bits", [8, 4, 64])
def test_rows_under_any_mask(ctx, bits):
    """Masks that no tree has: later rows seen, nothing seen at all, one row seen."""
    rng = np.random.default_rng(5)
    sees = rng.random((70, 70)) < 0.3
    sees[11] = False
    sees[12] = False
    sees[12, 69] = True
    sees[69] = True
    rows_case(ctx, bits, 8, 2, 64, 70, 0, 70, sees, rng)
    rows_case(ctx, bits, 8, 2, 64, 70, 33, 111, sees, rng)
    rows_case(ctx, bits, 8, 2, 64, 70, 0, 70, np.zeros((70, 70), bool), rng)


@pytest.mark.parametrize("bits", [8, 4, 64])
@pytest.mark.parametrize("T,p0", [(40, 1500), (300, 0), (9, 5000), (2, 20000)])
def test_rows_long(ctx, bits, T, p0):
    rows_case(ctx, bits, 8, 2, 64, T, p0, p0 + T + 1, None, np.random.default_rng(T))


@pytest.mark.parametrize("bits", [8, 4, 64])
@pytest.mark.parametrize("edit", [big_values, huge_scores, tiny, one_peak, zeros])
@pytest.mark.parametrize("T,p0", [(20, 0), (5, 300), (6, 3000)])
def test_rows_of_unusual_values(ctx, bits, edit, T, p0):
    rng = np.random.default_rng(T)
    sees, _ = P.tree(rng, T, 1)
    rows_case(ctx, bits, 8, 2, 64, T, p0, p0 + T, sees, rng, edit=edit)


def test_step_mode_and_graph(ctx):
    """Decode replayed from a graph, the position on the device: every replay
    against the eager form, across the positions where kernels change."""
    rng = np.random.default_rng(21)
    nh, nkv, hd, max_seq, n = 8, 2, 64, 3000, 5
    for start in (2, 2040, 2990):
        with intllm.Context(0) as c:
            c.rope_init(hd, max_seq, 10000)
            cache = Cache(c, 8, 1, max_seq, nkv, hd)
            cache.fill(0, acts(rng, start, nkv, hd), acts(rng, start, nkv, hd))
            other = Cache(c, 8, 1, max_seq, nkv, hd)
            for a, b in zip(other.bufs, cache.bufs):
                a.upload(b.download())
            q, kn, vn = (c.to_device(acts(rng, m, hd)) for m in (nh, nkv, nkv))
            out, want = c.buffer(nh * hd), c.buffer(nh * hd)
            logits = c.to_device(np.arange(8))
            toks = c.buffer(8)

            def step():
                c.attn_decode_rope_qcache(out.ptr, q.ptr, cache.c, kn.ptr, vn.ptr, 0, start, nh)
                intllm.check("q48_argmax_step", intllm.hip_lib().q48_argmax_step(
                    c.h, logits.ptr, 8, toks.ptr, 16))

            lib = intllm.hip_lib()
            intllm.check("step", lib.q48_step_set(c.h, 0, start))
            intllm.check("step", lib.q48_step_mode(c.h, 1))
            step()                                   # workspaces reach their size
            c.sync()
            intllm.check("step", lib.q48_step_set(c.h, 0, start))
            intllm.check("begin", lib.q48_graph_begin(c.h))
            step()
            intllm.check("end", lib.q48_graph_end(c.h))
            for i in range(n):
                intllm.check("launch", lib.q48_graph_launch(c.h, 1))
                got = out.download()
                intllm.check("step", lib.q48_step_mode(c.h, 0))
                c.attn_decode_rope_qcache(want.ptr, q.ptr, other.c, kn.ptr, vn.ptr, 0, start + i,
                                          nh)
                assert (want.download() == got).all(), (start, i)
                intllm.check("step", lib.q48_step_mode(c.h, 1))
            assert all((a.download() == b.download()).all()
                       for a, b in zip(cache.bufs, other.bufs))
            intllm.check("drop", lib.q48_graph_drop(c.h))
            cache.free()
            other.free()


def test_step_position_outside_the_cache_changes_nothing(ctx):
    lib = intllm.hip_lib()
    rng = np.random.default_rng(4)
    with intllm.Context(0) as c:
        cache = Cache(c, 4, 1, 50, 2, 64)
        before = cache.read()
        q, kn, vn = (c.to_device(acts(rng, m, 64)) for m in (4, 2, 2))
        out = c.to_device(np.full(256, 5, np.int64))
        intllm.check("mode", lib.q48_step_mode(c.h, 1))
        for pos in (50, 4000):       # (q48_step_set itself refuses a negative one)
            intllm.check("set", lib.q48_step_set(c.h, 0, pos))
            c.attn_decode_qcache(out.ptr, q.ptr, cache.c, kn.ptr, vn.ptr, 0, 3, 4)
        assert all((a == b).all() for a, b in zip(before, cache.read()))
        cache.free()


def test_two_contexts_at_once(ctx):
    """Two programs' calls in flight together, each on its own stream and workspace."""
    rng = np.random.default_rng(8)
    K, V = acts(rng, 2100, 2, 64), acts(rng, 2100, 2, 64)
    with intllm.Context(0) as a, intllm.Context(0) as b:
        state = []
        for c in (a, b):
            cache = Cache(c, 8, 1, 2100, 2, 64)
            cache.fill(0, K, V)
            q = acts(rng, 6, 12, 64)
            state.append((c, cache, q, c.to_device(q), c.buffer(6 * 8 * 64)))
        for _ in range(5):
            for c, cache, _, d, out in state:
                c.attn_rows_qcache(out.ptr, d.ptr, cache.c, 0, 2090, 6, 8)
        kv, vv = (P.values(*P.quantise(x, 8)) for x in (K, V))
        see = np.concatenate([np.ones((6, 2090), bool), np.tri(6, dtype=bool)], 1)
        for c, cache, q, _, out in state:
            want = P.attend(q[:, :8], kv[:2096], vv[:2096], see)
            assert (out.download().reshape(6, 8, 64) == want).all()
            cache.free()


def test_cache_past_four_gigabytes(ctx):
    """The last layer of a cache whose offsets pass 32 bits."""
    rng = np.random.default_rng(3)
    layers, max_seq, nkv, hd, nh = 131, 32767, 8, 128, 16
    codes, steps = intllm.qcache_bytes(8, layers, max_seq, nkv, hd)
    assert codes > 1 << 32
    bufs = [intllm.Buffer(ctx, n // 8) for n in (codes, codes, steps, steps)]
    cache = ctx.qcache(*(b.ptr for b in bufs), 8, layers, max_seq, nkv, hd)
    T, p0 = 40, 0
    K, V, qkv = acts(rng, T, nkv, hd), acts(rng, T, nkv, hd), acts(rng, T, nh + 2 * nkv, hd)
    dk, dv, dq = (ctx.to_device(x) for x in (K, V, qkv))
    out = ctx.buffer(T * nh * hd)
    ctx.qcache_store_rows(cache, layers - 1, p0, T, dk.ptr, dv.ptr, nkv * hd)
    ctx.attn_rows_qcache(out.ptr, dq.ptr, cache, layers - 1, p0, T, nh)
    kv, vv = (P.values(*P.quantise(x, 8)) for x in (K, V))
    want = P.attend(qkv[:, :nh], kv, vv, np.tri(T, dtype=bool))
    assert (out.download().reshape(T, nh, hd) == want).all()
    for b in bufs:
        b.free()


def test_int64_rows_equal_the_decode_and_prefill_entry_points(ctx):
    """attn_tree's causal form against q48_attn_prefill, and a tree's paths against
    q48_attn_decode of their own tokens."""
    rng = np.random.default_rng(6)
    nh, nkv, hd, T, p0, max_seq = 8, 2, 64, 12, 40, 64
    ctx.rope_init(hd, max_seq, 10000)
    K, V = acts(rng, max_seq, nkv, hd), acts(rng, max_seq, nkv, hd)
    qkv = acts(rng, T, nh + 2 * nkv, hd)
    dk, dv, dq = (ctx.to_device(x) for x in (K, V, qkv))
    a, b = ctx.buffer(T * nh * hd), ctx.buffer(T * nh * hd)
    ctx.attn_tree(a.ptr, dq.ptr, dk.ptr, dv.ptr, 0, p0, T, nh, nkv, hd, max_seq)
    ctx.attn_prefill(b.ptr, dq.ptr, dk.ptr, dv.ptr, 0, p0, T, nh, nkv, hd, max_seq)
    assert (a.download() == b.download()).all()
    sees, _ = P.tree(rng, T)
    m = ctx.to_device(P.mask_words(sees))
    ctx.attn_tree(a.ptr, dq.ptr, dk.ptr, dv.ptr, 0, p0, T, nh, nkv, hd, max_seq, m.ptr)
    got = a.download().reshape(T, nh, hd)
    for t in range(T):
        path = [*range(p0), *(p0 + np.nonzero(sees[t])[0])]
        k2, v2 = ctx.to_device(K[path]), ctx.to_device(V[path])
        kn, vn = ctx.to_device(K[path[-1]]), ctx.to_device(V[path[-1]])
        q, o = ctx.to_device(qkv[t, :nh]), ctx.buffer(nh * hd)
        ctx.attn_decode(o.ptr, q.ptr, k2.ptr, v2.ptr, kn.ptr, vn.ptr, 0, len(path) - 1, nh, nkv,
                        hd, len(path))
        assert (o.download().reshape(nh, hd) == got[t]).all()


def test_rope_store_rows_at(ctx):
    rng = np.random.default_rng(13)
    nh, nkv, hd, T, p0, max_seq, layers = 4, 2, 64, 6, 3, 16, 2
    ctx.rope_init(hd, max_seq, 10000)
    cos_t, sin_t = P.rope_tables(hd, max_seq)
    x = acts(rng, T, nh + 2 * nkv, hd)
    where = np.array([3, 4, 4, 16, -5, 15], dtype=np.int32)
    old = acts(rng, layers, max_seq, nkv, hd)
    dk, dv, d = ctx.to_device(old), ctx.to_device(old + 1), ctx.to_device(x)
    dw = ctx.to_device(where.view(np.int64))
    ctx.rope_store_rows_at(d.ptr, dk.ptr, dv.ptr, 1, p0, T, dw.ptr, nh, nkv, hd, max_seq)
    k, v, got = old.copy(), old + 1, x.copy()
    for t, pos in enumerate(where):
        if 0 <= pos < max_seq:
            got[t, :nh + nkv] = P.rope(x[t, :nh + nkv], cos_t, sin_t, int(pos))
            k[1, p0 + t], v[1, p0 + t] = got[t, nh:nh + nkv], x[t, nh + nkv:]
    assert (d.download() == got.ravel()).all()
    assert (dk.download() == k.ravel()).all() and (dv.download() == v.ravel()).all()


@pytest.mark.parametrize("rows", [[0], [2], [0, 1, 2], [1, 2, 3, 7], [0, 3, 4], [5, 6], [0, 99, -4]])
def test_keep_rows(ctx, rows):
    rng = np.random.default_rng(2)
    layers, max_seq, nkv, hd, p0 = 3, 12, 3, 64, 4
    d = ctx.to_device(np.array(rows + [0] * (len(rows) % 2), dtype=np.int32).view(np.int64))

    def keep(x):   # [layers][max_seq][...]
        y = x.copy()
        for i, r in enumerate(rows):
            if r > i and p0 + r < max_seq:
                y[:, p0 + i] = x[:, p0 + r]
        return y

    k, v = acts(rng, layers, max_seq, nkv, hd), acts(rng, layers, max_seq, nkv, hd)
    dk, dv = ctx.to_device(k), ctx.to_device(v)
    ctx.cache_keep_rows(dk.ptr, dv.ptr, layers, p0, d.ptr, len(rows), nkv, hd, max_seq)
    assert (dk.download() == keep(k).ravel()).all() and (dv.download() == keep(v).ravel()).all()
    for bits in (8, 4):
        cache = Cache(ctx, bits, layers, max_seq, nkv, hd)
        before = cache.read()
        ctx.qcache_keep_rows(cache.c, p0, d.ptr, len(rows))
        assert all((a == keep(b)).all() for a, b in zip(cache.read(), before))
        cache.free()


@pytest.mark.parametrize("bits", [8, 4, 64])
@pytest.mark.parametrize("p0", [0, 50, 2500])
def test_rows_never_stored_may_hold_anything(ctx, bits, p0):
    """A padded batch: the last rows are masked everywhere and their cache rows hold
    what memory held."""
    rng = np.random.default_rng(p0 + bits)
    nh, nkv, hd, T, pad = 8, 2, 64, 20, 3
    max_seq = p0 + T
    sees, _ = P.tree(rng, T, pad)
    sees[:, T - pad:] = False
    K, V = acts(rng, max_seq, nkv, hd), acts(rng, max_seq, nkv, hd)
    K[max_seq - pad:] = I64.min
    V[max_seq - pad:] = rng.integers(I64.min, I64.max, (pad, nkv, hd))
    qkv = acts(rng, T, nh + 2 * nkv, hd)
    mask = ctx.to_device(P.mask_words(sees))
    d, out = ctx.to_device(qkv), ctx.buffer(T * nh * hd)
    see = np.concatenate([np.ones((T, p0), bool), sees], 1)
    if bits == 64:
        dk, dv = ctx.to_device(K), ctx.to_device(V)
        ctx.attn_tree(out.ptr, d.ptr, dk.ptr, dv.ptr, 0, p0, T, nh, nkv, hd, max_seq, mask.ptr)
    else:
        cache = Cache(ctx, bits, 1, max_seq, nkv, hd)      # any bytes, steps too
        kv, vv = cache.fill(0, K[:-pad], V[:-pad])
        K[:-pad], V[:-pad] = kv, vv
        ctx.attn_rows_qcache(out.ptr, d.ptr, cache.c, 0, p0, T, nh, mask.ptr)
        cache.free()
    want = P.attend(qkv[:, :nh], K, V, see)
    assert (out.download().reshape(T, nh, hd) == want).all()


def test_more_rows_than_one_workspace(ctx):
    """Rows in several launches (a GiB of scores each): against q48_attn_prefill, and
    the quantised cache against the int64 cache of the values it stands for."""
    rng = np.random.default_rng(17)
    nh, nkv, hd, T, p0, max_seq = 64, 8, 32, 150, 16000, 16160
    ctx.rope_init(hd, max_seq, 10000)
    K, V = acts(rng, max_seq, nkv, hd), acts(rng, max_seq, nkv, hd)
    qkv = acts(rng, T, nh + 2 * nkv, hd)
    bufs = [ctx.to_device(x) for x in (K, V, qkv)]
    dk, dv, dq = bufs
    a, b = intllm.Buffer(ctx, T * nh * hd), intllm.Buffer(ctx, T * nh * hd)
    ctx.attn_tree(a.ptr, dq.ptr, dk.ptr, dv.ptr, 0, p0, T, nh, nkv, hd, max_seq)
    ctx.attn_prefill(b.ptr, dq.ptr, dk.ptr, dv.ptr, 0, p0, T, nh, nkv, hd, max_seq)
    assert (a.download() == b.download()).all()
    for bits in (8, 4):
        cache = Cache(ctx, bits, 1, max_seq, nkv, hd)
        ctx.qcache_store_rows(cache.c, 0, 0, max_seq, dk.ptr, dv.ptr, nkv * hd)
        back = [intllm.Buffer(ctx, K.size) for _ in range(2)]
        ctx.qcache_load_rows(back[0].ptr, back[1].ptr, cache.c, 0, 0, max_seq, nkv * hd)
        ctx.attn_rows_qcache(a.ptr, dq.ptr, cache.c, 0, p0, T, nh)
        ctx.attn_tree(b.ptr, dq.ptr, back[0].ptr, back[1].ptr, 0, p0, T, nh, nkv, hd, max_seq)
        assert (a.download() == b.download()).all()
        for x in back:
            x.free()
        cache.free()
    for x in (*bufs, a, b):
        x.free()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("p0", [20, 2500])
@pytest.mark.parametrize("top", [2 ** 51, 2 ** 52])
def test_codes_below_the_quantiser_s_lowest(ctx, bits, p0, top):
    """A cache may hold -128 (-8) too, which quantising never writes; around the largest
    steps whose values are summed in FP64."""
    rng = np.random.default_rng(p0 + bits)
    nh, nkv, hd, T = 8, 2, 64, 3
    cache = Cache(ctx, bits, 1, p0 + T, nkv, hd)
    low, Q = -(1 << (bits - 1)), P.LEVELS[bits]
    codes = rng.integers(low, low + 2, (2, p0 + T, nkv, hd))
    steps = np.stack([rng.integers(1, P.ONE >> 10, (p0 + T, nkv)),
                      top // Q - rng.integers(-1, 2, (p0 + T, nkv))])
    codes[0, p0 // 2] = -1                    # the only near key: nearly all the weight
    k, v, ks, vs = cache.read()
    k[0], v[0] = (P.pack(c, bits) for c in codes)
    ks[0], vs[0] = steps
    for b, x in zip(cache.bufs, (k, v, ks, vs)):
        b.upload(np.ascontiguousarray(x).view(np.int64).ravel())
    qkv = np.abs(acts(rng, T, nh + 2 * nkv, hd, sigma=4.0))
    d, out = ctx.to_device(qkv), ctx.buffer(T * nh * hd)
    ctx.attn_rows_qcache(out.ptr, d.ptr, cache.c, 0, p0, T, nh)
    kv, vv = (P.values(c, s) for c, s in zip(codes, steps))
    see = np.concatenate([np.ones((T, p0), bool), np.tri(T, dtype=bool)], 1)
    assert (out.download().reshape(T, nh, hd) == P.attend(qkv[:, :nh], kv, vv, see)).all()
    cache.free()


@pytest.mark.parametrize("bits", [8, 4, 64])
@pytest.mark.parametrize("p0", [40, 2500])
def test_verifying_captured(ctx, bits, p0):
    """Store, attend, keep as one graph, the rows, positions, mask and path changed
    between replays: against the same calls made eagerly on a twin."""
    rng = np.random.default_rng(p0 + bits)
    lib = intllm.hip_lib()
    nh, nkv, hd, T, n, max_seq = 8, 2, 64, 13, 4, p0 + 20
    with intllm.Context(0) as c:
        c.rope_init(hd, max_seq, 10000)
        words = T * (nh + 2 * nkv) * hd
        src, pos, mask, path = (c.buffer(m) for m in (words, 8, T, 2))
        K, V = acts(rng, max_seq, nkv, hd), acts(rng, max_seq, nkv, hd)
        sides = []
        for _ in range(2):
            qkv, out = c.buffer(words), c.buffer(T * nh * hd)
            if bits == 64:
                sides.append((qkv, out, [c.to_device(K), c.to_device(V)], None))
            else:
                q = Cache(c, bits, 1, max_seq, nkv, hd)
                q.fill(0, K, V)
                sides.append((qkv, out, q.bufs, q.c))

        def verify(qkv, out, bufs, cache):
            if bits == 64:
                k, v = (b.ptr for b in bufs)
                c.rope_store_rows_at(qkv.ptr, k, v, 0, p0, T, pos.ptr, nh, nkv, hd, max_seq)
                c.attn_tree(out.ptr, qkv.ptr, k, v, 0, p0, T, nh, nkv, hd, max_seq, mask.ptr)
                c.cache_keep_rows(k, v, 1, p0, path.ptr, n, nkv, hd, max_seq)
            else:
                c.rope_store_rows_qcache(qkv.ptr, cache, 0, p0, T, nh, pos.ptr)
                c.attn_rows_qcache(out.ptr, qkv.ptr, cache, 0, p0, T, nh, mask.ptr)
                c.qcache_keep_rows(cache, p0, path.ptr, n)

        def fresh():
            sees, parent = P.tree(rng, T, 0)
            x = acts(rng, words)
            for side in sides:
                side[0].upload(x)
            pos.upload(np.concatenate([p0 + sees.sum(1) - 1, np.zeros(16 - T)])
                       .astype(np.int32).view(np.int64))
            mask.upload(P.mask_words(sees).ravel())
            path.upload(np.sort(rng.choice(T, n, False)).astype(np.int32).view(np.int64))

        fresh()
        for side in sides:
            verify(*side)
        c.sync()
        intllm.check("begin", lib.q48_graph_begin(c.h))
        verify(*sides[0])
        intllm.check("end", lib.q48_graph_end(c.h))
        for _ in range(4):
            fresh()
            intllm.check("launch", lib.q48_graph_launch(c.h, 1))
            verify(*sides[1])
            for a, b in zip((*sides[0][:2], *sides[0][2]), (*sides[1][:2], *sides[1][2])):
                assert (a.download() == b.download()).all()
        intllm.check("drop", lib.q48_graph_drop(c.h))


@pytest.mark.parametrize("rows,near", [(64, 64), (64, 3), (4000, 64), (4000, 1000), (32767, 32767)])
def test_weights_of_chosen_scores(ctx, rows, near):
    """Scores given directly (q = 8 in one dim of a 64-wide head) and the softmax weights of
    64 rows read back (a value of ONE in a dim of its own): arguments at the clamp, at the
    truncation to 2^14ths and down to nothing, sums from one to 32767 times ONE."""
    hd, lim = 64, 10 << 48
    rng = np.random.default_rng(rows + near)
    edges = [0, 1, 2, (1 << 14) - 1, 1 << 14, (1 << 14) + 1, lim - (1 << 14), lim - 1, lim, lim + 1,
             lim + (1 << 14), 1 << 52, 1 << 61] + [1 << k for k in range(3, 51)]
    for first in (edges, None):
        u = np.full(rows, 1 << 60, np.int64)
        u[:near] = 0 if rows == near and rows > 64 else rng.integers(0, lim, near)
        n = min(64, near)
        if first:
            u[:n] = (first + [0] * 64)[:n] if n == 64 else first[:n]
        at = rng.permutation(rows)                # the rows read back, anywhere
        u = u[np.argsort(at)]
        K, V = np.zeros((rows, 1, hd), np.int64), np.zeros((rows, 1, hd), np.int64)
        K[:, 0, 5] = -u
        V[at[:64], 0, np.arange(64)] = P.ONE
        qkv = np.zeros((1, 3, hd), np.int64)
        qkv[0, 0, 5] = 8 * P.ONE
        d, dk, dv = (ctx.to_device(x) for x in (qkv, K, V))
        out = ctx.buffer(hd)
        ctx.attn_tree(out.ptr, d.ptr, dk.ptr, dv.ptr, 0, rows - 1, 1, 1, 1, hd, rows)
        want = P.attend(qkv[:, :1], K, V, np.ones((1, rows), bool))
        assert (out.download().reshape(1, 1, hd) == want).all()
        for b in (d, dk, dv, out):
            b.free()


def test_workspace_is_not_made_during_a_capture(ctx):
    """A shape that was never called is refused between begin and end; what was captured
    replays."""
    rng = np.random.default_rng(3)
    lib = intllm.hip_lib()
    nh, nkv, hd, T, V = 8, 2, 64, 3, 500
    with intllm.Context(0) as c:
        p0 = 9000                                # past LDS: scores in the workspace
        cache = Cache(c, 8, 1, p0 + T, nkv, hd)
        cache.fill(0, acts(rng, p0 + T, nkv, hd), acts(rng, p0 + T, nkv, hd))
        x = acts(rng, T, V, sigma=2.0)
        d, qkv = c.to_device(x), c.to_device(acts(rng, T, nh + 2 * nkv, hd))
        big = c.to_device(acts(rng, 1, 40000))
        out, ent = c.to_device(np.full(T * nh * hd, 5, np.int64)), c.buffer(T)
        intllm.check("begin", lib.q48_graph_begin(c.h))
        c.logprobs_rows(d.ptr, T, V, None, None, ent.ptr)
        for call in (lambda: c.attn_rows_qcache(out.ptr, qkv.ptr, cache.c, 0, p0, T, nh),
                     lambda: c.logprobs_rows(big.ptr, 1, 40000, None, None, ent.ptr)):
            with pytest.raises(intllm.Q48Error) as e:
                call()
            assert e.value.code == intllm.Q48_ESTATE
        intllm.check("end", lib.q48_graph_end(c.h))
        for _ in range(3):
            c.zero(ent.ptr, ent.nbytes)
            intllm.check("launch", lib.q48_graph_launch(c.h, 1))
            assert (ent.download() == P.logprobs(x, np.zeros(T, np.int64), 0)[1]).all()
        assert (out.download() == 5).all()
        intllm.check("drop", lib.q48_graph_drop(c.h))
        cache.free()


def tiles_of_sixteen(cus, nh, nkv, T):
    """Whether T rows have a block of 16 query vectors for every compute unit (the rule
    of q48_attn_rows_qcache for its largest tiles), and how many blocks that makes."""
    blocks = -(-T * (nh // nkv) // 16) * nkv
    return blocks >= cus, blocks


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("how", ["a block a unit", "scores fill the unit"])
@pytest.mark.parametrize("kind", ["causal", "tree", "nothing", "big_values", "huge_scores"])
def test_rows_of_sixteen_waves(ctx, bits, how, kind):
    """Rows of 64-wide heads whose blocks are alone on a compute unit, which take 16 waves:
    as many blocks as units, or more where two blocks' scores do not fit one unit (the last
    tile of them short)."""
    torch = pytest.importorskip("torch")
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    nh, nkv, hd = 32, 4, 64
    T, p0 = cus // nkv * 16 // (nh // nkv), 0
    if how == "scores fill the unit":
        T, p0 = T + 21, 700                    # 16 vectors of 849 scores: more than 80 KB
    full, blocks = tiles_of_sixteen(cus, nh, nkv, T)
    assert full and (blocks == cus if p0 == 0 else (p0 + T) * 16 * 8 > 80 << 10)
    rng = np.random.default_rng(T + bits)
    sees = None
    if kind in ("tree", "big_values"):
        sees, _ = P.tree(rng, T, 3)
    if kind == "nothing":
        sees = rng.random((T, T)) < 0.02
        sees[T // 2:] = False
    edit = dict(big_values=big_values, huge_scores=huge_scores).get(kind)
    rows_case(ctx, bits, nh, nkv, hd, T, p0, p0 + T, sees, rng, edit=edit, junk=sees is not None)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("max_seq,start,nh,nkv,hd", [(900, 2, 8, 2, 64), (3000, 2, 8, 2, 64),
                                                     (3000, 2990, 8, 2, 64), (20500, 2, 2, 1, 32)])
def test_one_graph_at_every_position(ctx, bits, max_seq, start, nh, nkv, hd):
    """One decode captured at a position and replayed at far and near ones, the position
    set on the device between replays: one launch, three chosen by the position it was
    captured at, and three because the cache's scores do not fit LDS."""
    rng = np.random.default_rng(max_seq + bits)
    lib = intllm.hip_lib()
    with intllm.Context(0) as c:
        c.rope_init(hd, max_seq, 10000)
        cache = Cache(c, bits, 1, max_seq, nkv, hd)
        cache.fill(0, acts(rng, max_seq, nkv, hd), acts(rng, max_seq, nkv, hd))
        q, kn, vn = (c.to_device(acts(rng, m, hd)) for m in (nh, nkv, nkv))
        out, want = c.buffer(nh * hd), c.buffer(nh * hd)

        def step(to, pos):
            c.attn_decode_rope_qcache(to.ptr, q.ptr, cache.c, kn.ptr, vn.ptr, 0, pos, nh)

        intllm.check("mode", lib.q48_step_mode(c.h, 1))
        intllm.check("set", lib.q48_step_set(c.h, 0, start))
        step(out, start)
        c.sync()
        intllm.check("begin", lib.q48_graph_begin(c.h))
        step(out, start)
        intllm.check("end", lib.q48_graph_end(c.h))
        for pos in (start, 700, max_seq - 1, 0, 31, max_seq - 2, 2040 % max_seq, start):
            intllm.check("set", lib.q48_step_set(c.h, 0, pos))
            intllm.check("launch", lib.q48_graph_launch(c.h, 1))
            got = out.download()
            intllm.check("mode", lib.q48_step_mode(c.h, 0))
            step(want, pos)
            assert (want.download() == got).all(), pos
            k, v, ks, vs = cache.read()
            kv, vv = (P.values(P.unpack(x[0, :pos + 1], bits), s[0, :pos + 1])
                      for x, s in ((k, ks), (v, vs)))
            cos_t, sin_t = P.rope_tables(hd, max_seq)
            qr = P.rope(q.download().reshape(nh, hd), cos_t, sin_t, pos)
            exp = P.attend(qr[None], kv, vv, np.ones((1, pos + 1), bool))
            assert (got.reshape(1, nh, hd) == exp).all(), pos
            intllm.check("mode", lib.q48_step_mode(c.h, 1))
        intllm.check("drop", lib.q48_graph_drop(c.h))
        cache.free()


@pytest.mark.parametrize("nkv,T,p0", [(240, 40, 32700), (1024, 1, 12000), (960, 20, 8100)])
def test_workspace_of_many_key_heads(ctx, nkv, T, p0):
    """One query head a KV head, so that a tile of 16 vectors is 16 rows: the scores stay
    within a GiB (and 2 / 64 of it for the maxima and sums of chunks of 64 rows), however
    the rows divide by 16.  Some heads against the plain form."""
    torch = pytest.importorskip("torch")
    hd, S, dev = 32, p0 + T, "cuda:0"
    g = torch.Generator(device=dev).manual_seed(nkv)
    codes = [torch.randint(-128, 128, (S, nkv, hd // 2), generator=g, device=dev, dtype=torch.int8)
             for _ in range(2)]
    steps = [torch.randint(1, 1 << 45, (S, nkv), generator=g, device=dev) for _ in range(2)]
    x = torch.randint(-P.ONE, P.ONE, (T, 3 * nkv, hd), generator=g, device=dev)
    out = torch.zeros(T, nkv, hd, dtype=torch.int64, device=dev)
    torch.cuda.synchronize()
    with intllm.Context(0) as c:
        cache = c.qcache(*(t.data_ptr() for t in (*codes, *steps)), 4, 1, S, nkv, hd)
        before = torch.cuda.mem_get_info()[0]
        c.attn_rows_qcache(out.data_ptr(), x.data_ptr(), cache, 0, p0, T, nkv)
        c.sync()
        used = before - torch.cuda.mem_get_info()[0]
        assert used <= (1 << 30) * 67 // 64, used
    see = np.concatenate([np.ones((T, p0), bool), np.tri(T, dtype=bool)], 1)
    for h in (0, nkv // 2 + 1, nkv - 1):
        kv, vv = (P.values(P.unpack(b[:, h].cpu().numpy().view(np.uint8), 4),
                           s[:, h].cpu().numpy())[:, None] for b, s in zip(codes, steps))
        want = P.attend(x[:, h:h + 1].cpu().numpy(), kv, vv, see)
        assert (out[:, h:h + 1].cpu().numpy() == want).all(), h


def test_a_cache_is_given_back(ctx):
    """A program that makes a cache for each conversation does not grow; a freed cache is
    refused."""
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(1)
    with intllm.Context(0) as c:
        x, out = c.to_device(acts(rng, 1, 12, 64)), c.buffer(4 * 64)

        def conversation():
            q = c.new_qcache(8, 22, 32767, 4, 64)          # 2 x 185 and 2 x 23 MB
            c.attn_rows_qcache(out.ptr, x.ptr, q, 21, 0, 1, 4)
            return q

        c.free_qcache(conversation())
        held, bufs = torch.cuda.mem_get_info()[0], len(c._bufs)
        for _ in range(6):
            q = conversation()
            assert held - torch.cuda.mem_get_info()[0] < 512 << 20
            c.free_qcache(q)
        assert len(c._bufs) == bufs and torch.cuda.mem_get_info()[0] >= held
        with pytest.raises(intllm.Q48Error) as e:
            c.attn_rows_qcache(out.ptr, x.ptr, q, 21, 0, 1, 4)
        assert e.value.code == intllm.Q48_EINVAL
        c.free_qcache(q)                                    # nothing left to give back
        mine = c.to_device(np.arange(4))
        c.free_qcache(c.qcache(mine.ptr, mine.ptr, mine.ptr, mine.ptr, 8, 1, 1, 1, 32))
        assert (mine.download() == np.arange(4)).all()


def test_arguments_off_their_boundary_are_refused(ctx):
    """Words at odd halves and ints at odd bytes, one argument at a time; nothing is
    launched."""
    rng = np.random.default_rng(1)
    nh, nkv, hd, S, T = 4, 2, 64, 12, 3
    ctx.rope_init(hd, S, 10000)
    cache = Cache(ctx, 8, 1, S, nkv, hd)
    before = cache.read()
    n = S * (nh + 2 * nkv) * hd
    bufs = [ctx.to_device(np.full(n, 5)) for _ in range(6)]
    w = [b.ptr for b in bufs]
    q, f = cache.c, intllm.hip_lib()
    calls = {        # the call, its words and its ints (places among the arguments)
        "q48_qcache_store_rows": ([q, 0, 0, T, w[0], w[1], nkv * hd], (4, 5), ()),
        "q48_qcache_load_rows": ([w[0], w[1], q, 0, 0, T, nkv * hd], (0, 1), ()),
        "q48_rope_store_rows_qcache": ([w[0], q, 0, 0, T, w[1], nh], (0,), (5,)),
        "q48_attn_decode_qcache": ([w[0], w[1], q, w[2], w[3], 0, 2, nh], (0, 1, 3, 4), ()),
        "q48_attn_decode_rope_qcache": ([w[0], w[1], q, w[2], w[3], 0, 2, nh], (0, 1, 3, 4), ()),
        "q48_attn_rows_qcache": ([w[0], w[1], q, 0, 0, T, nh, w[2]], (0, 1, 7), ()),
        "q48_attn_tree": ([w[0], w[1], w[2], w[3], 0, 0, T, nh, nkv, hd, S, w[4]], (0, 1, 2, 3, 11),
                          ()),
        "q48_rope_store_rows_at": ([w[0], w[1], w[2], 0, 0, T, w[3], nh, nkv, hd, S], (0, 1, 2),
                                   (6,)),
        "q48_cache_keep_rows": ([w[0], w[1], 1, 0, w[2], 2, nkv, hd, S], (0, 1), (4,)),
        "q48_qcache_keep_rows": ([q, 0, w[0], 2], (), (2,)),
        "q48_logprobs_rows": ([w[0], T, 100, w[1], w[2], w[3], 2, w[4], w[5]], (0, 4, 5, 8),
                              (3, 7)),
    }
    for name, (args, words, ints) in calls.items():
        for at, off in [(i, 4) for i in words] + [(i, 1) for i in words] + [(i, 2) for i in ints]:
            a = list(args)
            a[at] += off
            a = [C.byref(x) if isinstance(x, intllm.QCache) else x for x in a]
            assert getattr(f, name)(ctx.h, *a) == intllm.Q48_EINVAL, (name, at, off)
    assert all((a == b).all() for a, b in zip(before, cache.read()))
    assert all((b.download() == 5).all() for b in bufs)
    cache.free()
