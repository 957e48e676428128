"""The mixture-of-experts layer on the GPU, word for word against the plain form in
Python integers.
"""
import numpy as np
import pytest

import intllm
import w8_plain as W
from test_gpu_w8 import loaded, own, raw, weights, words  # noqa: F401

pytestmark = pytest.mark.gpu


class Layer:
    def __init__(self, rng, E, dim, ffn, sigma=0.02):
        self.E, self.dim, self.ffn = E, dim, ffn
        self.router = words(rng, E, dim, sigma=1.4 / dim ** 0.5)
        self.gate, self.up = weights(rng, E, ffn, dim, sigma=sigma), weights(rng, E, ffn, dim, sigma=sigma)
        self.down = weights(rng, E, dim, ffn, sigma=sigma)
        self.norm = W.ONE + words(rng, dim, sigma=0.1)

    def load(self, ctx, top, renorm):
        self.w = [loaded(ctx, *w) for w in (self.gate, self.up, self.down)]
        return ctx.moe(ctx.to_device(self.router).ptr, *self.w, top, renorm)

    def want(self, X, norm, top, renorm, base):
        return W.moe(X, self.norm if norm else None, self.router, self.gate, self.up, self.down, top,
                     renorm, base)


def check(ctx, layer, X, top, renorm, norm=True, base="X"):
    T, dim = X.shape
    rng = np.random.default_rng(T)
    m = layer.load(ctx, top, renorm)
    b = X if base == "X" else words(rng, T, dim) if base else None
    want = layer.want(X, norm, top, renorm, b)
    dX, dn = ctx.to_device(X), ctx.to_device(layer.norm) if norm else None
    db = dX if base == "X" else ctx.to_device(b) if base else None
    out = ctx.to_device(np.full(T * dim + 1, 5))
    ch, wt = raw(ctx, np.full(T * top + 1, 5, np.int32)), ctx.to_device(np.full(T * top + 1, 5))
    ctx.moe_w8(out.ptr, db and db.ptr, m, dX.ptr, dn and dn.ptr, T, ch.ptr, wt.ptr)
    ids = ch.download().view(np.int32)
    assert (ids[:T * top].reshape(T, top) == want[1]).all() and ids[T * top] == 5
    got = wt.download()
    assert (got[:-1].reshape(T, top) == want[2]).all() and got[-1] == 5
    got = out.download()
    assert (got[:-1].reshape(T, dim) == want[0]).all() and got[-1] == 5
    assert (dX.download() == X.ravel()).all()
    if db:                                     # in place, the choice not asked for
        ctx.moe_w8(db.ptr, db.ptr, m, dX.ptr, dn and dn.ptr, T)
        assert (db.download().reshape(T, dim) == want[0]).all()


@pytest.mark.parametrize("T", [1, 2, 7, 16, 17, 40, 130])
@pytest.mark.parametrize("E,top,renorm", [(1, 1, False), (2, 2, True), (8, 2, True), (8, 1, False),
                                          (60, 4, False), (64, 8, True), (65, 3, True)])
def test_layers(own, T, E, top, renorm):  # noqa: F811
    rng = np.random.default_rng(T * 100 + E)
    layer = Layer(rng, E, 96, 80)
    check(own, layer, words(rng, T, 96), top, renorm, norm=E % 2 == 0, base=("X", True, None)[T % 3])


@pytest.mark.parametrize("dim,ffn", [(1, 1), (64, 64), (63, 65), (65, 1), (1, 130), (256, 688), (1000, 33),
                                     (2048, 1024)])
@pytest.mark.parametrize("T", [1, 5])
def test_sizes(own, dim, ffn, T):  # noqa: F811
    rng = np.random.default_rng(dim + ffn)
    check(own, Layer(rng, 4, dim, ffn), words(rng, T, dim), 2, True)


@pytest.mark.parametrize("dim,ffn", [(2049, 40), (4000, 9000), (6144, 33), (6145, 33), (8300, 20)])
@pytest.mark.parametrize("T", [1, 3])
def test_long_rows(own, dim, ffn, T):  # noqa: F811
    rng = np.random.default_rng(dim)
    X = words(rng, T, dim)
    X[T - 1, dim // 2] = 40 * W.ONE
    check(own, Layer(rng, 3, dim, ffn), X, 2, T == 1)


@pytest.mark.parametrize("top", [2, 16])
def test_a_token_of_long_hidden_rows_in_a_used_buffer(own, top):  # noqa: F811
    """Hidden rows too long for the form of one token, where an earlier call left the
    buffer full of other words: no slot and no item of it may be taken for one of now."""
    rng = np.random.default_rng(top)
    big = loaded(own, *weights(rng, 16, 2048))
    X = rng.integers(-2 ** 62, 2 ** 62, (12000, 2048))
    Y = own.buffer(12000 * 16)
    own.gemm_w8(Y.ptr, None, big, own.to_device(X).ptr, None, 12000)
    check(own, Layer(rng, 16, 48, 8300), words(rng, 1, 48), top, True)


@pytest.mark.parametrize("T,E", [(60, 40), (200, 15), (256, 16), (257, 16), (300, 64), (307, 64), (308, 64),
                                 (768, 8), (769, 8), (1025, 4)])
def test_where_the_routing_changes(own, T, E):  # noqa: F811
    """A token's experts in one block, in several, in more blocks than are resident, and the
    separate launches."""
    rng = np.random.default_rng(E)
    check(own, Layer(rng, E, 100, 40), words(rng, T, 100), 3, False)


@pytest.mark.parametrize("T", [256, 512, 513])
def test_routing_of_longer_rows(own, T):  # noqa: F811
    rng = np.random.default_rng(T)
    check(own, Layer(rng, 3, 2050, 8), words(rng, T, 2050), 2, True)


@pytest.mark.parametrize("T", [1, 33])
def test_every_expert_and_many(own, T):  # noqa: F811
    """top_k of all experts; 64 of 1024."""
    rng = np.random.default_rng(T)
    check(own, Layer(rng, 5, 40, 70), words(rng, T, 40), 5, False)
    check(own, Layer(rng, 1024, 16, 3), words(rng, T, 16), 64, T == 1)


@pytest.mark.parametrize("T", [1, 20, 70])
def test_ties_go_to_the_lowest_expert(own, T):  # noqa: F811
    rng = np.random.default_rng(3)
    layer = Layer(rng, 70, 64, 32)
    layer.router[:] = layer.router[0]          # all alike
    layer.router[5::7] = layer.router[1]       # and ten others alike
    X = words(rng, T, 64)
    X[T // 2] = 0                              # a padded row: every logit 0
    check(own, layer, X, 12, True)
    check(own, layer, X, 12, False)


@pytest.mark.parametrize("T,E,top", [(300, 1, 1), (150, 2, 2), (700, 4, 2), (1100, 3, 1)])
def test_many_rows_an_expert(own, T, E, top):  # noqa: F811
    rng = np.random.default_rng(T)
    check(own, Layer(rng, E, 70, 130), words(rng, T, 70), top, True)


def test_all_tokens_to_one_expert(own):  # noqa: F811
    rng = np.random.default_rng(4)
    layer = Layer(rng, 6, 64, 48)
    X = np.abs(words(rng, 100, 64))
    layer.router = np.full((6, 64), -W.ONE)
    layer.router[4] = W.ONE
    check(own, layer, X, 1, True, norm=False)


@pytest.mark.parametrize("T", [1, 3, 40])
def test_extreme_words(own, T):  # noqa: F811
    """Logits that wrap, differences past 63 bits, rows of the ends of the words' range."""
    rng = np.random.default_rng(T)
    i64 = np.iinfo(np.int64)
    layer = Layer(rng, 9, 64, 48)
    layer.router[0] = i64.max
    layer.router[1] = i64.min
    layer.router[2] = 0
    layer.down[1][3] = i64.max
    X = rng.integers(i64.min, i64.max, (T, 64))
    X[0] = rng.choice([i64.min, i64.max], 64)
    check(own, layer, X, 4, True, norm=False, base=True)
    check(own, layer, X, 4, False, norm=True, base=None)


def test_weights_far_apart(own):  # noqa: F811
    """One expert ahead of the others by more than an exponential keeps: weights of 0."""
    rng = np.random.default_rng(8)
    layer = Layer(rng, 8, 64, 48)
    layer.router *= 200
    check(own, layer, words(rng, 9, 64), 4, True)


def test_long_inputs_in_passes(own):  # noqa: F811
    """More hidden words than a pass holds (a GiB): 70000 tokens of hidden rows of 1500, four
    passes, a token's words the same in each."""
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(8)
    distinct, dim, ffn, T = 10, 64, 1500, 70000
    X = words(rng, distinct, dim)
    layer = Layer(rng, 6, dim, ffn)
    with intllm.Context(0, stream=torch.cuda.current_stream(0).cuda_stream) as c:
        m = layer.load(c, 2, True)
        want, ids, wt = layer.want(X, True, 2, True, X)
        d = torch.from_numpy(X).to("cuda:0").repeat(T // distinct, 1)
        norm = torch.from_numpy(layer.norm).to("cuda:0")
        ch = torch.full((T, 2), 9, dtype=torch.int32, device="cuda:0")
        w = torch.full((T, 2), 9, dtype=torch.int64, device="cuda:0")
        c.moe_w8(d.data_ptr(), d.data_ptr(), m, d.data_ptr(), norm.data_ptr(), T, ch.data_ptr(), w.data_ptr())
        for got, one in ((d, want), (ch, ids), (w, wt)):
            one = torch.from_numpy(np.asarray(one).astype(np.int64)).to("cuda:0")
            assert bool((got.view(-1, *one.shape) == one).all())
        c.sync()


@pytest.mark.parametrize("T,top", [(1, 2), (5, 3), (90, 2)])
def test_captured_and_replayed(own, T, top):  # noqa: F811
    """A layer onto its own input as a graph, replayed among eager calls: each replay's
    choice differs from the last one's."""
    rng = np.random.default_rng(6)
    lib, c = intllm.hip_lib(), own
    layer = Layer(rng, 8, 64, 48, sigma=0.3)
    m = layer.load(c, top, True)
    x = words(rng, T, 64)
    dX, dn = c.to_device(x), c.to_device(layer.norm)
    ch, wt = c.buffer(T * top), c.buffer(T * top)
    c.moe_w8(dX.ptr, dX.ptr, m, dX.ptr, dn.ptr, T, ch.ptr, wt.ptr)
    c.sync()
    intllm.check("begin", lib.q48_graph_begin(c.h))
    c.moe_w8(dX.ptr, dX.ptr, m, dX.ptr, dn.ptr, T, ch.ptr, wt.ptr)
    intllm.check("end", lib.q48_graph_end(c.h))
    dX.upload(x)
    other = words(rng, 300, 64)
    do, oo = c.to_device(other), c.buffer(300 * 64)
    for i in range(4):
        intllm.check("launch", lib.q48_graph_launch(c.h, 1))
        x, ids, weight = layer.want(x, True, top, True, x)
        assert (dX.download().reshape(T, 64) == x).all(), i
        assert (ch.download().view(np.int32)[:T * top].reshape(T, top) == ids).all()
        assert (wt.download().reshape(T, top) == weight).all()
        if i < 2:
            c.moe_w8(oo.ptr, None, m, do.ptr, None, 300)
            assert (oo.download().reshape(300, 64) == layer.want(other, False, top, True, None)[0]).all()
    intllm.check("drop", lib.q48_graph_drop(c.h))


def grown(call):
    """Bytes of the card that a call keeps."""
    torch = pytest.importorskip("torch")
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    call()
    torch.cuda.synchronize()
    return free - torch.cuda.mem_get_info()[0]


def test_the_buffer_of_a_token_with_many_long_rows(own):  # noqa: F811
    """64 experts of hidden rows past 2^16 words for one token: its own 16 slots each."""
    rng = np.random.default_rng(12)
    E, ffn = 64, 66000
    gate, up, down = weights(rng, ffn, 1, sigma=0.3), weights(rng, ffn, 1, sigma=0.3), weights(rng, 1, ffn)
    w = []
    for codes, steps in (gate, up, down):      # the experts all alike
        a, dc, ds = own.new_w8(E, *codes.shape), raw(own, codes), own.to_device(steps)
        for e in range(E):
            own.w8_put(a, e, dc.ptr, ds.ptr)
        w.append(a)
    x, router = words(rng, 1, 1), words(rng, E, 1)
    m = own.moe(own.to_device(router).ptr, *w, E, False)
    out, dx = own.buffer(1), own.to_device(x)
    own.sync()
    most = 16 * E * ffn * 8                    # hidden words; their codes are an eighth
    assert grown(lambda: own.moe_w8(out.ptr, None, m, dx.ptr, None, 1)) < 1.5 * most < 1 << 30
    y = int(W.product(W.swiglu(x, None, gate, up), None, *down)[0, 0])
    _, weight = W.choose(W.logits(x, router)[0], E, False)
    assert int(out.download()[0]) == sum(a * y >> 48 for a in weight)


def test_the_buffer_of_many_experts(own):  # noqa: F811
    """A GiB of hidden words with every expert's last sixteen slots among them: 1024 experts
    of hidden rows of 8192, a pass after a pass."""
    rng = np.random.default_rng(13)
    E, dim, ffn, top, distinct, T = 1024, 2, 8192, 8, 5, 1000
    layer = Layer(rng, E, dim, ffn, sigma=0.3)
    m = layer.load(own, top, True)
    x = words(rng, distinct, dim)
    want = layer.want(x, False, top, True, None)
    dx, out = own.to_device(np.tile(x, (T // distinct, 1))), own.buffer(T * dim)
    ch, wt = own.buffer(T * top // 2), own.buffer(T * top)
    own.sync()
    assert grown(lambda: own.moe_w8(out.ptr, None, m, dx.ptr, None, T, ch.ptr, wt.ptr)) < 1.25 * 2 ** 30
    assert (out.download().reshape(-1, distinct, dim) == want[0]).all()
    assert (ch.download().view(np.int32).reshape(-1, distinct, top) == want[1]).all()
    assert (wt.download().reshape(-1, distinct, top) == want[2]).all()


@pytest.mark.parametrize("T,top", [(1, 2), (5, 3), (90, 2)])
def test_graphs_outlive_a_grown_buffer(own, T, top):  # noqa: F811
    """Eager layers of ever more tokens, past the context's first MiB, between the replays of
    a graph that holds the buffer's first address."""
    rng = np.random.default_rng(9)
    lib, c = intllm.hip_lib(), own
    layer = Layer(rng, 8, 64, 48, sigma=0.3)
    m = layer.load(c, top, True)
    x = words(rng, T, 64)
    dX = c.to_device(x)
    c.moe_w8(dX.ptr, dX.ptr, m, dX.ptr, None, T)
    c.sync()
    intllm.check("begin", lib.q48_graph_begin(c.h))
    c.moe_w8(dX.ptr, dX.ptr, m, dX.ptr, None, T)
    intllm.check("end", lib.q48_graph_end(c.h))
    dX.upload(x)
    some = words(rng, 50, 64)
    want = layer.want(some, False, top, True, None)[0]
    for i in range(4):
        intllm.check("launch", lib.q48_graph_launch(c.h, 1))
        x = layer.want(x, False, top, True, x)[0]
        assert (dX.download().reshape(T, 64) == x).all(), i
        n = 50 * (100 << i)                    # 5000 to 40000 tokens: another buffer each time
        do, oo = c.to_device(np.tile(some, (n // 50, 1))), c.buffer(n * 64)
        assert grown(lambda: c.moe_w8(oo.ptr, None, m, do.ptr, None, n)) > 0
        assert (oo.download().reshape(-1, 50, 64) == want).all()
        c.moe_w8(oo.ptr, None, m, do.ptr, None, 50)          # the new buffer's tickets
        assert (oo.download().reshape(-1, 50, 64)[0] == want).all()
    intllm.check("drop", lib.q48_graph_drop(c.h))
