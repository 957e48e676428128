"""Weights in 8 bits and their products on the GPU, word for word against the plain form
in Python integers.
"""
import numpy as np
import pytest

import intllm
import w8_plain as W

pytestmark = pytest.mark.gpu
I64 = np.iinfo(np.int64)


def words(rng, *shape, sigma=1.0):
    return (rng.standard_normal(shape) * (sigma * W.ONE)).astype(np.int64)


def weights(rng, *shape, sigma=0.02):
    c = np.clip(np.rint(rng.standard_normal(shape) * 32), -127, 127).astype(np.int8)
    return c, (rng.uniform(0.7, 1.3, shape[:-1]) * (sigma / 32 * W.ONE)).astype(np.int64)


def raw(ctx, a):
    """Any array's bytes on the device."""
    b = np.ascontiguousarray(a).view(np.uint8).ravel()
    return ctx.to_device(np.concatenate([b, np.zeros(-b.size % 8, np.uint8)]).view(np.int64))


def put(ctx, w, i, codes, steps):
    ctx.w8_put(w, i, raw(ctx, codes).ptr, ctx.to_device(steps).ptr)
    ctx.sync()


def loaded(ctx, codes, steps):
    """A matrix (or a stack of them) on the device."""
    c, s = (codes, steps) if codes.ndim == 3 else (codes[None], steps[None])
    w = ctx.new_w8(*c.shape)
    for i in range(c.shape[0]):
        put(ctx, w, i, c[i], s[i])
    return w


@pytest.fixture
def own():
    """A context whose buffers go with the test."""
    with intllm.Context(0) as c:
        yield c


SIZES = [(1, 1), (1, 64), (16, 64), (15, 63), (17, 65), (3, 1000), (33, 129), (100, 2048), (7, 5633)]
LONG = [(21, 2049), (5, 4096), (33, 4097), (17, 8193), (3, 16384), (2, 16385)]


@pytest.mark.parametrize("N,K", SIZES + LONG)
def test_weights_from_words(own, N, K):
    rng = np.random.default_rng(N * 10007 + K)
    x = words(rng, N, K, sigma=0.02)
    x[N // 2] = 0
    x[0, K // 2] = I64.min
    if N > 2:
        x[2] = rng.integers(-3, 4, K)          # steps of a word or two
    c, s = W.quantise(x)
    w = own.new_w8(1, N, K)
    bufs = w.bufs
    for b in bufs:
        b.upload(np.full(b.n, -1))
    own.w8_pack(w, 0, own.to_device(x).ptr)
    assert (bufs[1].download() == s).all()
    assert (bufs[0].download().view(np.int8) == W.tiles(c)).all()
    out = own.to_device(np.full(N * K + 1, 5))
    own.w8_values(out.ptr, w, 0)
    got = out.download()
    assert (got[:-1].reshape(N, K) == W.values(c, s)).all() and got[-1] == 5


@pytest.mark.parametrize("N", [1 << 24, (1 << 20) + 5])
def test_the_most_rows(own, N):
    """Codes put and read back, and a token's product, with as many rows as there may be."""
    rng = np.random.default_rng(7)
    codes, steps = rng.integers(-128, 128, (N, 1)).astype(np.int8), rng.integers(0, 1 << 40, N)
    w = loaded(own, codes, steps)
    out = own.buffer(N)
    own.w8_values(out.ptr, w, 0)
    assert (out.download() == codes[:, 0].astype(np.int64) * steps).all()
    own.gemm_w8(out.ptr, None, w, own.to_device(np.array([127 << 48])).ptr, None, 1)
    # 127 2^48: the code 127 and the step 2^48
    assert (out.download() == 127 * codes[:, 0].astype(np.int64) * steps).all()


def test_one_of_several_matrices(own):
    """The others stay as they are."""
    rng = np.random.default_rng(1)
    N, K, n = 21, 70, 3
    w = own.new_w8(n, N, K)
    codes, steps = weights(rng, n, N, K)
    steps[1, 3] = -5                           # counts as 0
    codes[1, 4, 5] = -128
    for i in (2, 0, 1):
        put(own, w, i, codes[i], steps[i])
    for i in range(n):
        out = own.buffer(N * K)
        own.w8_values(out.ptr, w, i)
        assert (out.download().reshape(N, K) == W.values(codes[i], steps[i].clip(0))).all()
    x = words(rng, N, K)
    own.w8_pack(w, 1, own.to_device(x).ptr)
    tiles = w.bufs[0].download().view(np.int8).reshape(n, -1)
    for i in range(n):
        assert (tiles[i] == W.tiles(W.quantise(x)[0] if i == 1 else codes[i])).all()


def check(ctx, T, N, K, norm, base, rng, X=None, codes=None, steps=None):
    X = words(rng, T, K) if X is None else X
    if codes is None:
        codes, steps = weights(rng, N, K)
    nw = W.ONE + words(rng, K, sigma=0.1) if norm else None
    b = words(rng, T, N) if base else None
    w = loaded(ctx, codes, steps)
    dX, dn = ctx.to_device(X), ctx.to_device(nw) if norm else None
    want = W.product(X, nw, codes, steps.clip(0), b)
    y = ctx.to_device(np.full(T * N + 1, 5))
    db = ctx.to_device(b) if base else None
    ctx.gemm_w8(y.ptr, db and db.ptr, w, dX.ptr, dn and dn.ptr, T)
    got = y.download()
    assert (got[:-1].reshape(T, N) == want).all() and got[-1] == 5
    assert (dX.download() == X.ravel()).all()
    if base:                                   # onto the base itself
        assert (db.download() == b.ravel()).all()
        ctx.gemm_w8(db.ptr, db.ptr, w, dX.ptr, dn and dn.ptr, T)
        assert (db.download().reshape(T, N) == want).all()


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("N,K", SIZES)
@pytest.mark.parametrize("T", [1, 3])
def test_products_of_few_rows(own, T, N, K, norm):
    check(own, T, N, K, norm, norm, np.random.default_rng(T * N + K))


@pytest.mark.parametrize("T,N,K", [(2, 40, 300), (15, 33, 130), (16, 64, 64), (17, 31, 257), (31, 48, 100),
                                   (32, 130, 64), (33, 100, 640), (63, 70, 65), (64, 64, 512),
                                   (65, 17, 700), (127, 129, 130), (128, 128, 128), (129, 255, 300),
                                   (200, 300, 200), (257, 257, 257), (300, 128, 1030)])
@pytest.mark.parametrize("norm,base", [(False, True), (True, False)])
def test_products_of_many_rows(own, T, N, K, norm, base):
    check(own, T, N, K, norm, base, np.random.default_rng(T * N + K))


@pytest.mark.parametrize("T", [1, 40])
def test_products_of_decode_shapes(own, T):
    check(own, T, 2048, 5632, False, True, np.random.default_rng(T))
    check(own, T, 2560, 2048, True, False, np.random.default_rng(T + 1))


@pytest.mark.parametrize("T", [1, 20, 150])
def test_the_longest_rows(own, T):
    """K = 131072 with every code at the end of its range: sums near 2^31."""
    rng = np.random.default_rng(5)
    K, N = 1 << 17, 5
    X = np.full((T, K), W.ONE)
    X[T // 2] = -W.ONE
    codes = np.full((N, K), 127, dtype=np.int8)
    codes[1] = -128
    codes[2, ::2] = -127
    steps = np.array([W.ONE // 5, W.ONE // 3, 7, (1 << 63) - 1, -1])
    check(own, T, N, K, False, False, rng, X, codes, steps)
    with pytest.raises(intllm.Q48Error):
        own.new_w8(1, N, K + 1)


@pytest.mark.parametrize("T", [1, 20, 150])
def test_extreme_words(own, T):
    """Rows of the ends of the words' range, of zeros, of single units; steps of 0, 1 and
    the largest: results mod 2^64."""
    rng = np.random.default_rng(T)
    N, K = 40, 200
    X = words(rng, T, K)
    X[0] = rng.choice([I64.min, I64.max, 0, 1, -1], K)
    if T > 5:
        X[1], X[2], X[3] = 0, I64.min, rng.integers(-2, 3, K)
        X[4] = rng.integers(I64.min, I64.max, K)
    codes, steps = weights(rng, N, K)
    steps[:6] = [0, 1, I64.max, I64.max // 127, W.ONE, W.ONE // 127]
    codes[7] = 0
    for norm in (False, True):
        check(own, T, N, K, norm, True, rng, X, codes, steps)


@pytest.mark.parametrize("T,N,K,norm", [(1, 5, 9, True), (1, 688, 256, True), (1, 1408, 2048, False),
                                        (1, 5632, 2048, True), (4, 33, 65, False), (16, 100, 300, True),
                                        (17, 50, 64, True), (65, 130, 128, True), (130, 200, 257, False),
                                        (300, 129, 256, True)])
def test_swiglu(own, T, N, K, norm):
    rng = np.random.default_rng(T + N)
    X = words(rng, T, K, sigma=2.0)
    gate, up = weights(rng, N, K, sigma=0.1), weights(rng, N, K, sigma=0.1)
    gate[1][N // 2] *= 40                       # past the sigmoid's 10 on both sides
    up[1][N // 3] = 0
    nw = W.ONE + words(rng, K, sigma=0.1) if norm else None
    g, u = loaded(own, *gate), loaded(own, *up)
    out = own.to_device(np.full(T * N + 1, 5))
    own.gemm_w8_swiglu(out.ptr, g, u, own.to_device(X).ptr, own.to_device(nw).ptr if norm else None,
                       T)
    got = out.download()
    assert (got[:-1].reshape(T, N) == W.swiglu(X, nw, gate, up)).all() and got[-1] == 5


@pytest.mark.parametrize("T", [1, 40, 1100])
def test_swiglu_of_large_gates(own, T):
    """Gates on either side of 10 in magnitude, where the sigmoid ends; results on either
    side of 2^51, 2^52 and 2^53."""
    rng = np.random.default_rng(T)
    N, K = 3000 if T == 1100 else 70, 130
    gate, up = weights(rng, N, K, sigma=0.5), weights(rng, N, K, sigma=0.5)
    X = words(rng, T, K)
    X[1::3] = X[1::3] // 16
    want = W.swiglu(X, None, gate, up)
    size = abs(want.ravel())
    assert (size < 2 ** 51).any() and (size > 2 ** 51).any() and (size > 2 ** 53).any()
    out = own.buffer(T * N)
    own.gemm_w8_swiglu(out.ptr, loaded(own, *gate), loaded(own, *up), own.to_device(X).ptr, None, T)
    assert (out.download().reshape(T, N) == want).all()


def test_rows_off_sixteen_bytes(own):
    """Words on the boundary of a word and no more."""
    rng = np.random.default_rng(9)
    for T, N, K in ((1, 65, 64), (3, 40, 2048), (1, 31, 5632), (70, 64, 128)):
        X, b = words(rng, T, K), words(rng, T, N)
        codes, steps = weights(rng, N, K)
        nw = W.ONE + words(rng, K, sigma=0.1)
        w = loaded(own, codes, steps)
        dX, dn = own.to_device(np.append(0, X)), own.to_device(np.append(0, nw))
        db, y = own.to_device(np.append(0, b)), own.buffer(T * N + 1)
        own.gemm_w8(y.at(1), db.at(1), w, dX.at(1), dn.at(1), T)
        assert (y.download()[1:].reshape(T, N) == W.product(X, nw, codes, steps, b)).all()


def test_weights_off_sixteen_bytes(own):
    rng = np.random.default_rng(10)
    for N, K in ((21, 300), (9, 2047), (17, 3001), (3, 4097)):
        x = words(rng, N, K)
        c, s = W.quantise(x)
        w = own.new_w8(1, N, K)
        own.w8_pack(w, 0, own.to_device(np.append(0, x)).at(1))
        out = own.to_device(np.full(N * K + 2, 5))
        own.w8_values(out.at(1), w, 0)
        got = out.download()
        assert got[0] == 5 and got[-1] == 5
        assert (got[1:-1].reshape(N, K) == W.values(c, s)).all()


@pytest.mark.parametrize("K", [2049, 4096, 4097, 6145, 8192, 8193, 9000, 16384, 16385])
@pytest.mark.parametrize("T", [1, 5, 300])
def test_long_rows(own, T, K):
    """Every form that a row's length selects, with an outlier past 32 in some rows."""
    rng = np.random.default_rng(K)
    X = words(rng, T, K)
    X[T // 2, K // 3] = 40 * W.ONE
    X[T - 1, K - 1] = -(1 << 60)
    codes, steps = weights(rng, 20, K)
    check(own, T, 20, K, K % 2 == 0, True, rng, X, codes, steps)
    w = own.new_w8(1, 20, K)
    x = words(rng, 20, K, sigma=0.02)
    own.w8_pack(w, 0, own.to_device(x).ptr)
    out = own.buffer(20 * K)
    own.w8_values(out.ptr, w, 0)
    assert (out.download().reshape(20, K) == W.values(*W.quantise(x))).all()


@pytest.mark.parametrize("N,T", [(1, 1100), (17, 2100), (2100, 1000), (4100, 700)])
def test_tiles_of_many_outputs(own, N, T):
    """Both forms for many rows, on either side of where they change."""
    rng = np.random.default_rng(N)
    check(own, T, N, 90, False, True, rng)
    X = words(rng, T, 600)
    gate, up = weights(rng, N, 600), weights(rng, N, 600)
    out = own.buffer(T * N)
    own.gemm_w8_swiglu(out.ptr, loaded(own, *gate), loaded(own, *up), own.to_device(X).ptr, None, T)
    assert (out.download().reshape(T, N) == W.swiglu(X, None, gate, up)).all()


def test_results_past_four_gib():
    """Offsets that pass 32 bits in the results, of products and of SwiGLU."""
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(5)
    distinct, N, K = 7, 2048, 70
    T = distinct * 40000                       # 4.6 GB of results
    X = words(rng, distinct, K)
    gate, up = weights(rng, N, K), weights(rng, N, K)
    with intllm.Context(0, stream=torch.cuda.current_stream(0).cuda_stream) as c:
        g, u = loaded(c, *gate), loaded(c, *up)
        d = torch.from_numpy(X).to("cuda:0").repeat(T // distinct, 1)
        y = torch.full((T, N), 3, dtype=torch.int64, device="cuda:0")
        c.gemm_w8(y.data_ptr(), y.data_ptr(), g, d.data_ptr(), None, T)
        want = torch.from_numpy(W.product(X, None, *gate).astype(np.int64) + 3).to("cuda:0")
        assert bool((y.view(-1, distinct, N) == want).all())
        c.gemm_w8_swiglu(y.data_ptr(), g, u, d.data_ptr(), None, T)
        want = torch.from_numpy(W.swiglu(X, None, gate, up).astype(np.int64)).to("cuda:0")
        assert bool((y.view(-1, distinct, N) == want).all())
        c.sync()


def test_on_the_callers_stream():
    """Rows that torch is still making when the product is enqueued, results that torch
    reads and rows that it overwrites right behind it."""
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(3)
    T, N, K = 40, 96, 700
    codes, steps = weights(rng, N, K)
    X = words(rng, T, K)
    want = W.product(X, None, codes, steps)
    for s in (torch.cuda.default_stream(0), torch.cuda.Stream(0)):
        with torch.cuda.stream(s), intllm.Context(0, stream=s.cuda_stream) as c:
            w = loaded(c, codes, steps)
            y = torch.zeros(T, N, dtype=torch.int64, device="cuda:0")
            d = torch.zeros(T, K, dtype=torch.int64, device="cuda:0")
            c.gemm_w8(y.data_ptr(), None, w, d.data_ptr(), None, T)
            host = torch.from_numpy(X).pin_memory()
            big = torch.randn(4096, 4096, device="cuda:0")
            for _ in range(3):
                for _ in range(4):
                    big = torch.mm(big, big) * 1e-4
                d.copy_(host, non_blocking=True)
                c.gemm_w8(y.data_ptr(), None, w, d.data_ptr(), None, T)
                got = y + 1
                d.zero_()
                y.zero_()
                assert (got.cpu().numpy() == want + 1).all()


def test_two_graphs_share_a_buffer(own):
    """Two captured products of one context, replayed in turns."""
    rng = np.random.default_rng(4)
    lib, c = intllm.hip_lib(), own
    import ctypes as C
    codes, steps = weights(rng, 50, 256)
    w = loaded(c, codes, steps)
    graphs = []
    for T in (3, 40):
        X = words(rng, T, 256)
        dX, y = c.to_device(X), c.buffer(T * 50)
        c.gemm_w8(y.ptr, None, w, dX.ptr, None, T)
        c.sync()
        intllm.check("capture", lib.q48_graph_capture(c.h))
        c.gemm_w8(y.ptr, None, w, dX.ptr, None, T)
        g = C.c_void_p()
        intllm.check("instantiate", lib.q48_graph_instantiate(c.h, C.byref(g)))
        graphs.append((g, X, dX, y))
    for i in range(3):
        for g, X, dX, y in graphs:
            dX.upload(X + i)
            y.upload(np.zeros(y.n, np.int64))
            intllm.check("replay", lib.q48_graph_replay(c.h, g, 1))
        for g, X, dX, y in graphs:
            assert (y.download().reshape(-1, 50) == W.product(X + i, None, codes, steps)).all()
    for g, *_ in graphs:
        intllm.check("destroy", lib.q48_graph_destroy(c.h, g))


def test_captured_and_replayed(own):
    """Products of one shape as a graph, its inputs changed between replays, eager calls
    of other shapes among them; a shape that was never called is refused in a capture."""
    rng = np.random.default_rng(2)
    lib, c = intllm.hip_lib(), own
    T, N, K = 3, 96, 300
    gate, up, down = weights(rng, N, K), weights(rng, N, K), weights(rng, K, N)
    g, u, d = (loaded(c, *w) for w in (gate, up, down))
    nw = W.ONE + words(rng, K, sigma=0.1)
    dn, dX, h = c.to_device(nw), c.buffer(T * K), c.buffer(T * N)

    def step():
        c.gemm_w8_swiglu(h.ptr, g, u, dX.ptr, dn.ptr, T)
        c.gemm_w8(dX.ptr, dX.ptr, d, h.ptr, None, T)

    step()
    c.sync()
    many, into = c.buffer(3990 * K), c.buffer(3990 * N)
    intllm.check("begin", lib.q48_graph_begin(c.h))
    step()
    with pytest.raises(intllm.Q48Error) as err:
        c.gemm_w8(into.ptr, None, g, many.ptr, None, 3990)
    assert err.value.code == intllm.Q48_ESTATE
    intllm.check("end", lib.q48_graph_end(c.h))
    x = words(rng, T, K)
    dX.upload(x)
    other = words(rng, 200, K)
    do, oo = c.to_device(other), c.buffer(200 * N)
    for i in range(4):
        intllm.check("launch", lib.q48_graph_launch(c.h, 1))
        x = W.product(W.swiglu(x, nw, gate, up), None, *down, x)
        assert (dX.download().reshape(T, K) == x).all(), i
        if i < 2:
            c.gemm_w8(oo.ptr, None, g, do.ptr, dn.ptr, 200)   # grows the context's buffer once
            assert (oo.download().reshape(200, N) == W.product(other, nw, *gate)).all()
    intllm.check("drop", lib.q48_graph_drop(c.h))


@pytest.mark.parametrize("N", [(1 << 24) - 7, (1 << 20) + 5])
def test_the_most_rows_from_words(N):
    """As many rows of words as there may be, of a length that takes four waves a row: every
    row's codes and step, in the layout that the header gives."""
    torch = pytest.importorskip("torch")
    K, KT, NT, at = 513, 9, (N + 15) // 16, "cuda:0"
    with intllm.Context(0, stream=torch.cuda.current_stream(0).cuda_stream) as c:
        assert intllm.w8_bytes(1, N, K) == (NT * KT * 1024, N * 8)
        g = torch.Generator(device=at).manual_seed(N)
        some = torch.randint(-(1 << 44), 1 << 44, (4096, K), generator=g, device=at)
        x = some.repeat((N + 4095) // 4096, 1)[:N]
        x[:, 7] = torch.arange(N, device=at) << 22                # every row another step
        codes = torch.full((NT, KT, 4, 16, 16), -1, dtype=torch.int8, device=at)
        steps = torch.full((N,), -1, dtype=torch.int64, device=at)
        c.w8_pack(c.w8(codes.data_ptr(), steps.data_ptr(), 1, N, K), 0, x.data_ptr())
        for n in range(0, NT * 16, 1 << 20):
            w, rows = x[n:n + (1 << 20)], codes[n // 16:(n + (1 << 20)) // 16]
            step = (w.abs().amax(1) + 126) // 127
            assert bool((steps[n:n + (1 << 20)] == step).all()), n
            got = rows.permute(0, 3, 1, 2, 4).reshape(-1, KT * 64)
            want = ((w.abs() + (step >> 1)[:, None]) // step[:, None]).clamp_(max=127) * w.sign()
            assert bool((got[:w.shape[0], :K] == want).all()), n
            assert not bool(got[w.shape[0]:].any()) and not bool(got[:, K:].any()), n
        c.sync()
    del x, codes, some
    torch.cuda.empty_cache()


def test_graphs_outlive_a_grown_buffer(own):
    """Eager products of ever more rows, past the context's first MiB, between the replays of
    a graph that holds the buffer's first address."""
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(12)
    lib, c = intllm.hip_lib(), own
    T, N, K = 3, 96, 300
    gate, up, down = weights(rng, N, K), weights(rng, N, K), weights(rng, K, N)
    g, u, d = (loaded(c, *w) for w in (gate, up, down))
    x = words(rng, T, K)
    dX, h = c.to_device(x), c.buffer(T * N)

    def step():
        c.gemm_w8_swiglu(h.ptr, g, u, dX.ptr, None, T)
        c.gemm_w8(dX.ptr, dX.ptr, d, h.ptr, None, T)

    step()
    c.sync()
    intllm.check("begin", lib.q48_graph_begin(c.h))
    step()
    intllm.check("end", lib.q48_graph_end(c.h))
    dX.upload(x)
    some = words(rng, 50, K)
    want = W.product(some, None, *gate)
    for i in range(3):
        intllm.check("launch", lib.q48_graph_launch(c.h, 1))
        x = W.product(W.swiglu(x, None, gate, up), None, *down, x)
        assert (dX.download().reshape(T, K) == x).all(), i
        n = 50 * (400 << i)
        do, oo = c.to_device(np.tile(some, (n // 50, 1))), c.buffer(n * N)
        torch.cuda.synchronize()
        free = torch.cuda.mem_get_info()[0]
        c.gemm_w8(oo.ptr, None, g, do.ptr, None, n)
        assert (oo.download().reshape(-1, 50, N) == want).all()
        assert torch.cuda.mem_get_info()[0] < free            # it has grown
    intllm.check("drop", lib.q48_graph_drop(c.h))


def test_weights_given_back(own):
    """The card has their memory again; they are refused, and the context works on."""
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(14)
    codes, steps = weights(rng, 40, 100)
    kept = loaded(own, codes, steps)
    x = words(rng, 3, 100)
    dx, y = own.to_device(x), own.buffer(3 * 40)
    own.gemm_w8(y.ptr, None, kept, dx.ptr, None, 3)
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    big = own.new_w8(3, 4096, 8192)
    put(own, big, 1, *weights(rng, 4096, 8192))
    assert torch.cuda.mem_get_info()[0] < free - 3 * 4096 * 8192 + 1
    own.free_w8(big)
    assert torch.cuda.mem_get_info()[0] > free - 2 * 4096 * 8192      # (the words that were put)
    with pytest.raises(intllm.Q48Error):
        own.w8_values(y.ptr, big, 1)
    own.free_w8(big)
    own.gemm_w8(y.ptr, None, kept, dx.ptr, None, 3)
    assert (y.download().reshape(3, 40) == W.product(x, None, codes, steps)).all()
