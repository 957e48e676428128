"""q48_logprobs_rows on the GPU, word for word against the plain form in Python
integers.
"""
import numpy as np
import pytest

import intllm
import serve_plain as P

pytestmark = pytest.mark.gpu
I64 = np.iinfo(np.int64)


def ints(ctx, a):
    """An int32 array on the device (in a buffer of 8-byte words)."""
    a = np.asarray(a, dtype=np.int32).ravel()
    return ctx.to_device(np.concatenate([a, np.zeros(a.size % 2, np.int32)]).view(np.int64))


def check_rows(ctx, x, tokens, top, ask=("logp", "entropy", "top")):
    T, V = x.shape
    d, tk = ctx.to_device(x), ints(ctx, tokens)
    logp, ent = ctx.to_device(np.full(T, 5)), ctx.to_device(np.full(T, 5))
    ids, tlp = ints(ctx, np.full(T * max(1, top), 5)), ctx.to_device(np.full(T * max(1, top), 5))
    ctx.logprobs_rows(d.ptr, T, V, tk.ptr, logp.ptr if "logp" in ask else None,
                      ent.ptr if "entropy" in ask else None, top if "top" in ask else 0, ids.ptr,
                      tlp.ptr)
    want = P.logprobs(x, tokens, top)
    none = np.full(T, 5)
    assert (logp.download() == (want[0] if "logp" in ask else none)).all()
    assert (ent.download() == (want[1] if "entropy" in ask else none)).all()
    if top and "top" in ask:
        got = ids.download().view(np.int32)[:T * top].reshape(T, top)
        assert (got == want[2]).all()
        assert (tlp.download().reshape(T, top) == want[3]).all()
    assert (d.download() == x.ravel()).all()


def logits(rng, T, V, sigma=2.5):
    return (rng.standard_normal((T, V)) * (sigma * P.ONE)).astype(np.int64)


@pytest.mark.parametrize("V", [1, 2, 3, 63, 64, 65, 255, 257, 1000, 4095, 4097, 9001, 32000])
@pytest.mark.parametrize("top", [0, 1, 5, 32])
def test_sizes(ctx, V, top):
    rng = np.random.default_rng(V)
    T = 3 if V < 9000 else 1
    x = logits(rng, T, V)
    check_rows(ctx, x, rng.integers(0, V, T), min(top, V))


@pytest.mark.parametrize("T", [1, 2, 7, 64, 300])
def test_rows(ctx, T):
    rng = np.random.default_rng(T)
    x = logits(rng, T, 400)
    tokens = rng.integers(0, 400, T)
    tokens[T // 2] = -1
    if T > 3:
        tokens[1], tokens[2] = 400, I64.min >> 40   # past the vocabulary; far negative
    check_rows(ctx, x, tokens, 20)


def test_a_large_vocabulary(ctx):
    rng = np.random.default_rng(1)
    check_rows(ctx, logits(rng, 2, 151937), [151936, 0], 20)


def batch(rng, T, V):
    """T rows of V logits that are eight rows over and over, and what they give."""
    x = logits(rng, 8, V)
    return np.tile(x, (T // 8 + 1, 1))[:T], lambda tokens, top: [
        np.tile(w, (T // 8 + 1,) + (1,) * (w.ndim - 1))[:T] for w in P.logprobs(x, tokens, top)]


@pytest.mark.parametrize("T,V", [(600, 3000), (300, 8192), (70, 12000), (300, 16384), (20, 12000),
                                 (140, 20000), (600, 32768), (130, 32767), (40, 32769), (40, 8200),
                                 (9, 70001)])
def test_many_rows(ctx, T, V):
    """More rows than a launch's blocks, and every form's largest row."""
    rng = np.random.default_rng(T + V)
    x, want = batch(rng, T, V)
    tokens = rng.integers(0, V, 8)
    d, tk = ctx.to_device(x), ints(ctx, np.tile(tokens, T // 8 + 1)[:T])
    logp, ent, ids, tlp = ctx.buffer(T), ctx.buffer(T), ctx.buffer(T * 9), ctx.buffer(T * 9)
    ctx.logprobs_rows(d.ptr, T, V, tk.ptr, logp.ptr, ent.ptr, 9, ids.ptr, tlp.ptr)
    w = want(tokens, 9)
    assert (logp.download() == w[0]).all() and (ent.download() == w[1]).all()
    assert (ids.download().view(np.int32)[:T * 9].reshape(T, 9) == w[2]).all()
    assert (tlp.download().reshape(T, 9) == w[3]).all()
    for b in (d, tk, logp, ent, ids, tlp):
        b.free()


def edges(width=300):
    rng = np.random.default_rng(0)
    x = logits(rng, 12, width)
    x[0] = 0                                  # all the same: ties to the lowest id
    x[1] = I64.min                            # the type's lowest value everywhere
    x[2, ::2] = I64.min                       # and as a mask
    x[3, 7], x[3, 8] = I64.max, I64.min       # u past 63 bits: the smallest log probability
    x[4] = -1
    x[4, -1] = 0                             # the last id alone
    x[5] >>= 40
    x[6, 3:9] = x[6].max() + 5                # ties at the top
    x[7] = np.arange(width) % 400 * (P.LN2 // 3)      # u at multiples of LN2
    x[8] = -(np.arange(width) % 4000) * (1 << 42)     # and of the table's step
    x[9] = I64.max - np.arange(width)
    x[10] = np.where(np.arange(width) == 40, 0, -(45 << 48))   # e below 2^-48 but one
    x[11] *= 40
    return x


@pytest.mark.parametrize("top", [0, 3, 32])
@pytest.mark.parametrize("width", [300, 9000])
def test_edges(ctx, top, width):
    x = edges(width)
    tokens = np.arange(12) * 24 + 8
    tokens[3] = 8
    check_rows(ctx, x, tokens, top)


@pytest.mark.parametrize("ask", [("logp",), ("entropy",), ("top",), ("logp", "top")])
def test_parts(ctx, ask):
    rng = np.random.default_rng(12)
    check_rows(ctx, logits(rng, 5, 777), rng.integers(0, 777, 5), 6, ask)


def test_probabilities_add_up(ctx):
    """Every token's log probability: their exponentials add up to one (each e^logp is
    within 2^-47 of its probability, 2000 of them within 2^-36)."""
    rng = np.random.default_rng(2)
    V = 2000
    row = logits(rng, 1, V)
    x = np.repeat(row, V, 0)
    d, tk, logp = ctx.to_device(x), ints(ctx, np.arange(V)), ctx.buffer(V)
    ctx.logprobs_rows(d.ptr, V, V, tk.ptr, logp.ptr, None)
    lp = logp.download().astype(np.float64) / P.ONE
    assert abs(np.exp(lp).sum() - 1) < 2.0 ** -36
    f = row[0].astype(np.float64) / P.ONE
    assert np.abs(lp - (f - np.log(np.exp(f - f.max()).sum()) - f.max())).max() < 2.0 ** -35


def test_captured(ctx):
    """Replays of a captured call, the logits changed between them."""
    rng = np.random.default_rng(5)
    lib = intllm.hip_lib()
    T, V, top = 5, 5000, 7
    with intllm.Context(0) as c:
        d, tk = c.buffer(T * V), ints(c, rng.integers(0, V, T))
        logp, ent, ids, tlp = c.buffer(T), c.buffer(T), c.buffer(T * top), c.buffer(T * top)

        def call():
            c.logprobs_rows(d.ptr, T, V, tk.ptr, logp.ptr, ent.ptr, top, ids.ptr, tlp.ptr)

        d.upload(logits(rng, T, V))
        call()
        c.sync()
        intllm.check("begin", lib.q48_graph_begin(c.h))
        call()
        intllm.check("end", lib.q48_graph_end(c.h))
        for _ in range(4):
            x = logits(rng, T, V)
            d.upload(x)
            intllm.check("launch", lib.q48_graph_launch(c.h, 1))
            got = [b.download() for b in (logp, ent, ids, tlp)]
            call()
            assert all((b.download() == g).all() for b, g in zip((logp, ent, ids, tlp), got))
        want = P.logprobs(x, tk.download().view(np.int32)[:T], top)
        assert (got[0] == want[0]).all() and (got[1] == want[1]).all()
        intllm.check("drop", lib.q48_graph_drop(c.h))


def test_captured_over_many_blocks(ctx):
    """The same where a row's blocks meet at a ticket, other calls between the replays."""
    rng = np.random.default_rng(6)
    lib = intllm.hip_lib()
    T, V, top = 3, 40000, 7
    with intllm.Context(0) as c:
        d, tk = c.buffer(T * V), ints(c, rng.integers(0, V, T))
        outs = [c.buffer(n) for n in (T, T, T * top, T * top)]

        def call(rows):
            logp, ent, ids, tlp = (b.ptr for b in outs)
            c.logprobs_rows(d.ptr, rows, V, tk.ptr, logp, ent, top, ids, tlp)

        d.upload(logits(rng, T, V))
        call(T)
        c.sync()
        intllm.check("begin", lib.q48_graph_begin(c.h))
        call(T)
        intllm.check("end", lib.q48_graph_end(c.h))
        for _ in range(4):
            d.upload(logits(rng, T, V))
            intllm.check("launch", lib.q48_graph_launch(c.h, 1))
            got = [b.download() for b in outs]
            call(1)                       # other chunks in the same workspace
            call(T)
            assert all((b.download() == g).all() for b, g in zip(outs, got))
        intllm.check("drop", lib.q48_graph_drop(c.h))


@pytest.mark.parametrize("width", [700, 9000])
def test_differences_at_multiples_of_ln2(ctx, width):
    """u = k LN2 and a word to either side, alone and with whole steps of the table, up to
    where e is 0: the quotient of u by LN2 is settled by a comparison there."""
    us = {max(0, k * P.LN2 + j * (1 << 42) + d) for k in range(51) for j in (0, 1, 22, 44)
          for d in (-1, 0, 1)}
    us = np.array(sorted(us), dtype=np.int64)
    assert us.size <= width
    rng = np.random.default_rng(width)
    x = np.full((4, width), -(60 * P.LN2), dtype=np.int64)
    for t, m in enumerate((0, 5 * P.ONE + 1, -(1 << 60), I64.max)):
        x[t] = m - 60 * P.LN2
        x[t, rng.permutation(width)[:us.size]] = m - us
    check_rows(ctx, x, rng.integers(0, width, 4), 32)
    for t in range(4):                         # each alone beside the largest: Z says what e is
        y = np.full((us.size, 2), x[t].max(), dtype=np.int64)
        y[:, 1] -= us
        check_rows(ctx, y, np.ones(us.size, np.int64), 2)


def test_sizes_out_of_range_are_refused(ctx):
    """Nothing is launched: the buffers are of one row."""
    d, e, ids, lp = ctx.to_device(np.full(64, 3)), ctx.to_device(np.full(2, 5)), *(
        ctx.buffer(64) for _ in range(2))
    big = (1 << 30) + 1
    for T, V, top in ((0, 1, 0), (-1, 1, 0), (big, 1, 0), ((1 << 31) - 1, 1, 0), (1, 0, 0),
                      (1, (1 << 22) + 1, 0), (1, 8, -1), (1, 8, 9), (1, 64, 33)):
        with pytest.raises(intllm.Q48Error) as err:
            ctx.logprobs_rows(d.ptr, T, V, None, None, e.ptr, top, ids.ptr, lp.ptr)
        assert err.value.code == intllm.Q48_EINVAL, (T, V, top)
    assert (e.download() == 5).all()


def test_outputs_over_the_inputs_are_refused(ctx):
    """A row's results are written while other rows are still read."""
    rng = np.random.default_rng(3)
    T, V, top = 600, 300, 2
    x, tokens = logits(rng, T, V), rng.integers(0, V, T)
    d, tk = ctx.to_device(x), ints(ctx, tokens)
    a, b, i, l = (ctx.to_device(np.full(T * top, 5)) for _ in range(4))
    inner = d.at(T * V - 1)
    for logp, ent, ids, tlp in ((d.ptr, b.ptr, i.ptr, l.ptr), (a.ptr, inner, i.ptr, l.ptr),
                                (a.ptr, b.ptr, d.ptr, l.ptr), (a.ptr, b.ptr, i.ptr, d.at(3)),
                                (tk.ptr, b.ptr, i.ptr, l.ptr), (a.ptr, b.ptr, tk.ptr, l.ptr),
                                (d.ptr - 8 * (T - 1), b.ptr, i.ptr, l.ptr)):
        with pytest.raises(intllm.Q48Error) as err:
            ctx.logprobs_rows(d.ptr, T, V, tk.ptr, logp, ent, top, ids, tlp)
        assert err.value.code == intllm.Q48_EINVAL
    assert (d.download() == x.ravel()).all() and (a.download() == 5).all()
    assert (tk.download().view(np.int32)[:T] == tokens).all()


@pytest.mark.parametrize("T,V", [(600, 300), (3, 20000)])
def test_the_most_probable_token_in_place_of_the_scored_one(ctx, T, V):
    rng = np.random.default_rng(V)
    x, tokens = logits(rng, T, V), rng.integers(0, V, T)
    d, tk, apart = ctx.to_device(x), ints(ctx, tokens), ints(ctx, tokens)
    a, b, l, ids = (ctx.buffer(T) for _ in range(4))
    ctx.logprobs_rows(d.ptr, T, V, apart.ptr, b.ptr, None, 1, ids.ptr, l.ptr)
    ctx.logprobs_rows(d.ptr, T, V, tk.ptr, a.ptr, None, 1, tk.ptr, l.ptr)
    assert (tk.download().view(np.int32)[:T] == x.argmax(1)).all()
    assert (a.download() == b.download()).all()
