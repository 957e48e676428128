"""Calls over weights in 8 bits that are refused before anything is enqueued (no GPU
needed: the context's memory is never looked at).
"""
import ctypes as C

import pytest

import intllm

CTX = C.create_string_buffer(4096)      # stands for a context: every call here is refused first
A = 1 << 30                             # addresses that nothing reads
MAX_N, MAX_K, MAX_COUNT, MAX_T = 1 << 24, 1 << 17, 1024, 1 << 20


def w8(codes=A, step=A + (1 << 36), count=1, N=64, K=128):
    return intllm.W8(codes, step, count, N, K)


def call(name, *a):
    a = [C.byref(x) if isinstance(x, C.Structure) else x for x in a]
    return getattr(intllm.hip_lib(), name)(*a)


def refused(name, *a):
    assert call(name, *a) == intllm.Q48_EINVAL, (name, a)


BAD = [dict(codes=None), dict(step=None), dict(codes=A + 8), dict(step=A + 4), dict(count=0),
       dict(count=MAX_COUNT + 1), dict(N=0), dict(N=-1), dict(N=MAX_N + 1), dict(K=0), dict(K=MAX_K + 1)]


@pytest.mark.parametrize("bad", BAD)
def test_descriptions(bad):
    w, Y, X = w8(**bad), 1 << 40, 1 << 41
    refused("q48_w8_pack", CTX, w, 0, X)
    refused("q48_w8_put", CTX, w, 0, X, Y)
    refused("q48_w8_values", CTX, Y, w, 0)
    refused("q48_gemm_w8", CTX, Y, None, w, X, None, 1)
    refused("q48_gemm_w8_swiglu", CTX, Y, w, w8(), X, None, 1)
    refused("q48_gemm_w8_swiglu", CTX, Y, w8(), w, X, None, 1)
    for part in ("gate", "up", "down"):
        m = moe()
        setattr(m, part, w8(**{**dict(count=4), **bad}))
        refused("q48_moe_w8", CTX, Y, None, m, X, None, 1, None, None)


def moe(top=2, router=1 << 42, E=4, dim=128, ffn=64):
    g, u, d = (w8(A + (i << 33), A + (i << 33) + (1 << 32), E, N, K)
               for i, (N, K) in enumerate(((ffn, dim), (ffn, dim), (dim, ffn))))
    return intllm.Moe(router, g, u, d, top, 1)


def test_sizes_of_arrays():
    c, s = C.c_size_t(), C.c_size_t()
    f = intllm.hip_lib().q48_w8_bytes
    assert f(3, 17, 65, C.byref(c), C.byref(s)) == 0
    assert (c.value, s.value) == (3 * 2 * 2 * 1024, 3 * 17 * 8)
    assert f(MAX_COUNT, MAX_N, MAX_K, C.byref(c), C.byref(s)) == 0
    assert c.value == MAX_COUNT * MAX_N * MAX_K
    for a in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (MAX_COUNT + 1, 1, 1), (1, MAX_N + 1, 1), (1, 1, MAX_K + 1)):
        assert f(*a, C.byref(c), C.byref(s)) == intllm.Q48_EINVAL
    assert f(1, 1, 1, None, C.byref(s)) == intllm.Q48_EINVAL
    assert f(1, 1, 1, C.byref(c), None) == intllm.Q48_EINVAL


def test_filling():
    w, X = w8(count=2), 1 << 41
    for name, a in (("q48_w8_pack", (X,)), ("q48_w8_put", (X, X + (1 << 20)))):
        refused(name, None, w, 0, *a)
        refused(name, CTX, None, 0, *a)
        refused(name, CTX, w, -1, *a)
        refused(name, CTX, w, 2, *a)
        for i in range(len(a)):
            refused(name, CTX, w, 0, *a[:i], None, *a[i + 1:])
    refused("q48_w8_pack", CTX, w, 0, X + 4)
    refused("q48_w8_put", CTX, w, 0, X, X + 4)
    refused("q48_w8_pack", CTX, w, 1, w.codes + 64 * 128)          # over what is written
    refused("q48_w8_pack", CTX, w, 0, w.step - 8 * 64 * 128 + 8)
    refused("q48_w8_put", CTX, w, 0, w.codes - 64 * 128 + 1, X)
    refused("q48_w8_put", CTX, w, 1, X, w.step + 8 * 64)
    refused("q48_w8_values", None, X, w, 0)
    refused("q48_w8_values", CTX, None, w, 0)
    refused("q48_w8_values", CTX, X + 4, w, 0)
    refused("q48_w8_values", CTX, X, None, 0)
    for i in (-1, 2):
        refused("q48_w8_values", CTX, X, w, i)
    refused("q48_w8_values", CTX, w.codes - 8, w, 0)
    refused("q48_w8_values", CTX, w.step, w, 0)


def test_products():
    w, Y, X, n, b = w8(), 1 << 40, 1 << 41, 1 << 42, 1 << 43
    up = w8(A + (1 << 32), A + (1 << 33))

    def both(Y, X, n, T, ctx=CTX, w=w):
        refused("q48_gemm_w8", ctx, Y, None, w, X, n, T)
        refused("q48_gemm_w8_swiglu", ctx, Y, w, up, X, n, T)

    both(Y, X, n, 1, ctx=None)
    both(Y, X, n, 1, w=None)
    both(None, X, n, 1)
    both(Y, None, n, 1)
    for T in (0, -1, MAX_T + 1):
        both(Y, X, n, T)
    for off in (1, 4):
        both(Y + off, X, n, 1)
        both(Y, X + off, n, 1)
        both(Y, X, n + off, 1)
    refused("q48_gemm_w8", CTX, Y, b + 4, w, X, n, 1)
    both(X, X, n, 1)                                    # outputs over inputs
    both(X + 8 * 127, X, n, 1)
    both(X - 8 * 63, X, n, 1)
    both(n + 8 * 127, X, n, 1)
    both(w.codes + 8, X, n, 1)
    both(w.step, X, n, 1)
    refused("q48_gemm_w8_swiglu", CTX, up.step, w, up, X, n, 1)
    refused("q48_gemm_w8_swiglu", CTX, up.codes, w, up, X, n, 1)
    refused("q48_gemm_w8", CTX, Y, Y + 8, w, X, n, 1)   # a base that is partly the output
    refused("q48_gemm_w8", CTX, Y, Y - 8 * 63, w, X, n, 1)
    refused("q48_gemm_w8", CTX, Y, None, w8(count=2), X, n, 1)
    refused("q48_gemm_w8_swiglu", CTX, Y, w, None, X, n, 1)
    for other in (w8(N=63), w8(K=127), w8(count=2)):
        refused("q48_gemm_w8_swiglu", CTX, Y, w, other, X, n, 1)


def test_experts():
    Y, X, n, ch, wt = 1 << 40, 1 << 41, 1 << 43, 1 << 44, 1 << 45
    T, dim = 3, 128

    def no(Y=Y, b=None, m=None, X=X, n=n, T=T, ch=ch, wt=wt, ctx=CTX):
        refused("q48_moe_w8", ctx, Y, b, m or moe(), X, n, T, ch, wt)

    no(ctx=None)
    refused("q48_moe_w8", CTX, Y, None, None, X, n, T, ch, wt)
    no(Y=None)
    no(X=None)
    no(m=moe(router=None))
    for t in (0, -1, MAX_T + 1):
        no(T=t)
    for top in (0, -1, 5):
        no(m=moe(top=top))
    no(m=moe(top=65, E=70))
    for part, shape in (("gate", dict(N=65, K=128)), ("up", dict(N=63, K=128)), ("up", dict(N=64, K=127)),
                        ("down", dict(N=129, K=64)), ("down", dict(N=128, K=63))):
        m = moe()
        old = getattr(m, part)
        setattr(m, part, w8(old.codes, old.step, 4, **shape))
        no(m=m)
        setattr(m, part, w8(old.codes, old.step, 3, old.N, old.K))
        no(m=m)
    for off in (1, 4):
        no(Y=Y + off)
        no(b=Y + (1 << 30) + off)
        no(X=X + off)
        no(n=n + off)
        no(wt=wt + off)
        no(m=moe(router=(1 << 42) + off))
    no(ch=ch + 2)
    no(Y=X)                                             # over the rows, which are not the base
    no(Y=X, b=Y)
    no(Y=X + 8 * dim, b=X + 8 * dim)
    no(b=Y + 8)
    m = moe()
    for at in (n + 8 * (dim - 1), m.router, m.gate.codes, m.gate.step, m.up.codes, m.up.step, m.down.codes,
               m.down.step):
        no(Y=at)
        no(ch=at)
        no(wt=at)
    for at in (Y, X):
        no(ch=at)
        no(wt=at)
    no(b=wt)
    no(ch=wt + 8)


class Room:
    """Stands for a buffer of a context."""
    def __init__(self, ptr):
        self.ptr = ptr

    def free(self):
        self.ptr = None


def test_layers_of_weights_that_were_given_back():
    """A layer holds copies of its weights' descriptions: with the weights these are refused
    too, however the layer came by them; other weights' are left alone."""
    ctx = object.__new__(intllm.Context)
    ctx.h, ctx._bufs = C.addressof(CTX), []
    Y, X = 1 << 44, 1 << 45

    def new(i, E, N, K):
        at = A + (i << 33)
        w = ctx.w8(at, at + (1 << 32), E, N, K)
        w.bufs = [Room(w.codes), Room(w.step)]
        ctx._bufs += w.bufs
        return w

    shapes = dict(gate=(4, 64, 128), up=(4, 64, 128), down=(4, 128, 64))
    for part in shapes:
        w = {n: new(i, *s) for i, (n, s) in enumerate(shapes.items())}
        layers = [ctx.moe(1 << 43, *w.values(), 2, True), intllm.Moe(1 << 43, **w, top_k=2, renorm=1),
                  intllm.Moe(router=1 << 43, top_k=2)]
        for n, m in w.items():
            setattr(layers[2], n, m)
        other = ctx.moe(1 << 43, *w.values(), 2, True)
        setattr(other, part, new(5, *shapes[part]))
        kept = getattr(other, part).codes
        ctx.free_w8(w[part])
        for m in layers:
            for n in shapes:
                assert (getattr(m, n).codes is None) == (getattr(m, n).step is None) == (n == part)
            refused("q48_moe_w8", CTX, Y, None, m, X, None, 1, None, None)
            with pytest.raises(intllm.Q48Error) as err:
                ctx.moe_w8(Y, None, m, X, None, 1)
            assert err.value.code == intllm.Q48_EINVAL
        assert getattr(other, part).codes == kept
        refused("q48_w8_values", CTX, Y, w[part], 0)
        ctx.free_w8(w[part])                                # nothing is left to give back
        mine = w8(count=4, N=64, K=128)
        m = ctx.moe(1 << 43, mine, mine, w["down"], 2, True)
        ctx.free_w8(mine)                                   # the caller's memory
        assert mine.codes == m.gate.codes == A
