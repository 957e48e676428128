"""Products with weights in 8 bits whose words lie next to 2^53, where the FP64 form of a
scaled product ends, in every kernel that has it: word for word against integers.
"""
import random

import numpy as np
import pytest

import w8_plain as W
from test_gpu_w8 import loaded, own, words  # noqa: F401
from test_w8_edge import edge_rows

pytestmark = pytest.mark.gpu
A, SA = [127, -70, 31, 5], 3 * (1 << 37) + 12345
DISTINCT = 16


@pytest.fixture(scope="module")
def rows():
    """Weight rows at the edge for the row of codes A and the step SA."""
    r = edge_rows(random.Random(21), A, SA, DISTINCT)
    return np.array([c for c, _ in r], np.int8), np.array([s for _, s in r])


def wide(a, K):
    """The columns of a, and zeros up to K."""
    return np.concatenate([a, np.zeros((*a.shape[:-1], K - a.shape[-1]), a.dtype)], -1)


@pytest.mark.parametrize("T,copies,K", [(1, 1, 4), (1, 1, 8200), (3, 1, 4), (40, 1, 700), (2048, 80, 4),
                                        (2048, 64, 600), (4096, 64, 600)])
def test_products(own, rows, T, copies, K):  # noqa: F811
    """A row alone, few rows, and many in tiles by one and by two groups of waves."""
    codes, steps = np.tile(wide(rows[0], K), (copies, 1)), np.tile(rows[1], copies)
    x = wide(np.array(A) * SA, K)
    want = W.wrap(W.times(np.array([A]), np.array([SA]), *rows))
    assert (abs(abs(want) - (1 << 53)) <= 2).all()
    y = own.buffer(T * codes.shape[0])
    own.gemm_w8(y.ptr, None, loaded(own, codes, steps), own.to_device(np.tile(x, (T, 1))).ptr, None, T)
    assert (y.download().reshape(T, copies, DISTINCT) == want).all()


@pytest.mark.parametrize("T,copies", [(1, 1), (3, 1), (4096, 64)])
def test_swiglu(own, rows, T, copies):  # noqa: F811
    """Up projections at the edge, gates of 1: a unit more or less of a negative one shows in
    the result."""
    ones = np.zeros_like(rows[0])
    ones[:, 0] = 127
    one_steps = np.full(DISTINCT, (1 << 96) // (127 * 127 * SA))
    g = W.wrap(W.times(np.array([A]), np.array([SA]), ones, one_steps))
    u = W.wrap(W.times(np.array([A]), np.array([SA]), *rows))
    want = W.silu_mul(g, u)
    assert (abs(want) < 1 << 53).all() and (want != W.silu_mul(g, u - 1)).any()
    gate = loaded(own, np.tile(ones, (copies, 1)), np.tile(one_steps, copies))
    up = loaded(own, np.tile(rows[0], (copies, 1)), np.tile(rows[1], copies))
    out = own.buffer(T * copies * DISTINCT)
    x = np.tile(np.array(A) * SA, (T, 1))
    own.gemm_w8_swiglu(out.ptr, gate, up, own.to_device(x).ptr, None, T)
    assert (out.download().reshape(T, copies, DISTINCT) == want).all()


@pytest.mark.parametrize("T,dim", [(1, 16), (3, 16), (4096, 1024)])
def test_experts(own, T, dim):  # noqa: F811
    """The down projection of an expert at the edge: a token alone, few, and many."""
    rng = np.random.default_rng(dim)
    ffn = 16
    x = words(rng, 1, dim)
    gate, up = ((rng.integers(-127, 128, (1, ffn, dim)).astype(np.int8),
                 np.full((1, ffn), W.ONE // 127 // max(16, dim // 8))) for _ in range(2))
    c, s = W.quantise(W.swiglu(x, None, (gate[0][0], gate[1][0]), (up[0][0], up[1][0])))
    r = edge_rows(random.Random(dim), c[0].tolist(), int(s[0]), DISTINCT)
    down = (np.array([a for a, _ in r], np.int8), np.array([b for _, b in r]))
    want = np.tile(W.wrap(W.times(c, s, *down))[0], dim // DISTINCT)
    assert (abs(abs(want) - (1 << 53)) <= 2).all()
    copies = dim // DISTINCT
    m = own.moe(own.to_device(words(rng, 1, dim)).ptr, loaded(own, *gate), loaded(own, *up),
                loaded(own, np.tile(down[0], (copies, 1))[None], np.tile(down[1], copies)[None]), 1, True)
    out = own.buffer(T * dim)
    own.moe_w8(out.ptr, None, m, own.to_device(np.tile(x, (T, 1))).ptr, None, T)
    assert (out.download().reshape(T, dim) == want).all()
