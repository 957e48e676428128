"""The integer definitions of the serving operators, on the CPU: how far the
log-probability steps are from the mathematics, the quantised cache's rounding,
and the refusals of every entry point (a zeroed context: nothing is launched for a
call that is refused).
"""
import ctypes as C
import random
from decimal import Decimal, getcontext

import numpy as np
import pytest

import intllm
import serve_plain as P

EINVAL, ERANGE, ESTATE = intllm.Q48_EINVAL, intllm.Q48_ERANGE, intllm.Q48_ESTATE


def test_exponential_is_near_e_to_the_minus_u():
    """|e_i - 2^48 e^-u| <= 4: the table and six Horner steps round once each (the
    steps' errors shrink by s < 2^-6), the series' end and LN2's half unit times n 2^-n
    stay below one, the last shift floors."""
    getcontext().prec = 60
    rng = random.Random(1)
    for _ in range(3000):
        u = int(rng.choice([rng.uniform(0, 1), rng.uniform(0, 40)]) * P.ONE)
        want = (Decimal(-u) / P.ONE).exp() * P.ONE
        assert abs(P.expn(u) - want) <= 4
    assert P.expn(0) == P.ONE
    assert P.expn(49 * P.LN2) == 0 and P.expn((1 << 64) - 1) == 0


def test_log_is_near_log():
    """|logsum - 2^48 log| <= 20: the reciprocal and its product 2 units, nine
    Horner steps and the table one each, b half units of LN2 (b <= 22 here)."""
    getcontext().prec = 60
    rng = random.Random(2)
    for _ in range(3000):
        z = int(P.ONE * 2 ** rng.uniform(0, 22)) + rng.randrange(3)
        got, b = P.logsum(z)
        assert abs(got - (Decimal(z) / P.ONE).ln() * P.ONE) <= 20 and (z >> b) >> 48 == 1
    assert P.logsum(P.ONE) == (0, 0)


@pytest.mark.parametrize("bits", [8, 4])
def test_quantised_value_is_at_most_half_a_step_off(bits):
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((200, 64)) * P.ONE).astype(np.int64)
    x[:20] = rng.integers(-300, 300, (20, 64))
    x[20] = 0
    x[21, 5] = np.iinfo(np.int64).min
    x[22, 7] = np.iinfo(np.int64).max
    c, st = P.quantise(x, bits)
    v = P.values(c, st)
    assert abs(c).max() <= P.LEVELS[bits]
    off = abs(v.astype(object) - x.astype(object))
    # |x_d| / step passes Q only where the step is cut to 63 bits: a few words more
    assert all(off[i].max() <= st[i] // 2 + (st[i] % 2) + (130 if i in (21, 22) else 0)
               for i in range(200))
    assert (P.unpack(P.pack(c, bits), bits) == c).all()


def fake():
    """A zeroed q48_ctx: enough for a call that is refused by its arguments."""
    return C.create_string_buffer(1 << 16)


def cache(**kw):
    d = dict(k=4096, v=8192, k_step=64, v_step=128, bits=8, layers=2, max_seq=100, n_kv=2,
             head_dim=64)
    d.update(kw)
    return intllm.QCache(*d.values())


BAD_CACHES = [dict(k=None), dict(v=None), dict(k_step=None), dict(v_step=None), dict(k=4104),
              dict(v=8193), dict(k_step=68), dict(bits=6), dict(bits=0), dict(layers=0),
              dict(layers=65536), dict(n_kv=65536),
              dict(max_seq=0), dict(max_seq=32768), dict(n_kv=0), dict(head_dim=48),
              dict(head_dim=256)]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_bad_cache_is_refused(bad):
    lib, c, x = intllm.hip_lib(), fake(), C.byref(cache(**bad))
    assert lib.q48_qcache_store_rows(c, x, 0, 0, 1, 64, 64, 128) == EINVAL
    assert lib.q48_qcache_load_rows(c, 64, 64, x, 0, 0, 1, 128) == EINVAL
    assert lib.q48_rope_store_rows_qcache(c, 64, x, 0, 0, 1, None, 4) == EINVAL
    assert lib.q48_attn_decode_qcache(c, 64, 1 << 20, x, 1 << 21, 1 << 22, 0, 0, 4) == EINVAL
    assert lib.q48_attn_decode_rope_qcache(c, 64, 1 << 20, x, 1 << 21, 1 << 22, 0, 0, 4) == EINVAL
    assert lib.q48_attn_rows_qcache(c, 64, 1 << 20, x, 0, 0, 1, 4, None) == EINVAL
    assert lib.q48_qcache_keep_rows(c, x, 0, 64, 1) == EINVAL


def test_refusals():
    lib, c, q = intllm.hip_lib(), fake(), cache()
    x = C.byref(q)
    far = 1 << 24
    # store and load: layer, rows, stride, pointers
    for a, want in [((2, 0, 1, 64, 64, 128), EINVAL), ((-1, 0, 1, 64, 64, 128), EINVAL),
                    ((0, 0, 0, 64, 64, 128), EINVAL), ((0, 0, 1, None, 64, 128), EINVAL),
                    ((0, 0, 1, 64, None, 128), EINVAL), ((0, 0, 1, 64, 64, 127), EINVAL),
                    ((0, -1, 1, 64, 64, 128), ERANGE), ((0, 100, 1, 64, 64, 128), ERANGE),
                    ((0, 99, 2, 64, 64, 128), ERANGE),
                    ((0, 50, (1 << 31) - 1, 64, 64, 128), ERANGE)]:
        layer, p0, T, K, V, ld = a
        assert lib.q48_qcache_store_rows(c, x, layer, p0, T, K, V, ld) == want, a
        assert lib.q48_qcache_load_rows(c, K, V, x, layer, p0, T, ld) == want, a
        assert lib.q48_qcache_store_rows(None, x, layer, p0, T, K, V, ld) == EINVAL
    # decode
    dec = lib.q48_attn_decode_qcache
    assert dec(c, 64, far, x, far, far, 0, 100, 4) == ERANGE
    assert dec(c, 64, far, x, far, far, 0, -1, 4) == ERANGE
    assert dec(c, 64, far, x, far, far, 2, 0, 4) == EINVAL
    assert dec(c, 64, far, x, far, far, 0, 0, 3) == EINVAL
    assert dec(c, 64, far, x, far, far, 0, 0, 0) == EINVAL
    assert dec(c, 64, far, x, far, far, 0, 0, 1026) == EINVAL
    assert dec(c, far, far, x, 64, 64, 0, 0, 4) == EINVAL          # out over q
    assert dec(c, far, 64, x, far + 8, 64, 0, 0, 4) == EINVAL      # out over k_new
    assert dec(c, far, 64, x, 64, far + 2040, 0, 0, 4) == EINVAL   # out's last word in v_new
    assert lib.q48_attn_decode_rope_qcache(c, 64, far, x, far, far, 0, 0, 4) == ESTATE
    assert lib.q48_rope_store_rows_qcache(c, far, x, 0, 0, 1, None, 4) == ESTATE
    # rows
    rows = lib.q48_attn_rows_qcache
    assert rows(c, 64, far, x, 0, 99, 2, 4, None) == ERANGE
    assert rows(c, 64, far, x, 0, 0, 0, 4, None) == EINVAL
    assert rows(c, 64, far, x, 0, 0, 1, 5, None) == EINVAL
    assert rows(c, 64, far, x, 0, 0, 1, 1026, None) == EINVAL
    assert rows(c, far + 64, far, x, 0, 0, 1, 4, None) == EINVAL
    t = lib.q48_attn_tree
    assert t(c, 64, far, far, far, 0, 0, 1, 4, 2, 48, 100, None) == EINVAL
    assert t(c, 64, far, far, far, 0, 0, 1, 4, 3, 64, 100, None) == EINVAL
    assert t(c, 64, far, far, far, 0, 99, 2, 4, 2, 64, 100, None) == ERANGE
    assert t(c, 64, far, far, far, 0, 32767, 1, 4, 2, 64, 40000, None) == ERANGE
    assert t(c, 64, far, None, far, 0, 0, 1, 4, 2, 64, 100, None) == EINVAL
    assert t(c, far, far, far, far, 0, 0, 1, 4, 2, 64, 100, None) == EINVAL
    at = lib.q48_rope_store_rows_at
    assert at(c, 64, far, far, 0, 0, 1, None, 4, 2, 64, 100) == EINVAL
    assert at(c, 64, far, far, 0, 0, 1, far, 4, 2, 64, 100) == ESTATE
    # keep
    assert lib.q48_qcache_keep_rows(c, x, 0, None, 1) == EINVAL
    assert lib.q48_qcache_keep_rows(c, x, 0, 64, 0) == EINVAL
    assert lib.q48_qcache_keep_rows(c, x, 99, 64, 2) == ERANGE
    assert lib.q48_cache_keep_rows(c, 64, 64, 1, 99, 64, 2, 2, 64, 100) == ERANGE
    assert lib.q48_cache_keep_rows(c, 64, 64, 0, 0, 64, 2, 2, 64, 100) == EINVAL
    # log probabilities
    lp = lib.q48_logprobs_rows
    assert lp(c, 64, 1, 10, None, None, None, 0, None, None) == EINVAL       # nothing asked
    assert lp(c, 64, 1, 10, None, 64, None, 0, None, None) == EINVAL         # logp, no tokens
    assert lp(c, 64, 1, 10, None, None, None, 11, 64, 64) == EINVAL          # top_n > vocab
    assert lp(c, 64, 1, 100, None, None, None, 33, 64, 64) == EINVAL
    assert lp(c, 64, 1, 100, None, None, None, 3, None, 64) == EINVAL
    assert lp(c, 64, 1, 100, None, None, None, -1, 64, 64) == EINVAL
    assert lp(c, 64, 0, 100, None, None, 64, 0, None, None) == EINVAL
    assert lp(c, 64, 1, (1 << 22) + 1, None, None, 64, 0, None, None) == EINVAL
    assert lp(None, 64, 1, 100, None, None, 64, 0, None, None) == EINVAL


def test_cache_sizes():
    assert intllm.qcache_bytes(8, 22, 2048, 4, 64) == (22 * 2048 * 4 * 64, 22 * 2048 * 4 * 8)
    assert intllm.qcache_bytes(4, 1, 3, 1, 128) == (192, 24)
    with pytest.raises(intllm.Q48Error):
        intllm.qcache_bytes(5, 1, 3, 1, 128)
