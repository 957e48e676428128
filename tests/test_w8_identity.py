"""The FP64 forms of csrc/q48_w8.hpp, restated with every operation rounded down as on the
device, against integer arithmetic (no GPU):

1. a scaled product (w8_scaled_double): where it is sure it is the floor, and it is
   sure but for fractions next to 1;
2. SwiGLU (w8_silu_mul): the same, past |g| = 10 too, whatever first
   approximations of the two reciprocals within 2^-20 the hardware gives;
3. a normed word and its code (RowWords).
"""
import math
import random
from fractions import Fraction as F

from test_round_down_identity import ONE, fma, rd, rn

UNIT = F(1, 1 << 48)


def mul(a, b):
    return rd(F(a) * F(b))


def add(a, b):
    return rd(F(a) + F(b))


def scaled(S, sa, sw):
    sw = F(sw) * UNIT
    p = mul(sa, sw)
    pl = fma(sa, sw, -p)
    h = mul(S, p)
    hl = fma(S, p, -h)
    f = F(math.floor(h))
    t = add(add(h, -f), fma(S, pl, hl))
    g = F(math.floor(t))
    sure = abs(h) < 1 << 53 and add(t, -g) < 1 - F(1, 1 << 40)
    return int(add(f, g)), sure


def test_scaled_products():
    rng = random.Random(1)
    unsure = 0
    cases = []
    for _ in range(4000):
        S = rng.randrange(-(1 << 31), 1 << 31) >> rng.choice([0, 4, 8, 20, 31])
        sa = rng.randrange(1 << 53) >> rng.choice([0, 5, 9, 20, 52])
        sw = rng.randrange(1 << 53) >> rng.choice([0, 9, 16, 20, 52])
        cases.append((S, sa, sw))
    for S in (0, 1, -1, (1 << 31) - 1, -(1 << 31), 127 * 127 * 5632):
        for sa in (0, 1, ONE // 127, ONE - 1, ONE, (1 << 53) - 1):
            for sw in (0, 1, ONE // 127, ONE + 1, (1 << 53) - 1):
                cases.append((S, sa, sw))
    for _ in range(1000):   # products a hair below a whole number
        sa, k = rng.randrange(1 << 30, 1 << 44), rng.randrange(1 << 36, 1 << 50)
        S = rng.randrange(1, 1 << 20)
        cases.append((S, sa, min((k << 48) // (S * sa), (1 << 53) - 1)))
    for _ in range(2000):   # up to the last that a double holds
        sa, S = rng.randrange(1 << 40, 1 << 53), rng.choice([-1, 1]) * rng.randrange(1 << 10, 1 << 31)
        sw = (rng.randrange(1 << 50, 1 << 53) << 48) // (abs(S) * sa)
        cases.append((S, sa, min(sw, (1 << 53) - 1)))
    for S, sa, sw in cases:
        want = S * sa * sw >> 48
        got, sure = scaled(S, sa, sw)
        if sure:
            assert got == want, (S, sa, sw)
        elif abs(want) < 1 << 52:
            unsure += 1
            assert S * sa * sw % (1 << 48) > (1 << 48) - (1 << 10), (S, sa, sw)
    assert unsure < 20


def fp_silu(x):
    if abs(x) > 10 * ONE:
        s = ONE if x > 0 else 0
    else:
        r = ONE + (abs(x) >> 14)
        for _ in range(14):
            r = r * r >> 48
        s = (1 << 96) // (ONE + ((1 << 96) // r if x >= 0 else r))
    return x * s >> 48


def rcp(d, rel):
    return rn(F(1) / F(d) * (1 + F(rel)))


def silu_mul(g, u, rel1, rel2):
    ok = True
    p52, m28, r24 = F(1 << 52), F(-(1 << 28)), F(1, 1 << 24)
    h = fma(min(abs(g), 10 * ONE), F(1, 1 << 14), p52 + ONE)
    for _ in range(12):
        y = fma(h, r24, m28)
        h = fma(y, y, p52)
    y = fma(h, r24, m28)
    r = mul(y, y)
    A = F(math.floor(r))
    T = F(math.floor(add(add(r, -A), fma(y, y, -r))))
    A, T = A * r24, T * r24
    r = mul(A, A)
    q = fma(T, T, fma(2 * A, T, fma(A, A, -r)))
    A = F(math.floor(r))
    q = add(add(r, -A), q)
    T = F(math.floor(q))
    ok = ok and add(q, -T) < 1 - F(1, 1 << 30)
    c = F(0) if g > 0 else F(ONE)
    r = add(A, c)
    T = add(T, add(c, -add(r, -A)))
    A = r
    r = rcp(A, rel1)
    y = fma(-A, r, 1)
    r = fma(r, fma(y, y, y), r)
    r = fma(-mul(r, T), r, r)
    low = 16 - UNIT / 2
    q = add(fma(r, ONE, low), -16)
    y = fma(-q, A, ONE)
    h = add(q, UNIT)
    q = h if add(y, -(A * UNIT)) >= mul(h, T) else q
    A = add(q, 1)
    r = rcp(A, rel2)
    y = fma(-A, r, 1)
    r = fma(r, fma(y, y, y), r)
    r = add(add(r, low), -16)
    h = add(r, UNIT)
    r = h if fma(-h, A, 1) >= 0 else r
    r = r if c == 0 else q
    r = F(1) if g > 10 * ONE else F(0) if g < -10 * ONE else r
    out = F(math.floor(mul(math.floor(mul(g, r)), F(u) * UNIT)))
    return int(out), ok and abs(out) < 1 << 53


def test_swiglu():
    rng = random.Random(2)
    rel = lambda: (rng.random() - 0.5) * 2.0 ** -19  # noqa: E731
    gs = [0, 1, -1, 1 << 14, -(1 << 14), ONE, -ONE, 10 * ONE, -10 * ONE, 10 * ONE - 1, 1 - 10 * ONE]
    # around the powers of two that the squares cross
    for e in (48, 49, 50, 51, 52, 53, 54, 55, 56, 60, 62):
        x = int((e - 48) * math.log(2) * ONE)
        gs += [s * min(x + d, 10 * ONE) for s in (1, -1) for d in (-(1 << 20), -1, 0, 1, 1 << 20)]
    gs += [rng.randrange(-10 * ONE, 10 * ONE + 1) >> rng.choice([0, 0, 0, 2, 10, 40]) for _ in range(1200)]
    unsure = 0
    for g in gs:
        u = rng.randrange(-(1 << 52), 1 << 52) >> rng.choice([0, 2, 4, 30])
        got, ok = silu_mul(g, u, rel(), rel())
        want = fp_silu(g) * u >> 48
        if ok:
            assert got == want, (g, u)
        elif abs(want) < (1 << 53) - 1:
            unsure += 1
    assert unsure < 20
    for g in (10 * ONE + 1, -10 * ONE - 1, (1 << 52) - 1, 1 - (1 << 52), 12 * ONE + 5, -15 * ONE):
        for u in (ONE, -ONE, 1, -1, 0, ONE // 3):
            assert silu_mul(g, u, rel(), rel()) == (fp_silu(g) * u >> 48, True), (g, u)


def test_silu_squares_remainders():
    """A quotient's remainder and what it is compared with fit a double for every size of
    the square (the comments' bounds)."""
    rng = random.Random(3)
    for _ in range(2000):
        A = F(rng.randrange(1 << 52, 1 << 53)) * (1 << rng.randrange(0, 11))
        A = A if A < 1 << 63 else A / 2
        ulp = F(1) if A < 1 << 53 else F(1 << (A.numerator.bit_length() - 53))
        T = rng.randrange(0, int(4 * ulp) + 8)
        q = (1 << 96) // int(A + T)
        y = (1 << 96) - q * A                     # exact in FP64
        assert rd(y) == y and rd((q + 1) * T) == (q + 1) * T


LIM = (1 << 53) - (1 << 47)


def normed(x, r, w):
    low = max(0, r.bit_length() - 53)
    rl = r & ((1 << low) - 1)
    rh, rdd = F(r - rl) * UNIT, F(rl) * UNIT
    y = F(math.floor(fma(x, rh, mul(x, rdd))))
    z = F(math.floor(mul(y, F(w) * UNIT)))
    return int(z), max(abs(y), abs(z), abs(w)) < LIM


def test_normed_words():
    rng = random.Random(4)
    n = 0
    for _ in range(6000):
        r = rng.randrange(1 << 62) >> rng.choice([0, 2, 8, 14, 20])
        x = rng.randrange(-(1 << 53) + 1, 1 << 53) >> rng.choice([0, 3, 8, 20, 50])
        w = rng.randrange(-(1 << 53) + 1, 1 << 53) >> rng.choice([0, 3, 5, 30])
        z, fits = normed(x, r, w)
        if fits:
            n += 1
            assert z == (x * r >> 48) * w >> 48, (x, r, w)
    assert n > 3000


def code(z, step, rel):
    rc = rcp(step, rel)
    rc = fma(rc, fma(-step, rc, 1), rc)
    n = abs(z) + (step >> 1)
    q = math.floor(mul(n, rc))
    rem = n - q * step
    assert rd(F(rem)) == rem
    q += -1 if rem < 0 else 1 if rem >= step else 0
    return min(q, 127) * (-1 if z < 0 else 1)


def test_codes():
    rng = random.Random(5)
    for _ in range(4000):
        top = rng.randrange(1, LIM) >> rng.choice([0, 1, 10, 40, 52])
        step = max(1, -(-top // 127))
        k = rng.randrange(0, 128)
        for z in (top, rng.randrange(0, top + 1), min(top, k * step + step // 2),
                  min(top, max(0, k * step - step // 2 - 1))):
            z *= rng.choice([1, -1])
            want = min(127, (abs(z) + (step >> 1)) // step) * (-1 if z < 0 else 1)
            assert code(z, step, (rng.random() - 0.5) * 2.0 ** -19) == want, (z, step)
