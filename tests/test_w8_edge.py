"""The FP64 form of a scaled product (w8_scaled_double of csrc/q48_w8.hpp) next to 2^53,
the last whole number that a double holds with all below it: restated with every operation
rounded down as on the device, against integer arithmetic (no GPU).
"""
import math
import random
from fractions import Fraction as F

from test_round_down_identity import fma
from test_w8_identity import UNIT, add, mul

EDGE = 1 << 53


def scaled(S, sa, sw, limit=EDGE - (1 << 32)):
    """The form's result and whether it is sure of it; limit: of the rounded product."""
    sw = F(sw) * UNIT
    p = mul(sa, sw)
    pl = fma(sa, sw, -p)
    h = mul(S, p)
    hl = fma(S, p, -h)
    f = F(math.floor(h))
    t = add(add(h, -f), fma(S, pl, hl))
    g = F(math.floor(t))
    return int(add(f, g)), abs(h) < limit and add(t, -g) < 1 - F(1, 1 << 40)


def edge_products(rng, n):
    """Steps and sums whose product comes within 3 of 2^53, on both sides of 0."""
    out = []
    while len(out) < n:
        S = rng.choice([rng.randrange(1, 1 << 20) | 1, (1 << rng.randrange(1, 21)) - 1,
                        rng.randrange(1, 1 << 31) >> rng.randrange(0, 31) | 1])
        sw = rng.randrange(1, EDGE) >> rng.choice([0, 2, 5, 10, 20])
        want = EDGE + rng.randrange(-3, 4)
        sa = -(-(want << 48) // (S * max(sw, 1)))
        if 0 < sa < EDGE and sw and abs((S * sa * sw >> 48) - EDGE) <= 3:
            out.append((S * rng.choice([1, -1]), sa, sw))
    return out


def edge_rows(rng, codes, sa, n):
    """n weight rows (codes and a step) whose products with a row of these codes and the step
    sa come within 2 of 2^53 in magnitude, and where a limit of 2^53 on the rounded product
    lets a wrong word pass as sure."""
    out = []
    while len(out) < n:
        c = [rng.randrange(-127, 128) for _ in codes]
        S = sum(a * b for a, b in zip(codes, c))
        at = (EDGE << 48) // max(abs(S) * sa, 1)
        for sw in range(at - 2, at + 3):
            if abs(S) * sa >> 47 and 0 < sw < EDGE:
                got, sure = scaled(S, sa, sw, EDGE)
                if sure and got != S * sa * sw >> 48:
                    out.append((c, sw))
                    break
    return out


def test_sure_only_of_what_a_double_holds():
    rng = random.Random(11)
    cases = edge_products(rng, 3000) + [(7, 7772727593286963, 46597012622995)]
    below = 0
    for S, sa, sw in cases:
        got, sure = scaled(S, sa, sw)
        assert not sure or got == S * sa * sw >> 48, (S, sa, sw)
        below += sure
    assert below == 0                       # all of them within 2^32 of the edge: integers
    # the smaller limit is needed: without it some of these pass as sure and are wrong
    assert any(s and g != S * sa * sw >> 48
               for S, sa, sw in cases for g, s in [scaled(S, sa, sw, EDGE)])


def test_what_remainders_add_stays_below_the_limit():
    """The floor of a rounded product and of what the remainders add to it: at most 4 away
    from the rounded product, so a double wherever that is below 2^53 - 2^32."""
    rng = random.Random(12)
    for _ in range(3000):
        S = rng.choice([1, -1]) * (rng.randrange(1, 1 << 31) >> rng.randrange(0, 31) | 1)
        sa = rng.randrange(1, EDGE) >> rng.choice([0, 3, 10, 30])
        top = min(EDGE - 1, (((EDGE - (1 << 33)) << 48) // (abs(S) * max(sa, 1))))
        for sw in (top, max(0, top - 1), top // 3):
            got, sure = scaled(S, max(sa, 1), sw)
            want = S * max(sa, 1) * sw >> 48
            assert abs(want) < EDGE
            assert got == want if sure else S * max(sa, 1) * sw % (1 << 48) > (1 << 48) - (1 << 10)


def test_rows_at_the_edge():
    """What the GPU's cases are made of: such rows exist for either sign."""
    rng = random.Random(5)
    a, sa = [127, -70, 31, 5], 3 * (1 << 37) + 12345
    signs = set()
    for c, sw in edge_rows(rng, a, sa, 6):
        S = sum(x * y for x, y in zip(a, c))
        assert abs(abs(S * sa * sw >> 48) - EDGE) <= 2
        assert not scaled(S, sa, sw)[1]
        signs.add(S > 0)
    assert signs == {True, False}
