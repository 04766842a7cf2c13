"""What the layer operators' numerics rest on, as far as it can be tried without a GPU."""
import numpy as np

F, WIDE = np.float32, np.longdouble


def test_quotients_by_a_reciprocal_fall_on_the_same_side_of_8_bits_middles_as_by_a_division():
    """q = RN(q0 + (u - q0 v) y) with y = RN(1 / v), q0 = RN(u y), for a quotient that is rounded to E4M3 (middles m of five bits).

    With v of 2^23 <= v < 2^24 and 1 <= m < 2: q is the quotient, off by less than 2^-22 of its unit, rounded; so it can differ from RN(u / v) only where u / v is that near to the
    middle between two numbers of 32 bits, and the difference be seen in 8 bits only where m is one of those two: u = v (m +- 2^-24 + d), |d| <= 2^-45.  u is whole and v m a multiple
    of 1/16, so that v 2^-24 is within 2^-21 of a multiple of 1/16: v is within eight of a multiple of 2^20.  All of those are tried, 64 and less on either side, with every u up to 40 from v m."""
    v = np.unique(np.concatenate([np.arange(max(2 ** 23, i * 2 ** 20 - 64), min(2 ** 24, i * 2 ** 20 + 65)) for i in range(8, 17)]))
    differ = []
    for k in range(16, 32):
        for d in range(-40, 41):
            u = v * k // 16 + d
            held = (u < 2 ** 24) | (u % 2 == 0)              # (32 bits have 24 of mantissa)
            a, b = u[held].astype(F), v[held].astype(F)
            y = F(1) / b
            q = a * y
            left = (a.astype(WIDE) - q.astype(WIDE) * b.astype(WIDE)).astype(F)
            q = (q.astype(WIDE) + left.astype(WIDE) * y.astype(WIDE)).astype(F)
            m = F(k / 16)
            wrong = np.sign(q - m) != np.sign(a / b - m)
            differ += [(k, int(i), int(j)) for i, j in zip(a[wrong], b[wrong])]
    # the one that is left to division: every bit of v's mantissa is set
    assert differ == [(16, 2 ** 24, 2 ** 24 - 1)]
