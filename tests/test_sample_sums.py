"""How far the sampling's sums are from the real numbers that they stand for, on the CPU: the device's steps restated with
its own constants (csrc/sample.hip), each rounded as there, against 60 decimal digits.  The bound is the one that
include/syntropy_hip.h gives: 2^(11 - b) of the sum, b = min(50, 62 - log2 vocab rounded up).  (vocab 2^-62 of a weight is
none: equal logits are off by more.)"""
import decimal
import os
import random
import re
from fractions import Fraction

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
BINS = 2048
decimal.getcontext().prec = 60
LN2 = decimal.Decimal(2).ln()


def constants(name):
    src = open(os.path.join(HERE, "..", "syntropy_amd", "csrc", "sample.hip")).read()
    body = re.search(name + r"\[\d+\] = \{([^}]*)\}", src).group(1)
    return [float.fromhex(v.strip()) for v in body.split(",")]


STEPS, EXPS = constants("STEPS"), constants("EXPS")


def power(s: float) -> decimal.Decimal:
    """2^(-s / 32)"""
    return (-LN2 * decimal.Decimal(s) / 32).exp()


def exactly(d: decimal.Decimal) -> Fraction:
    return Fraction(d)


def fma(a, b, c) -> float:
    return float(Fraction(a) * Fraction(b) + Fraction(c))


def bits_of(vocab):
    return min(50, 62 - ((vocab - 1) | 1).bit_length())


def part(s: float, bits: int):
    """(bin, whole number) of a distance"""
    n = round(s)  # (half to even, as the device)
    y, one = s - n, float(1 << bits)
    p = fma(y, EXPS[4], EXPS[3])
    for e in (EXPS[2], EXPS[1], EXPS[0]):
        p = fma(p, y, e)
    return n, int(fma(p * one, y, one + 2.0 ** 52) - 2.0 ** 52)


def sums(row, vocab):
    """(the device's sum, the exact one) of a row of {distance: how many}"""
    bits, masses = bits_of(vocab), {}
    exact = Fraction(0)
    for s, n in row.items():
        b, whole = part(s, bits)
        masses[b] = masses.get(b, 0) + n * whole
        exact += n * exactly(power(s))
    got = sum(round(float(m) * STEPS[b & 31] * 2.0 ** -(b >> 5)) for b, m in masses.items())
    assert got < 1 << 63
    return Fraction(got, 1 << bits), exact


def rows(vocab, rng):
    """The greatest value and vocab - 1 more: all alike, at a bin's ends and its middle; in as many bins as there are; spread"""
    for s in (0.0, 0.25, 0.4999, 0.5001, 1.5, 33.49, 320.51, 2040.3):
        yield {0.0: 1, s: vocab - 1} if s else {0.0: vocab}
    bins = min(BINS - 1, vocab - 1)
    each = (vocab - 1) // bins
    for off in (0.0, 0.499, -0.499):
        yield {0.0: 1, **{b + off: each for b in range(1, bins + 1)}}
    yield {0.0: 1, **{rng.uniform(0, BINS - 2): max(1, (vocab - 1) // 3000) for _ in range(min(3000, vocab - 1))}}


def test_the_constants():
    for j, v in enumerate(STEPS):
        assert abs(Fraction(v) - exactly(power(j))) <= Fraction(1, 1 << 53)
    worst = 0.0
    for i in range(-500, 501):
        y = i / 1000
        p = Fraction(1)
        p += sum(Fraction(e) * Fraction(y) ** (n + 1) for n, e in enumerate(EXPS))
        worst = max(worst, abs(float(p / exactly(power(y)) - 1)))
    assert 2.0 ** -49 < worst < 2.0 ** -48  # (the sixth power's share: (ln 2 / 64)^6 / 720)


@pytest.mark.parametrize("vocab", [2, 1000, 50257, 128256, 1 << 20, 1 << 24])
def test_sums(vocab):
    bits, rng, over = bits_of(vocab), random.Random(vocab), 0
    for i, row in enumerate(rows(vocab, rng)):
        got, exact = sums(row, vocab)
        off = abs(got - exact)
        assert off <= Fraction(2) ** (10 - bits) + exact * (Fraction(1, 1 << 48) + Fraction(102, 100) * Fraction(1, 1 << (bits + 1))), i
        assert off <= exact * Fraction(2) ** (11 - bits), i
        over += off > Fraction(vocab, 1 << 62)
    assert over or vocab == 2
