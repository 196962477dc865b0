"""Angles of the rotary operator from exact fractions."""
import math
from fractions import Fraction

# pi to 70 digits: 1 / (2 pi) times a frequency of up to 2^20 is right to 2^-200
PI = Fraction(31415926535897932384626433832795028841971693993751058209749445923078164, 10 ** 70)


def turns(freq):
    """freq radians as a fraction of a turn."""
    return Fraction(freq) / (2 * PI)


def off(freq, fixed):
    """How far the 64-bit fraction `fixed` is from freq, in 2^-64 turns."""
    e = (turns(freq) * 2 ** 64 - fixed) % 2 ** 64
    return float(min(e, 2 ** 64 - e))


def cos_sin(pos, freq):
    """cos and sin of pos * freq, right to 64 bits: the fraction of a turn is
    brought to [-1/2, 1/2] before it becomes a float."""
    t = (turns(freq) * int(pos)) % 1
    a = 2 * math.pi * float(t - 1 if t > Fraction(1, 2) else t)
    return math.cos(a), math.sin(a)
