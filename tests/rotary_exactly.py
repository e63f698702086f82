"""Angles of rotary positions from whole numbers: the double frequency as it is, 2 pi to 60 digits, no rounding before the last."""
import math
from fractions import Fraction

TWO_PI = 2 * Fraction(314159265358979323846264338327950288419716939937510582097494, 10 ** 59)


def turns(position, frequency):
    """position frequency / 2 pi less the next whole number, a Fraction from -1/2 to 1/2."""
    t = position * Fraction(frequency) / TWO_PI
    return t - round(t)


def angle_bound(position, angle):
    """Turns that the angle (radians, -pi to pi) may be off: a table's entry by 2^-64 turns a position, the cut to 32 bits by half of 2^-32, and
    float32's rounding of what is left, half of its steps relative to the angle."""
    return abs(position) * 2.0 ** -64 + 2.0 ** -33 + 2.0 ** -24 * abs(angle) / (2 * math.pi)
