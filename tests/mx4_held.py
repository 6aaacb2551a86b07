"""Inputs and bars of the tests that every value is held: sheets with one code a row, so that an output is one
value passed through (TEST INFRASTRUCTURE ONLY)."""
import numpy as np

import mx4_oracle as mx

# what five terms leave of a group: half the widest step of the last, of a scale that the largest passes 1.875 of
HELD = 2.0 ** -23 / 1.875


def passing(at, cols):
    """Packed codes and scales of rows that pass column at[n] through."""
    code = np.zeros((len(at), cols), np.uint8)
    code[np.arange(len(at)), at] = 2  # the level 1
    return mx.pack(code), np.full((len(at), cols // 32), 127, np.uint8)


def top_of(x):
    """Of every value the largest of its 32."""
    return np.repeat(np.abs(x).reshape(len(x), -1, 32).max(-1), 32, 1)


def hidden_case(lanes, width, gate):
    """(lanes, columns of gate rows, of up rows, hidden values): lanes of a few binades, which are held
    exactly however a group of them is cut, and hidden values of many."""
    rng = np.random.default_rng(lanes + width)
    x = mx.bf16(rng.uniform(0.25, 3.9, size=(lanes, width)) * rng.choice([-1, 1], size=(lanes, width)))
    a, b = rng.permutation(width), rng.permutation(width)
    g = x.astype(np.float64)
    return x, a, b, gate(g[:, a]) * g[:, b]


def hidden_bar(h):
    """The gate's argument is off by four roundings, 11 at most, its exponential and quotient by sixteen more,
    2^-18 together; then a group is held, and five terms are added."""
    return 1.1 * 2.0 ** -18 * np.abs(h) + HELD * top_of(h)
