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


# A product's forms (planmx_form: 0 few, 1 head, 2 tiles of few lanes, 3 and 4 of many, 5 of a tall sheet; a token's
# step has none of its own): (lanes, rows, cols, form of fp32 lanes, of bf16 ones, of microscaled ones)
STEP, FEW, HEAD, SMALL, LARGE, WHOLE, TALL = -1, 0, 1, 2, 3, 4, 5
FORMS = [(1, 416, 416, STEP, STEP, FEW), (3, 1000, 96, STEP, STEP, FEW), (5, 300, 416, FEW, FEW, FEW), (40, 416, 416, FEW, FEW, FEW),
         (150, 70, 1056, FEW, FEW, FEW), (5, 32776, 1760, HEAD, HEAD, FEW), (3, 32776, 1760, HEAD, HEAD, FEW),
         (16, 32776, 1760, TALL, TALL, FEW), (70, 2400, 4128, SMALL, SMALL, SMALL), (21, 4100, 4128, SMALL, SMALL, FEW),
         (300, 1537, 544, SMALL, SMALL, FEW), (513, 4100, 288, SMALL, SMALL, SMALL), (500, 6150, 416, SMALL, LARGE, SMALL),
         (1540, 7690, 160, LARGE, WHOLE, LARGE), (2050, 8190, 416, LARGE, WHOLE, LARGE)]

# of rows that lie apart (bytes; None: as far as reaches past 4 GiB)
FAR = [(5, 32776, 1760, HEAD, HEAD, FEW), (16, 32776, 1760, TALL, TALL, FEW), (70, 2400, 4128, SMALL, SMALL, SMALL),
       (300, 1537, 544, SMALL, SMALL, FEW), (500, 6150, 416, SMALL, LARGE, SMALL), (1540, 7690, 160, LARGE, WHOLE, LARGE),
       (21, 272, 3232, SMALL, SMALL, FEW), (3, 272, 3232, STEP, STEP, FEW)]
STRIDES = [None] * 6 + [1 << 24] * 2

# Experts' blocks that pass values through: (lanes, hidden, inner), and the places of their tiles (0: a token's step)
BLOCKS = [(1, 512, 512, 0), (5, 96, 96, 0), (40, 512, 512, 16), (600, 2048, 2048, 32), (1200, 2048, 2048, 64)]
UPS = [(1, 512, 256, 0), (5, 64, 32, 0), (40, 512, 256, 16), (600, 4096, 2048, 32), (1200, 4096, 2048, 64)]
# of many slots: (experts, hidden, inner, choices, lanes, places for fp32 lanes, for bf16 ones)
SLOTS = [(6, 64, 32, 6, 520, 16, 16), (16, 64, 32, 8, 2048, 64, 64), (16, 32, 32, 8, 2049, 64, 64), (16, 64, 32, 8, 4096, 64, 64),
         (130, 32, 64, 5, 3300, 32, 64), (4, 32, 32, 1, 20000, 64, 64), (3, 96, 2080, 2, 2500, 64, 64),
         (40, 32, 1056, 4, 1500, 32, 64), (200, 32, 32, 64, 1100, 64, 64)]
# of many choices
CHOICES = [(64, 160, 96, 9, 1, 0, 0), (90, 320, 64, 64, 1, 0, 0), (128, 96, 160, 16, 4, 0, 0), (40, 64, 224, 17, 2, 0, 0),
           (40, 64, 96, 20, 37, 16, 16), (70, 96, 32, 64, 50, 16, 16)]


def wide_lanes(lanes, cols, bf16, spread=3.0):
    """Lanes whose groups span many binades."""
    rng = np.random.default_rng(lanes + cols)
    x = (rng.normal(size=(lanes, cols)) * np.exp(spread * rng.normal(size=(lanes, cols)))).astype(np.float32)
    return mx.bf16(x) if bf16 else x


def value_bar(x, bf16):
    """Of a value passed through: five terms and their adds; bf16's digits are held exactly down to 2^-16 of the
    largest, where the last term's step is theirs."""
    a, top = np.abs(x.astype(np.float64)), top_of(x.astype(np.float64))
    return np.where(a >= 2.0 ** -16 * top, 0.0, HELD * top) if bf16 else HELD * top + 5 * 2.0 ** -24 * 1.1 * a


def outlier_lanes(lanes, cols, bf16, times):
    """(lanes of normals in which a channel of every 32 is `times` the others, those channels)."""
    rng = np.random.default_rng(lanes * 3 + cols)
    x, loud = rng.normal(size=(lanes, cols)), np.arange(cols // 32) * 32 + rng.integers(0, 32, size=cols // 32)
    x[:, loud] *= times
    x = x.astype(np.float32)
    return (mx.bf16(x) if bf16 else x), loud


def up_case(lanes, width, bf16):
    """(lanes, columns of gate rows, of up rows, up's values, what multiplies them): the gate reads lanes of a few
    binades, up reads lanes of many."""
    rng = np.random.default_rng(lanes + width)
    x, half = wide_lanes(lanes, width, bf16), width // 2
    x[:, :half] = mx.bf16(rng.uniform(1, 1.9, size=(lanes, half)))
    return x, rng.permutation(half), half + rng.permutation(half)


def up_bar(x, a, b, bf16, gate):
    """gate(x_a) times what passes through up, then as a hidden value."""
    g = gate(x.astype(np.float64))[:, a]
    h = g * x.astype(np.float64)[:, b]
    return 1.01 * g * value_bar(x, bf16)[:, b] + hidden_bar(h)
