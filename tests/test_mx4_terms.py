"""The arithmetic of microscaled rows on the CPU: lanes of floats as terms of a
narrower form, with mistakes planted in the model, and the oracle of the GPU
tests against plainer words."""
import numpy as np
import pytest

import mx4_oracle as mx

# e2m3: a sign, two bits of exponent, three of mantissa
E2M3 = np.array([m / 8 for m in range(8)] + [(1 + m / 8) * 2 ** e for e in range(3) for m in range(8)])


def e2m3(x):
    """The nearest level, ties to the even code, 7.5 at most."""
    a = np.minimum(np.abs(x), 7.5)
    low = np.clip(np.searchsorted(E2M3, a, side="right") - 1, 0, len(E2M3) - 2)
    under, over = a - E2M3[low], E2M3[low + 1] - a
    at = np.where((under > over) | ((under == over) & (low % 2 == 1)), low + 1, low)
    return np.copysign(E2M3[at], x)


def cut(x, terms, bits=5, most=3.75, least=20):
    """(what the terms of groups add up to, their first scale byte): a scale that takes the largest below `most`, a
    term the nearest level of what is left, each 2^bits finer."""
    top = np.abs(x).max(-1, keepdims=True)
    s = np.maximum(np.ceil(np.log2(np.maximum(top, 2.0 ** -149) / most)) + 127, least)
    step = 2.0 ** (s - 127)
    left, total = x / step, np.zeros_like(x)
    for t in range(terms):
        term = e2m3(left)
        total += term * 2.0 ** (-bits * t)
        left = (left - term) * 2.0 ** bits
    return total * step, s


def groups(kind):
    rng = np.random.default_rng(7)
    x = rng.normal(size=(3000, 32)) * np.exp(rng.normal(size=(3000, 1)) * rng.choice([0.1, 3, 20], size=(3000, 1)))
    x[:500] *= np.exp(3 * rng.normal(size=(500, 32)))
    x[500:1000] = rng.uniform(1.8750001, 3.75, size=(500, 32)) * rng.choice([-1, 1], size=(500, 32))
    x[1000:1100, 0] = 1.8751
    x[1100:1200, 0] = 3.75
    x = x.astype(np.float32)
    return (mx.bf16(x) if kind == "bf16" else x).astype(np.float64)


FORMS = [("f32", 5, -23), ("bf16", 3, -13)]


@pytest.mark.parametrize("kind,terms,power", FORMS)
def test_terms_hold_a_group(kind, terms, power):
    x = groups(kind)
    got, s = cut(x, terms)
    top = np.abs(x).max(-1, keepdims=True)
    assert (top > 1.875 * 2.0 ** (s - 127))[s > 20].all()
    assert (np.abs(got - x) <= 2.0 ** power / 1.875 * top)[np.broadcast_to(s > 20, x.shape)].all()
    assert (s - 5 * (terms - 1) >= 0).all()  # the last term's scale is a byte
    # and groups of nothing but small numbers, by their scale's floor
    small = x * 2.0 ** -138 / top
    got, s = cut(small, terms)
    assert (s == 20).all() and (np.abs(got - small) <= 2.0 ** (20 - 127 - 5 * (terms - 1) - 3)).all()


@pytest.mark.parametrize("kind,terms,power", FORMS)
@pytest.mark.parametrize("mistake", [dict(terms=-1), dict(most=7.5), dict(bits=6), dict(bits=4)])
def test_a_planted_mistake_is_seen(kind, terms, power, mistake):
    """A term less, a largest value up to 7.5 (what is left of it passes 7.5 when widened), a step too wide or too
    narrow for what a term leaves."""
    x = groups(kind)
    extra = dict(mistake)
    got, _ = cut(x, terms + extra.pop("terms", 0), **extra)
    assert (np.abs(got - x) > 2.0 ** power / 1.875 * np.abs(x).max(-1, keepdims=True)).any()


def test_levels_and_scales_of_the_oracle():
    """quantise against trying every code."""
    rng = np.random.default_rng(1)
    x = (rng.normal(size=(40, 64)) * np.exp(4 * rng.normal(size=(40, 1)))).astype(np.float32)
    x[0], x[1, :32] = 0, 2.5
    code, scale = mx.quantise(x)
    for m in range(len(x)):
        for g in range(2):
            v = x[m, 32 * g:32 * g + 32].astype(np.float64)
            top = np.abs(v).max()
            power = -127 if top == 0 else int(np.floor(np.log2(top))) - 2
            assert scale[m, g] == power + 127
            for i, value in enumerate(v / 2.0 ** power):
                far = np.abs(mx.CODES[:8] - min(abs(value), 6.0))
                best = [c for c in range(8) if far[c] == far.min()]
                assert code[m, 32 * g + i] == (best[0] if len(best) == 1 or best[0] % 2 == 0 else best[1]) + 8 * np.signbit(value)
    assert np.array_equal(mx.unpack(mx.pack(code)), code)


def test_the_choice_of_the_oracle():
    rng = np.random.default_rng(2)
    x = rng.normal(size=(50, 24)).astype(np.float32)
    pick, weight = mx.route(x, {"top": 5, "score": "softmax"})
    assert np.array_equal(pick, np.argsort(-x, 1)[:, :5])
    e = np.exp(np.take_along_axis(x, pick, 1).astype(np.float64))
    assert np.allclose(weight, e / e.sum(1, keepdims=True), rtol=1e-12, atol=0)
    bias = rng.normal(size=24).astype(np.float32)
    pick, weight = mx.route(x, {"top": 3, "score": "sigmoid", "groups": 6, "kept": 2, "best": 2, "renorm": 0}, bias)
    s = 1 / (1 + np.exp(-x.astype(np.float64)))
    c = (s + bias).reshape(50, 6, 4)
    score = np.sort(c, 2)[:, :, 2:].sum(2)
    kept = np.argsort(-score, 1)[:, :2]
    assert all(p // 4 in kept[m] for m in range(50) for p in pick[m])
    assert np.array_equal(weight, np.take_along_axis(s, pick, 1))
    best = np.where((np.arange(6)[None, :, None] == kept[:, None, :]).any(2)[:, :, None], c, -9).reshape(50, 24)
    assert np.array_equal(pick, np.argsort(-best, 1)[:, :3])


def test_the_blocks_of_the_oracle():
    rng = np.random.default_rng(3)
    gate_up, down = rng.normal(size=(3 * 2 * 8, 6)), rng.normal(size=(3 * 6, 8))
    x, pick, weight = rng.normal(size=(4, 6)), np.array([[0, 2], [1, 1], [-1, 5], [2, -1]]), rng.normal(size=(4, 2))
    for gate in (mx.gelu, mx.silu):
        got, reach = mx.experts(x, gate_up, down, pick, weight, 8, gate)
        want = np.zeros_like(got)
        for m in range(4):
            for j in range(2):
                e = pick[m, j]
                if 0 <= e < 3:
                    both = gate_up[16 * e:16 * e + 16] @ x[m]
                    want[m] += weight[m, j] * (down[6 * e:6 * e + 6] @ (gate(both[:8]) * both[8:]))
        assert np.allclose(got, want, rtol=1e-12, atol=1e-12) and (np.abs(got) <= reach + 1e-12).all()
        assert (got[2] == 0).all()
