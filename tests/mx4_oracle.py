"""Microscaled 4-bit rows, the choice of experts and the experts' blocks from their
definitions, in 64 bits (TEST INFRASTRUCTURE ONLY)."""
import math

import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
CODES = np.concatenate([LEVELS, -LEVELS])


def quantise(x):
    """(codes [n, cols], scale bytes [n, cols / 32]) of rows of floats."""
    x = np.asarray(x, np.float64)
    g = x.reshape(len(x), -1, 32)
    top = np.abs(g).max(-1)
    bad = ~np.isfinite(top)
    power = np.frexp(np.where(bad | (top == 0), 1.0, top))[1] - 3
    power = np.where(top == 0, -127, np.maximum(power, -127))
    m = np.abs(np.where(np.isfinite(g), g, 0.0)) / np.ldexp(1.0, power)[..., None]
    low = np.clip(np.searchsorted(LEVELS, m, side="right") - 1, 0, 6)
    under, over = m - LEVELS[low], LEVELS[low + 1] - m
    code = np.where((under > over) | ((under == over) & (low % 2 == 1)), low + 1, low)
    code = np.where(m >= 6.0, 7, code) + 8 * np.signbit(g)
    code = np.where(bad[..., None], 0, code)
    return code.reshape(x.shape).astype(np.uint8), np.where(bad, 255, power + 127).astype(np.uint8)


def pack(code):
    return np.ascontiguousarray(code[:, 0::2] | (code[:, 1::2] << 4)).astype(np.uint8)


def unpack(packed):
    return np.stack([packed & 15, packed >> 4], -1).reshape(len(packed), -1)


def values(packed, scale):
    """What rows of codes two a byte and scale bytes stand for."""
    step = np.where(scale == 255, np.nan, np.ldexp(1.0, scale.astype(np.int64) - 127))
    return CODES[unpack(packed)] * np.repeat(step, 32, 1)


def bf16(x):
    """The nearest bf16 numbers, as float32."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16 << 16).astype(np.uint32)
    return np.where(np.isnan(x), np.float32(np.nan), r.view(np.float32))


def bf16_bits(x):
    """The bits of bf16 numbers given as float32."""
    return (np.ascontiguousarray(x, np.float32).view(np.uint32) >> 16).astype(np.uint16)


def bits_float(b):
    return (b.astype(np.uint32) << 16).view(np.float32)


def gelu(x):
    return 0.5 * x * (1 + np.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))


def silu(x):
    return x / (1 + np.exp(-np.clip(x, -700, 700)))


def route(logits, rule, bias=None, gain=None):
    """(picks, weights) of rows of logits by an igl_route-like rule, one lane and one expert at a time."""
    lanes, count = logits.shape
    picks = np.full((lanes, rule["top"]), -1, np.int32)
    weights = np.zeros((lanes, rule["top"]))
    groups = rule.get("groups", 1)
    each = count // groups
    for m in range(lanes):
        x = logits[m].astype(np.float64)
        x = np.where(np.isnan(x), -np.inf, np.minimum(x, 3.4028234663852886e38))
        with np.errstate(invalid="ignore", over="ignore"):
            if rule["score"] == "softmax":
                s = np.where(x == -np.inf, 0.0, np.exp(x - x.max())) if np.isfinite(x.max()) else np.zeros(count)
                s = s / s.sum() if s.sum() > 0 else s
            else:
                s = np.where(x == -np.inf, 0.0, 1 / (1 + np.exp(-x)))
        c = s + (bias.astype(np.float64) if bias is not None else 0.0)
        if bias is None and groups == 1:
            c = x.copy()
        c[(x == -np.inf) | np.isnan(c)] = -np.inf
        if groups > 1:
            score = []
            for k in range(groups):
                best = sorted((v for v in c[k * each:(k + 1) * each] if v > -np.inf), reverse=True)
                score.append(sum(best[:rule.get("best", 1)]) if best else -np.inf)
            order = sorted(range(groups), key=lambda k: (-score[k], k))
            for k in range(groups):
                if k not in order[:rule["kept"]]:
                    c[k * each:(k + 1) * each] = -np.inf
        order = sorted((e for e in range(count) if c[e] > -np.inf), key=lambda e: (-c[e], e))[:rule["top"]]
        total = sum(s[e] for e in order)
        for j, e in enumerate(order):
            w = s[e]
            if rule.get("renorm", 1):
                w = w / total if total > 0 else 0.0
            picks[m, j] = e
            weights[m, j] = w * rule.get("scale", 1.0) * (float(gain[e]) if gain is not None else 1.0)
    return picks, weights


def experts(x, gate_up, down, pick, weight, inner, gate=gelu):
    """(out, h of every slot, reach of every output: the sum of the magnitudes that make it up)."""
    hidden = x.shape[1]
    out = np.zeros(x.shape)
    reach = np.zeros(x.shape)
    count = len(down) // hidden
    for m in range(len(x)):
        for j, e in enumerate(pick[m]):
            if not 0 <= e < count:
                continue
            w = gate_up[e * 2 * inner:(e + 1) * 2 * inner]
            both = w @ x[m]
            size = np.abs(w) @ np.abs(x[m])
            g, u = both[:inner], both[inner:]
            h = gate(g) * u
            # |gate'| is at most 1.13 and |gate(g)| at most |g|
            spread = 1.13 * size[:inner] * np.abs(u) + np.abs(g) * size[inner:] + np.abs(h)
            d = down[e * hidden:(e + 1) * hidden]
            out[m] += float(weight[m, j]) * (d @ h)
            reach[m] += abs(float(weight[m, j])) * (np.abs(d) @ spread)
    return out, reach
