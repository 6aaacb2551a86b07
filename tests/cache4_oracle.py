"""The 4-bit key/value ring in 64 bits, from its definition (numpy): what a row
is stored as, what codes and gains stand for, and attention over a ring.

Every 32 values of a head share a gain, an e4m3 byte; a code stands for level *
gain * scale.  Written rows: the e4m3 value nearest amax / (top scale), 448 at
most, and the level nearest value / (gain scale), ties to even; NaN is zero.
"""
import numpy as np

GROUP = 32
INT4, E2M1 = 0, 1
TOP = {INT4: 7, E2M1: 6}
HALF = {INT4: np.arange(8.0), E2M1: np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])}
LEVELS = {INT4: np.arange(16.0) - 8, E2M1: np.concatenate([HALF[E2M1], -HALF[E2M1]])}
# real8 of every byte: 0x7F is 480 as the byte ring reads it
_MAG = np.array([m / 512 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)])
REAL8 = np.concatenate([_MAG, -_MAG])


def nearest(x, table):
    """Index of the entry of an ascending table nearest x >= 0; halfway, the even index."""
    low = np.clip(np.searchsorted(table, x, side="right"), 1, len(table) - 1) - 1
    under, over = x - table[low], table[low + 1] - x
    return np.where((under > over) | ((under == over) & (low % 2 == 1)), low + 1, low)


def quantise(rows, fmt, scale):
    """(codes, gains) of float32 rows [n, width]: one code a value, one e4m3 byte a group."""
    x = np.asarray(rows, np.float32).astype(np.float64).reshape(len(rows), -1, GROUP)
    s = float(np.float32(scale))
    x = np.where(np.isnan(x), 0.0, x)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        gain = nearest(np.minimum(np.abs(x).max(-1) / (TOP[fmt] * s), 1e9), _MAG[:127])
        step = (_MAG[gain] * s)[..., None]
        level = nearest(np.where(step > 0, np.minimum(np.abs(x) / np.where(step > 0, step, 1), 1e9), 0), HALF[fmt])
    if fmt == INT4:
        code = np.where(x < 0, 8 - level, 8 + level)
    else:
        code = level + 8 * ((x < 0) & (level > 0))
    return code.astype(np.uint8).reshape(len(rows), -1), gain.astype(np.uint8)


def values(codes, gains, fmt, scale):
    """What codes [n, width] and gain bytes [n, width / 32] stand for."""
    v = LEVELS[fmt][codes].reshape(len(codes), -1, GROUP) * (REAL8[gains] * float(np.float32(scale)))[..., None]
    return v.reshape(len(codes), -1)


def pack(codes):
    return codes[:, 0::2] | (codes[:, 1::2] << 4)


def unpack(packed):
    return np.stack([packed & 15, packed >> 4], -1).reshape(len(packed), -1)


def slot(place, sinks, span):
    place = np.asarray(place)
    return np.where(place < sinks, place, sinks + (place - sinks) % (span - sinks))


def seen(pos, window, sinks):
    """The positions a lane at `pos` sees."""
    t = np.arange(pos + 1)
    return t if window == 0 else t[(t > pos - window) | (t < sinks)]


def attend(rows, share, head, query, place, window, sinks, score_scale):
    """Attention of lanes query [n, kv * share * head] at place .. place + n - 1.
    rows(side, places) gives a side's rows of positions in 64 bits.  Also the
    largest sum of |q k| score_scale, which bounds the scores' rounding."""
    n, kv = len(query), query.shape[1] // (share * head)
    q = query.astype(np.float64).reshape(n, kv, share, head)
    out = np.empty_like(q)
    reach, top = 0.0, 0.0
    for i in range(n):
        t = seen(place + i, window, sinks)
        k, v = rows(0, t).reshape(len(t), kv, head), rows(1, t).reshape(len(t), kv, head)
        for j in range(kv):
            s = q[i, j] @ k[:, j].T * score_scale
            reach = max(reach, float((np.abs(q[i, j]) @ np.abs(k[:, j]).T).max()) * abs(score_scale))
            w = np.exp(s - s.max(-1, keepdims=True))
            out[i, j] = w @ v[:, j] / w.sum(-1, keepdims=True)
        top = max(top, float(np.abs(v).max()))
    return out.reshape(n, -1), reach, top
