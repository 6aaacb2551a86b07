"""GPU parity of the 4-bit key/value ring: what is laid, what is read back, and
attention over it, against the ring's definition in 64 bits (cache4_oracle).

Codes and gains are whole numbers decided exactly: every byte of the ring has
to be equal, and the bytes of other slots and of the gain rows' padding
untouched.  A read value is one rounding of level * gain * scale: equal to the
bit.

Bar of attention, from the arithmetic: with reach = max sum |q k| score_scale
and vmax the largest value, queries and probabilities in two binary16 terms are
off by 2^-22 of themselves, a score's fp32 sums, scaling and exponent by fewer
than 2^-20 reach more, so a weight by 2^-19 reach, a blend by twice that times
vmax (weights and their sum); the blocks' sums add at most half a unit, 2^-24,
for each of 64 + blocks steps.
"""
import ctypes

import numpy as np
import pytest

import cache4_oracle as c4
from igllm_amd import native

pytestmark = pytest.mark.gpu

SCALE = 6.0 / 448.0


class At:
    """A device address inside a buffer."""

    def __init__(self, buf, offset):
        self.ptr = buf.ptr + offset


def room(span):
    return (span + 63) // 64 * 64


def ring_bytes(rng, span, width, fmt):
    """A ring's four buffers, every slot filled: codes of unit-variance rows, gains among e4m3's middle."""
    out = []
    for _ in range(2):
        out.append(rng.integers(0, 256, size=(span, width // 2), dtype=np.uint8))
        out.append(rng.integers(0x28, 0x50, size=(width // 32, room(span)), dtype=np.uint8))  # 1/16 .. 2
    return out


def open_ring(backend, fmt, span, sinks, kv, head, host, scale=SCALE):
    bufs = [backend.upload(b) for b in host]
    return backend.cache4(fmt, span, sinks, kv, head, scale, 0.75 * scale, *bufs)


def close(*things):
    for t in things:
        for b in t.buffers if hasattr(t, "buffers") else [t]:
            b.free()


def rows_of(host, fmt, span, sinks, scale=SCALE):
    def rows(side, places):
        at = c4.slot(places, sinks, span)
        return c4.values(c4.unpack(host[2 * side][at]), host[2 * side + 1][:, at].T, fmt, scale * (0.75 if side else 1))
    return rows


def special_rows(rng, lanes, width):
    """Rows of normals with groups of everything a quotient can be."""
    x = (rng.normal(size=(lanes, width)) * np.exp(0.5 * rng.normal(size=(1, width)))).astype(np.float32)
    g = x.reshape(-1, 32)
    for i, group in enumerate([
            np.zeros(32), np.full(32, -0.0), np.full(32, np.nan), [np.nan] * 31 + [1.0], [np.inf] + [3.0] * 31,
            [-np.inf] * 32, np.full(32, 1e30), np.full(32, 1e-30), [np.inf, np.nan] + [-1e-40] * 30,
            np.full(32, 3e38), np.linspace(-448, 448, 32) * SCALE * 7, np.linspace(0, 1, 32) * SCALE * 7 * 2.0 ** -9,
            np.linspace(0, 1, 32) * SCALE * 7 * 2.0 ** -10, np.linspace(-500, 500, 32) * SCALE * 8]):
        if i < len(g):
            g[len(g) - 1 - i] = np.asarray(group, np.float32)
    return x


def lay_case(backend, fmt, kv, head, sinks, span, place, lanes, pad, off, rows, scale=SCALE):
    width = kv * head
    host = [np.full((span, width // 2), 0xA5, np.uint8), np.full((width // 32, room(span)), 0x5A, np.uint8)] * 2
    store = open_ring(backend, fmt, span, sinks, kv, head, host, scale)
    stride = width + pad
    bufs = []
    for side in range(2):
        x = np.zeros((lanes, stride), np.float32)
        x[:, :width] = rows[side]
        bufs.append(backend.alloc(x.nbytes + 16).put(x, off))
    backend.cache4_lay_dev(store, At(bufs[0], off), At(bufs[1], off), stride, place, lanes)
    backend.sync()
    at = c4.slot(np.arange(place, place + lanes), sinks, span)
    for side in range(2):
        codes, gains = c4.quantise(rows[side], fmt, scale * (0.75 if side else 1))
        want_c, want_g = host[0].copy(), host[1].copy()
        want_c[at], want_g[:, at] = c4.pack(codes), gains.T
        got_c = store.buffers[2 * side].get(np.uint8, want_c.size).reshape(want_c.shape)
        got_g = store.buffers[2 * side + 1].get(np.uint8, want_g.size).reshape(want_g.shape)
        assert np.array_equal(got_g, want_g), side
        assert np.array_equal(got_c, want_c), side
    close(store, *bufs)


@pytest.mark.parametrize("fmt", [c4.INT4, c4.E2M1])
@pytest.mark.parametrize("kv,head,sinks,span,place,lanes,pad,off", [
    (1, 256, 4, 516, 700, 1, 0, 0),      # one decode row past the wrap
    (1, 64, 0, 1, 5, 1, 0, 0),           # the smallest ring
    (1, 512, 0, 700, 0, 700, 0, 0),      # a ring filled
    (3, 128, 5, 105, 3, 102, 0, 0),      # across the sinks' end, the whole ring
    (2, 64, 7, 60, 5000, 53, 3, 4),      # across the wrap, rows off 16-byte alignment
    (8, 128, 0, 130, 128, 100, 4, 0),    # padded rows
    (5, 64, 1, 9, 0, 1, 1, 12),          # one row, one sink
])
def test_lay_is_bit_exact(backend, fmt, kv, head, sinks, span, place, lanes, pad, off):
    print("case lay", fmt, kv, head, sinks, span, place, lanes, pad, off, flush=True)
    rng = np.random.default_rng(head + lanes)
    lay_case(backend, fmt, kv, head, sinks, span, place, lanes, pad, off,
             [special_rows(rng, lanes, kv * head) for _ in range(2)])


@pytest.mark.parametrize("fmt", [c4.INT4, c4.E2M1])
@pytest.mark.parametrize("scale", [2.0 ** -6, SCALE, 1e-30, 3e-44, 1e36])
def test_lay_next_to_every_border(backend, fmt, scale):
    """Values at, one float below and one above halfway between levels, and group
    peaks so near halfway between gains."""
    print("case borders", fmt, scale, flush=True)
    s, top = float(np.float32(0.75 * scale)), c4.TOP[fmt]  # the value side's
    rows = []
    half = c4.HALF[fmt]
    mids = (half[1:] + half[:-1]) / 2
    with np.errstate(over="ignore", under="ignore"):
        for gain in (1, 7, 8, 9, 15, 40, 77, 119, 126):
            step = c4.REAL8[gain] * s
            ties = np.repeat(np.float32(mids * step), 3)
            ties[0::3] = np.nextafter(ties[0::3], np.float32(0))
            ties[2::3] = np.nextafter(ties[2::3], np.float32(np.inf))
            row = np.zeros(32, np.float32)
            row[:21] = ties * np.where(np.arange(21) % 2, -1, 1)
            row[31] = top * step
            rows.append(row)
        for gain in range(126):  # peaks at the borders between gains
            mid = np.float32((c4.REAL8[gain] + c4.REAL8[gain + 1]) / 2 * top * s)
            for peak in (np.nextafter(mid, np.float32(0)), mid, np.nextafter(mid, np.float32(np.inf))):
                rows.append(np.linspace(-1, 1, 32).astype(np.float32) * peak)
    rows = np.stack(rows[:len(rows) // 2 * 2]).reshape(-1, 64)
    rows = np.where(np.isfinite(rows), rows, 0).astype(np.float32)
    lay_case(backend, fmt, 1, 64, 0, len(rows), 0, len(rows), 0, 0, [rows, rows], scale)


@pytest.mark.parametrize("fmt", [c4.INT4, c4.E2M1])
@pytest.mark.parametrize("kv,head,sinks,span,place,lanes,pad,off,sides", [
    (1, 64, 3, 300, 7, 256, 0, 0, 3), (2, 256, 0, 65, 100, 65, 5, 4, 3), (3, 128, 2, 40, 1, 30, 0, 0, 1),
    (1, 512, 0, 33, 32, 1, 0, 0, 2)])
def test_read_is_bit_exact(backend, fmt, kv, head, sinks, span, place, lanes, pad, off, sides):
    """Every code with every gain byte, and floats outside the rows untouched."""
    print("case read", fmt, kv, head, lanes, sides, flush=True)
    rng = np.random.default_rng(head + lanes)
    width, stride = kv * head, kv * head + pad
    host = ring_bytes(rng, span, width, fmt)
    for side in range(2):
        host[2 * side + 1][:] = np.arange(host[2 * side + 1].size).reshape(host[2 * side + 1].shape) % 256
    store = open_ring(backend, fmt, span, sinks, kv, head, host)
    fill = np.full(lanes * stride + 4, 7.0, np.float32)
    outs = [backend.upload(fill) if sides >> side & 1 else None for side in range(2)]
    backend.cache4_read_dev(store, place, lanes, *[At(o, off) if o else None for o in outs], stride)
    backend.sync()
    rows = rows_of(host, fmt, span, sinks)
    for side, out in enumerate(outs):
        if not out:
            continue
        want = fill.copy()
        view = want[off // 4:off // 4 + lanes * stride].reshape(lanes, stride)
        view[:, :width] = rows(side, np.arange(place, place + lanes)).astype(np.float32)
        assert np.array_equal(out.get(np.float32, want.size), want)
        out.free()
    close(store)


def attend(backend, store, share, query, place, window, score, pad=0, off=0):
    lanes, heads = query.shape
    stride = heads + pad
    x = np.full((lanes, stride), np.nan, np.float32)
    x[:, :heads] = query
    dq = backend.alloc(x.nbytes + 16).put(x, off)
    do = backend.alloc(x.nbytes + 16).put(np.full(lanes * stride + 4, 7.0, np.float32))
    backend.attend4_lanes_dev(store, share, At(dq, off), stride, place, window, lanes, score, At(do, off))
    backend.sync()
    got = do.get(np.float32, lanes * stride + 4)
    close(dq, do)
    inside = np.zeros(lanes * stride + 4, bool)
    inside[off // 4:off // 4 + lanes * stride].reshape(lanes, stride)[:, :heads] = True
    assert np.all(got[~inside] == 7.0)
    return got[inside].reshape(lanes, heads)


def check(got, query, rows, share, head, place, window, sinks, score, picks=None):
    """Sampled lanes against 64 bits; the largest error over the bar's unit."""
    lanes = len(query)
    picks = sorted({0, 1, lanes // 3, lanes // 2, lanes - 2, lanes - 1} & set(range(lanes))) if picks is None else picks
    worst = 0.0
    for lane in picks:
        want, reach, vmax = c4.attend(rows, share, head, query[lane:lane + 1], place + lane, window, sinks, score)
        blocks = (len(c4.seen(place + lane, window, sinks)) + 63) // 64 + 3
        bar = vmax * (2 * reach * 2.0 ** -19 + (64 + blocks) * 2.0 ** -24)
        err = float(np.abs(got[lane] - want[0]).max())
        assert err <= bar, (lane, err, bar)
        worst = max(worst, err / float(np.abs(want).max()))
    print("worst error over the largest output", worst, flush=True)


@pytest.mark.parametrize("fmt", [c4.INT4, c4.E2M1])
@pytest.mark.parametrize("kv,share,head,sinks,span,place,window,lanes,pad,off", [
    (1, 8, 256, 0, 1, 0, 0, 1, 0, 0),           # one position
    (1, 8, 256, 4, 516, 5000, 512, 1, 0, 0),    # a sliding layer's step with sinks
    (1, 8, 256, 4, 516, 2, 512, 1, 0, 0),       # before the sinks are full
    (1, 8, 512, 0, 512, 1023, 512, 1, 0, 0),    # the whole ring, no sinks, at its wrap
    (1, 8, 256, 0, 4096, 4095, 0, 1, 0, 0),     # a global layer
    (1, 8, 512, 0, 9000, 8999, 0, 1, 0, 0),
    (2, 4, 128, 70, 200, 1000, 100, 1, 0, 0),   # sinks past a block
    (1, 1, 64, 0, 333, 332, 0, 1, 0, 0),        # one head
    (3, 5, 64, 1, 77, 400, 70, 3, 0, 0),        # odd shares, a few lanes
    (1, 16, 128, 0, 1000, 900, 0, 7, 3, 4),     # sixteen heads, rows off alignment
    (1, 64, 64, 2, 300, 200, 0, 2, 0, 0),       # sixty-four heads
    (1, 8, 512, 0, 3000, 2000, 0, 5, 0, 0),     # a block
    (2, 7, 64, 1, 1100, 3001, 1024, 37, 0, 0),  # a short turn
    (1, 8, 256, 4, 2600, 0, 512, 700, 0, 0),    # a prompt from the first position
    (1, 8, 512, 0, 700, 0, 0, 600, 0, 0),
    (2, 3, 128, 0, 130, 0, 0, 130, 2, 8),
    (1, 12, 256, 3, 900, 3000, 300, 400, 0, 0),
    (1, 8, 256, 0, 5000, 4500, 100, 300, 0, 0),  # a window far inside a ring that keeps all
    (1, 8, 64, 4, 70, 30, 2, 40, 0, 0),          # a window of two
    (1, 8, 256, 4, 70, 30, 1, 3, 0, 0),          # itself and the sinks
    (1, 2, 512, 0, 65, 64, 65, 1, 0, 0),         # one slot of a second block
    (8, 1, 64, 0, 40000, 39999, 0, 1, 0, 0),     # long steps
    (8, 1, 128, 9, 41000, 90000, 40900, 1, 0, 0),  # across the wrap
    (16, 1, 64, 0, 40000, 39999, 0, 1, 0, 0),    # in deep blocks
    (16, 1, 128, 9, 41000, 90000, 40900, 1, 0, 0),
    (1, 64, 128, 5, 300, 290, 0, 9, 4, 4),       # steps of many rows
    # tiles of 64 rows
    (16, 4, 128, 0, 700, 440, 0, 250, 0, 0),     # as many blocks each
    (8, 8, 256, 5, 560, 3000, 300, 250, 4, 4),   # windows across the wrap, rows off alignment
    (4, 16, 512, 3, 720, 9000, 450, 250, 0, 0),
    (2, 8, 128, 3, 6500, 9000, 6400, 60, 0, 0),  # segments of every tile, the last one short
    (2, 8, 512, 0, 4400, 4310, 0, 90, 0, 0),
    (2, 8, 256, 0, 1100, 0, 0, 1100, 0, 0),      # a prompt, its long tiles cut
    (1, 8, 512, 7, 1500, 0, 0, 1400, 0, 0),
    (4, 7, 256, 70, 1170, 2000, 600, 500, 0, 0),  # odd shares, sinks past a block
])
def test_attend(backend, fmt, kv, share, head, sinks, span, place, window, lanes, pad, off):
    print("case attend", fmt, kv, share, head, sinks, span, place, window, lanes, pad, off, flush=True)
    rng = np.random.default_rng(head + lanes + place)
    host = ring_bytes(rng, span, kv * head, fmt)
    store = open_ring(backend, fmt, span, sinks, kv, head, host)
    query = rng.normal(size=(lanes, kv * share * head)).astype(np.float32)
    score = 10.0 / np.sqrt(head)  # scores of deviation 1 to 4: the ring's values are about 1/10 to 1/3
    got = attend(backend, store, share, query, place, window, score, pad, off)
    check(got, query, rows_of(host, fmt, span, sinks), share, head, place, window, sinks, score)
    close(store)


FORMS = [(1, 8, 128, 1, 400), (1, 8, 512, 7, 400), (16, 8, 128, 130, 600), (8, 8, 256, 260, 700), (8, 16, 512, 130, 500)]


@pytest.mark.parametrize("fmt", [c4.INT4, c4.E2M1])
@pytest.mark.parametrize("kv,share,head,lanes,span", FORMS)
@pytest.mark.parametrize("low,high,scale", [(0, 8, 16.0), (0, 256, 2.0 ** -9), (0x78, 0x80, 2.0 ** -13)])
def test_gains_of_every_size(backend, fmt, kv, share, head, lanes, span, low, high, scale):
    """Gains below e4m3's normal numbers, any byte (signs too), the largest."""
    print("case gains", fmt, kv, share, head, lanes, low, flush=True)
    rng = np.random.default_rng(low + head)
    host = ring_bytes(rng, span, kv * head, fmt)
    for side in (1, 3):
        host[side][:] = rng.integers(low, high, size=host[side].shape, dtype=np.uint8)
    place = span - lanes
    store = backend.cache4(fmt, span, 0, kv, head, scale, 0.75 * scale, *(backend.upload(b) for b in host))
    query = rng.normal(size=(lanes, kv * share * head)).astype(np.float32)
    score = 1.0 / np.sqrt(head)
    got = attend(backend, store, share, query, place, 0, score)
    check(got, query, rows_of(host, fmt, span, 0, scale), share, head, place, 0, 0, score, [0, lanes - 1])
    close(store)


@pytest.mark.parametrize("kv,share,head,lanes,span", FORMS)
@pytest.mark.parametrize("score", [0.0, -0.7, 1e-38, -1e-30])
def test_score_scales(backend, kv, share, head, lanes, span, score):
    """No scale at all (the mean of what is seen), one below zero, and the least."""
    print("case score", kv, share, head, lanes, score, flush=True)
    rng = np.random.default_rng(head)
    host = ring_bytes(rng, span, kv * head, c4.E2M1)
    place = span - lanes
    store = open_ring(backend, c4.E2M1, span, 0, kv, head, host)
    query = rng.normal(size=(lanes, kv * share * head)).astype(np.float32)
    got = attend(backend, store, share, query, place, 0, score)
    check(got, query, rows_of(host, c4.E2M1, span, 0), share, head, place, 0, 0, score, [0, lanes - 1])
    close(store)


@pytest.mark.parametrize("kv,share,head,lanes,span", FORMS)
@pytest.mark.parametrize("scale", [2.0 ** 121, 2.0 ** -100])
def test_scales_near_a_floats_ends(backend, kv, share, head, lanes, span, scale):
    """Layers' scales that a float just holds, the largest value below its end; and
    queries of zero beside a factor that no float holds, which see the mean."""
    print("case ends", kv, share, head, lanes, scale, flush=True)
    rng = np.random.default_rng(head)
    host = ring_bytes(rng, span, kv * head, c4.INT4)
    place = span - lanes
    store = open_ring(backend, c4.INT4, span, 0, kv, head, host, scale)
    query = rng.normal(size=(lanes, kv * share * head)).astype(np.float32)
    score = float(np.float32(10.0 / np.sqrt(head) * SCALE / scale))
    rows = rows_of(host, c4.INT4, span, 0, scale)
    got = attend(backend, store, share, query, place, 0, score)
    check(got, query, rows, share, head, place, 0, 0, score, [0, lanes - 1])
    query[:] = 0.0
    got = attend(backend, store, share, query, place, 0, 1e30)
    check(got, query, rows, share, head, place, 0, 0, 1e30, [0, lanes - 1])
    close(store)


@pytest.mark.parametrize("kv,share,head,lanes,span", FORMS)
def test_calls_on_two_desks(backend, kv, share, head, lanes, span):
    """Two desks, each on its stream and with its own workspace, at once: what each
    gives alone, to the bit, call after call."""
    from igllm_amd.backend import Backend
    print("case two desks", kv, share, head, lanes, flush=True)
    rng = np.random.default_rng(head)
    host = ring_bytes(rng, span, kv * head, c4.INT4)
    place, stride = span - lanes, kv * share * head
    query = [rng.normal(size=(lanes, stride)).astype(np.float32) for _ in range(2)]
    other = Backend()
    desks = [backend, other]
    stores = [open_ring(d, c4.INT4, span, 0, kv, head, host) for d in desks]
    want = [attend(d, s, share, q, place, 0, 0.1) for d, s, q in zip(desks, stores, query)]
    dq = [d.upload(q) for d, q in zip(desks, query)]
    do = [[d.alloc(q.nbytes) for _ in range(6)] for d, q in zip(desks, query)]
    for turn in range(6):
        for i, d in enumerate(desks):
            d.attend4_lanes_dev(stores[i], share, dq[i], stride, place, 0, lanes, 0.1, do[i][turn])
    for i, d in enumerate(desks):
        d.sync()
        for out in do[i]:
            assert np.array_equal(out.get(np.float32, want[i].size).reshape(want[i].shape), want[i])
        close(stores[i], dq[i], *do[i])
    other.close()


@pytest.mark.parametrize("fmt", [c4.INT4, c4.E2M1])
@pytest.mark.parametrize("head,lanes", [(256, 1), (256, 9), (64, 70), (512, 40)])
def test_slots_without_rows_count_for_nothing(backend, fmt, head, lanes):
    """Slots that no position was laid in, and the gain rows' padding, hold the
    largest codes and gains: lanes that do not see them are as in a clean ring."""
    print("case unwritten", fmt, head, lanes, flush=True)
    rng = np.random.default_rng(head)
    span, sinks, place = 500, 4, 100
    host = ring_bytes(rng, span, head, fmt)
    query = rng.normal(size=(lanes, 8 * head)).astype(np.float32)
    got = []
    for byte in (0xFF, 0x00):
        for b in host[0], host[2]:
            b[place + lanes:] = byte
        for g in host[1], host[3]:
            g[:, place + lanes:] = 0x7F if byte else 0
        store = open_ring(backend, fmt, span, sinks, 1, head, host)
        got.append(attend(backend, store, 8, query, place, 0, 1.0))
        close(store)
    assert np.array_equal(got[0].view(np.uint32), got[1].view(np.uint32))


@pytest.mark.parametrize("head,lanes", [(64, 1), (256, 1), (512, 3), (256, 70)])
def test_queries_of_any_size(backend, head, lanes):
    """Queries far past binary16's range, up and down, and a NaN or an infinity
    that stays in its own head."""
    print("case query range", head, lanes, flush=True)
    rng = np.random.default_rng(head + 1)
    host = ring_bytes(rng, 200, head, c4.INT4)
    store = open_ring(backend, c4.INT4, 200, 0, 1, head, host)
    place = 200 - lanes
    query = rng.normal(size=(lanes, 8 * head)).astype(np.float32)
    for size in (1e30, 1e-30):
        q = (query * np.float32(size)).astype(np.float32)
        score = 10.0 / np.sqrt(head) / size
        got = attend(backend, store, 8, q, place, 0, score)
        check(got, q, rows_of(host, c4.INT4, 200, 0), 8, head, place, 0, 0, score)
    score = 10.0 / np.sqrt(head)
    clean = attend(backend, store, 8, query, place, 0, score)
    query[0, 2 * head + 5] = np.nan
    query[0, 5 * head + 1] = np.inf
    got = attend(backend, store, 8, query, place, 0, score).reshape(lanes, 8, head)
    assert np.all(np.isnan(got[0, [2, 5]]))
    got[0, [2, 5]] = clean.reshape(lanes, 8, head)[0, [2, 5]]
    assert np.array_equal(got.reshape(clean.shape), clean)
    close(store)


@pytest.mark.parametrize("head,lanes,span", [(256, 1, 3000), (512, 1, 3000), (128, 70, 3000), (512, 70, 600)])
def test_a_peaked_position(backend, head, lanes, span):
    """One position whose score lies 18 (26 powers of two) above all others and
    whose value is zero: the blend is the sum of weights near 2^-26 of the
    largest.  A block's largest weight is held as 2^8 or more, so in its own block
    such a weight is 2^-18 or more, which binary16's smallest step, 2^-24, holds to
    2^-7 of itself."""
    print("case peaked", head, lanes, span, flush=True)
    rng = np.random.default_rng(head)
    host = ring_bytes(rng, span, head, c4.INT4)
    host[0][:] = 0x88  # keys of zero
    host[0][3] = 0x99  # but one
    host[1][:] = 0x38  # gain 1
    host[2][3] = 0x88
    store = open_ring(backend, c4.INT4, span, 0, 1, head, host)
    query = np.ones((lanes, 8 * head), np.float32)
    score = 18.0 / (head * float(np.float32(SCALE)))
    place = span - lanes
    got = attend(backend, store, 8, query, place, 0, score)
    rows = rows_of(host, c4.INT4, span, 0)
    want, _, _ = c4.attend(rows, 8, head, query[:1], place, 0, 0, score)
    size, _, _ = c4.attend(lambda side, t: np.abs(rows(side, t)), 8, head, query[:1], place, 0, 0, score)
    err = float(np.abs(got[0] - want[0]).max() / size.max())
    print("error over the weighted sizes", err, flush=True)
    assert err <= 2.0 ** -7
    close(store)


def test_a_run_of_steps(backend):
    """A session's layer: a prompt laid and attended in one pass, then decode
    steps past the ring's wrap, each row laid and attended; every blend against
    the rows in 64 bits as they were laid, and the last rows read back."""
    print("case run", flush=True)
    rng = np.random.default_rng(11)
    head, share, sinks, window, fmt = 256, 8, 4, 60, c4.E2M1
    span, prompt, steps = sinks + 100, 41, 150
    store = backend.cache4(fmt, span, sinks, 1, head, SCALE, SCALE)
    rows = (rng.normal(size=(2, prompt + steps, head))).astype(np.float32)
    kept = [c4.values(*c4.quantise(rows[s], fmt, SCALE), fmt, SCALE) for s in range(2)]
    query = rng.normal(size=(prompt + steps, share * head)).astype(np.float32)
    dk, dv, dq = backend.upload(rows[0]), backend.upload(rows[1]), backend.upload(query)
    do = backend.alloc(query.nbytes)
    place = 0
    for lanes in [prompt] + [1] * steps:
        backend.cache4_lay_dev(store, At(dk, place * head * 4), At(dv, place * head * 4), head, place, lanes)
        at = place * share * head * 4
        backend.attend4_lanes_dev(store, share, At(dq, at), share * head, place, window, lanes, 1 / 16, At(do, at))
        place += lanes
    out = backend.alloc(50 * head * 4)
    backend.cache4_read_dev(store, place - 50, 50, out, None, head)
    backend.sync()
    got = do.get(np.float32, query.size).reshape(query.shape)
    check(got, query, lambda side, t: kept[side][t], share, head, 0, window, sinks, 1 / 16,
          [0, 1, 5, 40, 41, 63, 64, 65, 100, 103, 104, 105, 150, 190])
    assert np.array_equal(out.get(np.float32, 50 * head).reshape(50, head), kept[0][-50:].astype(np.float32))
    close(store, dk, dv, dq, do, out)


@pytest.mark.parametrize("lanes,place,head", [(1, 4000, 256), (3, 3000, 512), (100, 1900, 256), (130, 0, 512),
                                              (200, 9000, 256), (1500, 0, 512)])
def test_recorded_and_replayed(backend, lanes, place, head):
    """Rows laid and attended in a recording, replayed over other rows with the
    program's own calls between: every replay equals the eager calls to the bit,
    and no call moves the desk's workspaces, one beside a live replay included."""
    print("case replay", lanes, place, head, flush=True)
    rng = np.random.default_rng(lanes)
    span = place + lanes
    host = ring_bytes(rng, span, head, c4.INT4)
    store = open_ring(backend, c4.INT4, span, 0, 1, head, host)
    stride = 8 * head
    dk, dv = backend.alloc(lanes * head * 4), backend.alloc(lanes * head * 4)
    dq, do = backend.alloc(lanes * stride * 4), backend.alloc(lanes * stride * 4)
    side = open_ring(backend, c4.INT4, span, 0, 1, head, host)
    do2 = backend.alloc(lanes * stride * 4)
    generation = backend.lib.igl_desk_generation
    generation.argtypes, generation.restype = [ctypes.c_void_p], ctypes.c_uint
    before = generation(ctypes.byref(backend.desk))

    def step(ring, out):
        backend.cache4_lay_dev(ring, dk, dv, head, place, lanes)
        backend.attend4_lanes_dev(ring, 8, dq, stride, place, 0, lanes, 1 / 16, out)

    backend.record_begin()
    step(store, do)
    replay = backend.record_end()
    try:
        for turn in range(4):
            for buf, n in ((dk, head), (dv, head), (dq, stride)):
                buf.put(rng.normal(size=(lanes, n)).astype(np.float32))
            backend.replay_run(replay)
            step(side, do2)
            backend.replay_run(replay)
            backend.sync()
            a, b = (x.get(np.uint32, lanes * stride) for x in (do, do2))
            assert np.array_equal(a, b), turn
            assert np.all(np.isfinite(a.view(np.float32)))
    finally:
        backend.replay_free(replay)
    assert generation(ctypes.byref(backend.desk)) == before
    close(store, side, dk, dv, dq, do, do2)


@pytest.mark.parametrize("kv,share,head,lanes,span", FORMS[2:])
def test_tiles_beside_slots_without_rows(backend, kv, share, head, lanes, span):
    """Tiles of 64 rows: slots that no position was laid in, and a NaN in a query,
    touch no other row."""
    print("case tiles unwritten", kv, share, head, lanes, flush=True)
    rng = np.random.default_rng(head)
    held = span - 70
    host = ring_bytes(rng, span, kv * head, c4.INT4)
    query = rng.normal(size=(lanes, kv * share * head)).astype(np.float32)
    bad = (3 * share + 1) * head
    got = []
    for byte in (0xFF, 0x00):
        for b in host[0], host[2]:
            b[held:] = byte
        for g in host[1], host[3]:
            g[:, held:] = 0x7F if byte else 0
        store = open_ring(backend, c4.INT4, span, 0, kv, head, host)
        got.append(attend(backend, store, share, query, held - lanes, 0, 0.1))
        close(store)
        query[5, bad] = np.nan  # the second time
    assert np.all(np.isnan(got[1][5, bad:bad + head]))
    got[1][5, bad:bad + head] = got[0][5, bad:bad + head]
    assert np.array_equal(got[0], got[1])


def test_offsets_past_32_bits(backend):
    """A ring of more than 2^32 bytes of codes: rows past them laid, read and seen."""
    print("case long", flush=True)
    head, fmt, window = 512, c4.E2M1, 100
    span = (1 << 24) + 5000
    sizes = [span * head // 2, head // 32 * room(span)] * 2
    bufs = [backend.alloc(n) for n in sizes]
    store = backend.cache4(fmt, span, 0, 1, head, SCALE, SCALE, *bufs)
    rng = np.random.default_rng(3)
    place, lanes = (1 << 24) + 3000, 130
    rows = rng.normal(size=(2, lanes, head)).astype(np.float32)
    dk, dv = backend.upload(rows[0]), backend.upload(rows[1])
    backend.cache4_lay_dev(store, dk, dv, head, place, lanes)
    out = backend.alloc(lanes * head * 4)
    backend.cache4_read_dev(store, place, lanes, None, out, head)
    backend.sync()
    kept = [c4.values(*c4.quantise(rows[s], fmt, SCALE), fmt, SCALE) for s in range(2)]
    assert np.array_equal(out.get(np.float32, lanes * head).reshape(lanes, head), kept[1].astype(np.float32))
    for first, n in ((lanes - 1, 1), (lanes - 21, 21)):
        query = rng.normal(size=(n, 8 * head)).astype(np.float32)
        got = attend(backend, store, 8, query, place + first, window, 1 / 16)
        for lane in {0, n - 1}:
            t = np.arange(first + lane - window + 1, first + lane + 1)
            k, v = kept[0][t], kept[1][t]
            s = query[lane].reshape(8, head).astype(np.float64) @ k.T / 16
            w = np.exp(s - s.max(-1, keepdims=True))
            want = (w @ v / w.sum(-1, keepdims=True)).reshape(-1)
            reach = float((np.abs(query[lane].reshape(8, head)) @ np.abs(k).T).max()) / 16
            assert np.abs(got[lane] - want).max() <= np.abs(v).max() * (2 * reach * 2.0 ** -19 + 70 * 2.0 ** -24)
    close(store, dk, dv, out)


def test_refusals_leave_the_outputs(backend):
    """A refused call writes nothing and the desk goes on."""
    print("case refused", flush=True)
    lib, desk = backend.lib, ctypes.byref(backend.desk)
    store = backend.cache4(c4.INT4, 100, 4, 1, 64, SCALE, SCALE)
    out = backend.upload(np.full(8 * 64, 7.0, np.float32))
    assert lib.igl_attend4_lanes_dev(desk, ctypes.byref(store.cache), 8, out.ptr, 512, 200, 97, 1, 1.0, out.ptr) == \
        native.IGL_FAIL_ARGUMENT
    assert backend.error_take() == native.IGL_FAIL_ARGUMENT
    assert np.all(out.get(np.float32, 512) == 7.0)
    backend.cache4_lay_dev(store, out, out, 64, 0, 1)
    backend.sync()
    close(store, out)
