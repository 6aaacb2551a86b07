"""GPU attention over the 4-bit ring at the ends of its numbers: scales, scores
and weights far from one another, against 64 bits."""
import ctypes

import numpy as np
import pytest

import cache4_oracle as c4
from test_gpu_cache4 import SCALE, attend, check, close, open_ring, ring_bytes, rows_of

pytestmark = pytest.mark.gpu


def keyed_ring(rng, span, width, high):
    """A ring whose keys are zero but at slots `high`, there one level of gain 1."""
    host = ring_bytes(rng, span, width, c4.INT4)
    host[0][:] = 0x88
    host[0][high] = 0x99
    host[1][:] = 0x38
    return host


@pytest.mark.parametrize("every", [350, 1 << 20])
@pytest.mark.parametrize("kv,share,head,sinks,span,place,window,lanes", [
    (8, 1, 64, 0, 40000, 39999, 0, 1),     # eight rows, folded
    (16, 1, 64, 0, 40000, 39999, 0, 1),    # in long blocks
    (1, 8, 64, 0, 2047, 0, 0, 2047),       # sixteen, in one segment
    (1, 8, 256, 4, 2600, 0, 512, 2047),    # tiles
    (1, 8, 512, 7, 1500, 0, 0, 1400),      # folded
    (2, 8, 128, 3, 6500, 9000, 6400, 60),
])
def test_value_scales_under_falling_peaks(backend, kv, share, head, sinks, span, place, window, lanes, every):
    """Positions (one, or one in 350) 64 powers of two above those after them, so that a row's sums grow
    by 2^58 as its base follows the peaks down, under a value scale of 2^-100: no
    product of the scale with the sums' reciprocal is a float, each blend is."""
    print("case falling", kv, share, head, span, lanes, every, flush=True)
    rng = np.random.default_rng(head + lanes)
    host = keyed_ring(rng, span, kv * head, slice(3, None, every))
    scales = SCALE, 2.0 ** -100
    store = backend.cache4(c4.INT4, span, sinks, kv, head, *scales, *(backend.upload(b) for b in host))
    query = np.ones((lanes, kv * share * head), np.float32)
    score = 64.0 * np.log(2.0) / (head * float(np.float32(SCALE)))
    got = attend(backend, store, share, query, place, window, score)

    def rows(side, places):
        at = c4.slot(places, sinks, span)
        return c4.values(c4.unpack(host[2 * side][at]), host[2 * side + 1][:, at].T, c4.INT4, scales[side])

    check(got, query, rows, share, head, place, window, sinks, score)
    close(store)


@pytest.mark.parametrize("fmt", [c4.INT4, c4.E2M1])
@pytest.mark.parametrize("kv,share,head,span", [(16, 1, 64, 40000), (16, 1, 128, 40000), (8, 4, 128, 65600)])
def test_a_peaked_position_of_long_blocks(backend, fmt, kv, share, head, span):
    """A position of zero value 26 powers of two above zero, all others' scores within
    `near` powers of it, in blocks of 512 slots, and values in its own block alone:
    weights are held to half of binary16's smallest step, 2^-25, beside one of 2^8 or
    more, so the others, 2^(-18 - near) at least, to 2^(near - 7) of themselves."""
    print("case peaked long", fmt, kv, share, head, span, flush=True)
    rng = np.random.default_rng(head)
    host = ring_bytes(rng, span, kv * head, fmt)
    zero = 0x88 if fmt == c4.INT4 else 0x00
    host[0][3] = 0x99 if fmt == c4.INT4 else 0x22  # level 1
    host[1][:] = 0x08 if fmt == c4.INT4 else 0x10  # 2^-6 and 2^-5: others' scores are near zero
    host[1][:, 3] = 0x38
    host[2][3] = host[2][512:] = zero
    store = open_ring(backend, fmt, span, 0, kv, head, host)
    query = np.ones((1, kv * share * head), np.float32)
    score = 18.0 / (head * float(np.float32(SCALE)))
    got = attend(backend, store, share, query, span - 1, 0, score).reshape(kv, share, head)
    rows = rows_of(host, fmt, span, 0)
    s = rows(0, np.arange(span)).reshape(span, kv, head).sum(-1) * score
    near = np.abs(np.delete(s, 3, 0)).max() / np.log(2.0)
    w = np.exp(s)
    v = rows(1, np.arange(512)).reshape(512, kv, head)
    err = np.abs(got - (w[:512, :, None] * v).sum(0)[:, None] / w.sum(0)[:, None, None]).max()
    size = ((w[:512, :, None] * np.abs(v)).sum(0) / w.sum(0)[:, None]).max()
    print("near", near, "error over the weighted sizes", err / size, flush=True)
    assert near < 4.0
    assert err <= 2.0 ** (near - 7) * size
    close(store)


@pytest.mark.parametrize("kv,share,head,sinks,span,place,window,lanes", [
    (1, 8, 256, 0, 4096, 4095, 0, 1), (16, 1, 64, 0, 40000, 39999, 0, 1), (1, 8, 512, 0, 3000, 2000, 0, 5),
    (2, 8, 128, 3, 6500, 9000, 6400, 60), (1, 8, 512, 7, 1500, 0, 0, 1400)])
def test_launches_without_room_for_partials(backend, kv, share, head, sinks, span, place, window, lanes):
    """What a desk without partials launches: every row's blocks in one segment."""
    print("case no partials", kv, share, head, span, lanes, flush=True)
    rng = np.random.default_rng(head + lanes)
    host = ring_bytes(rng, span, kv * head, c4.E2M1)
    store = open_ring(backend, c4.E2M1, span, sinks, kv, head, host)
    stride = kv * share * head
    query = rng.normal(size=(lanes, stride)).astype(np.float32)
    score = 10.0 / np.sqrt(head)
    dq, do = backend.upload(query), backend.alloc(query.nbytes)
    stream = backend.lib.igl_desk_stream
    stream.restype, stream.argtypes = ctypes.c_void_p, [ctypes.c_void_p]
    launch = backend.lib.igl_launch_attend4
    launch.restype = ctypes.c_int
    launch.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p] + [ctypes.c_int] * 4 + [
        ctypes.c_float, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p]
    assert launch(ctypes.byref(store.cache), share, dq.ptr, stride, place, window, lanes, score, do.ptr, None,
                  stream(ctypes.byref(backend.desk))) == 0
    backend.sync()
    got = do.get(np.float32, query.size).reshape(query.shape)
    check(got, query, rows_of(host, c4.E2M1, span, sinks), share, head, place, window, sinks, score)
    close(store, dq, do)


@pytest.mark.parametrize("fmt", [c4.INT4, c4.E2M1])
@pytest.mark.parametrize("kv,share,head,sinks,span,place,window", [
    (2, 8, 64, 0, 131072, 131071, 0), (2, 4, 128, 0, 131072, 131071, 0), (8, 4, 128, 4, 45004, 90000, 45000),
    (8, 1, 64, 3, 45000, 44999, 0), (16, 1, 128, 9, 41000, 90000, 40900)])
def test_steps_in_blocks_between(backend, fmt, kv, share, head, sinks, span, place, window):
    """Steps in blocks of 256 slots: long contexts of few heads, and the wrap."""
    print("case between", fmt, kv, share, head, span, place, flush=True)
    rng = np.random.default_rng(head + kv)
    host = ring_bytes(rng, span, kv * head, fmt)
    store = open_ring(backend, fmt, span, sinks, kv, head, host)
    query = rng.normal(size=(1, kv * share * head)).astype(np.float32)
    score = 10.0 / np.sqrt(head)
    got = attend(backend, store, share, query, place, window, score)
    check(got, query, rows_of(host, fmt, span, sinks), share, head, place, window, sinks, score)
    close(store)


@pytest.mark.parametrize("kv,share,head,lanes,span", [(1, 8, 128, 1, 400), (1, 8, 512, 7, 400), (16, 1, 64, 1, 40000),
                                                      (8, 8, 256, 260, 700), (8, 16, 512, 130, 500)])
@pytest.mark.parametrize("score", [np.inf, -np.inf, np.nan])
def test_score_scales_that_are_no_numbers(backend, kv, share, head, lanes, span, score):
    """Infinite scores differ by no number: no blend is one, of queries of zero either."""
    print("case no score", kv, share, head, lanes, score, flush=True)
    rng = np.random.default_rng(head)
    host = ring_bytes(rng, span, kv * head, c4.INT4)
    store = open_ring(backend, c4.INT4, span, 0, kv, head, host)
    query = rng.normal(size=(lanes, kv * share * head)).astype(np.float32)
    query[0] = 0.0
    assert np.all(np.isnan(attend(backend, store, share, query, span - lanes, 0, score)))
    close(store)


@pytest.mark.parametrize("kv,share,head,sinks,span,place,window,lanes", [
    (1, 8, 128, 0, 400, 399, 0, 1), (16, 1, 64, 0, 40000, 39999, 0, 1), (2, 8, 64, 0, 131072, 131071, 0, 1),
    (1, 8, 512, 0, 3000, 2000, 0, 5), (1, 8, 64, 0, 700, 0, 0, 600), (8, 8, 256, 5, 560, 3000, 300, 250),
    (8, 16, 512, 0, 500, 370, 0, 130), (2, 8, 128, 3, 6500, 9000, 6400, 60)])
@pytest.mark.parametrize("power", [20, 24, 27, 33, 60, 110])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_far_apart(backend, kv, share, head, sinks, span, place, window, lanes, power, sign):
    """Scores of zero and of 1.3 times 2^power, positive or negative, in powers of two: a
    row sees the mean of the higher ones' values, however coarse a float is there."""
    print("case far", kv, share, head, span, lanes, power, sign, flush=True)
    rng = np.random.default_rng(head + power)
    host = ring_bytes(rng, span, kv * head, c4.E2M1)
    host[0][:] = 0x00
    host[0][5::90] = 0x22  # level 1
    host[1][:] = 0x38
    store = open_ring(backend, c4.E2M1, span, sinks, kv, head, host)
    query = np.ones((lanes, kv * share * head), np.float32)
    query[:] *= 1.0 + rng.integers(0, 64, size=(lanes, 1)).astype(np.float32) / 64
    score = sign * 1.3 * 2.0 ** power * np.log(2.0) / (head * float(np.float32(SCALE)))
    got = attend(backend, store, share, query, place, window, score).reshape(lanes, kv, share, head)
    rows = rows_of(host, c4.E2M1, span, sinks)
    for lane in sorted({0, lanes // 2, lanes - 1}):
        t = c4.seen(place + lane, window, sinks)
        far = c4.slot(t, sinks, span) % 90 == 5
        high = far if sign > 0 and far.any() else ~far if sign < 0 and not far.all() else np.ones(len(t), bool)
        v = rows(1, t[high]).reshape(-1, kv, head)
        err = np.abs(got[lane] - v.mean(0)[:, None]).max()
        assert err <= np.abs(v).max() * (64 + (len(t) + 63) // 64 + 3) * 2.0 ** -24, (lane, err)
    close(store)
