"""GPU parity of microscaled 4-bit rows: what is laid, what is read back, and
products, against their definitions in 64 bits (mx4_oracle).

Codes and scales are decided exactly: every byte equal, bytes of other rows and
between rows untouched.  A read value is exact.

Bar of a product, from the arithmetic.  A lane's group is held to e = 2^-23 / 1.875
(fp32 lanes) or 2^-13 / 1.875 (bf16 lanes) of its largest value: the largest lies
above 1.875 of its scale, and what five terms leave is at most half the widest step,
1/8, of the last, 2^-20 of the first's (test_mx4_terms); so an output is off by
e * sum |w| top(group); the sums are fp32 adds, sixteen an instruction and an
instruction for every 128 columns and term, each off by 2^-24 of what it holds,
at most 1.1 sum |w x| (the terms together are no larger than x by a sixteenth).
An output in bf16 is rounded by 2^-8 more.
"""
import ctypes

import numpy as np
import pytest

import mx4_oracle as mx
from igllm_amd import native

pytestmark = pytest.mark.gpu

F32, BF16 = native.IGL_STORE_F32, native.IGL_STORE_BF16
TERMS = {F32: 5, BF16: 3}
HELD = {F32: 2.0 ** -23 / 1.875, BF16: 2.0 ** -13 / 1.875}


class At:
    """A device address inside a buffer."""

    def __init__(self, buf, offset):
        self.ptr = buf.ptr + offset


def close(*things):
    for t in things:
        for b in t.buffers if hasattr(t, "buffers") else [t]:
            b.free()


def special_rows(rng, rows, cols):
    """Rows of normals with groups of everything a group can be."""
    x = (rng.normal(size=(rows, cols)) * np.exp(0.5 * rng.normal(size=(1, cols)))).astype(np.float32)
    g = x.reshape(-1, 32)
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0])
    ties = np.concatenate([ties, np.nextafter(ties.astype(np.float32), 0), np.nextafter(ties.astype(np.float32), 9)])
    for i, group in enumerate([
            np.zeros(32), np.full(32, -0.0), [np.nan] + [1.0] * 31, [1.0] * 31 + [np.inf], [-np.inf] * 32,
            np.full(32, 3.4e38), np.full(32, 1e-38), np.full(32, 1e-45), [1e-40, -3e-39] * 16,
            np.concatenate([ties, -ties[:8]]), np.concatenate([ties, -ties[:8]]) * 2.0 ** 100,
            np.concatenate([ties, -ties[:8]]) * 2.0 ** -120, np.concatenate([ties, -ties[:8]]) * 2.0 ** -127,
            np.linspace(-8, 8, 32), np.linspace(-1, 1, 32) * 7.999999, [1e30] + [1e-30] * 31]):
        if i < len(g):
            g[len(g) - 1 - i] = np.asarray(group, np.float32)
    return x


def put(backend, x, kind):
    return backend.upload(mx.bf16_bits(x) if kind == BF16 else np.ascontiguousarray(x, np.float32))


def get(buf, shape, kind, offset=0):
    count = int(np.prod(shape))
    raw = buf.get(np.uint16 if kind == BF16 else np.float32, count, offset)
    return (mx.bits_float(raw) if kind == BF16 else raw).reshape(shape)


def sheet(rng, rows, cols, low=118, high=126):
    """Random codes and scales."""
    return (rng.integers(0, 256, size=(rows, cols // 2), dtype=np.uint8),
            rng.integers(low, high, size=(rows, cols // 32)).astype(np.uint8))


def hold(backend, packed, scale, pad=0, scale_pad=0):
    """Rows in device memory, bytes of 0xEE between them."""
    out = []
    for a, p in ((packed, pad), (scale, scale_pad)):
        host = np.full((len(a), a.shape[1] + p), 0xEE, np.uint8)
        host[:, :a.shape[1]] = a
        out.append((backend.upload(host), a.shape[1] + p))
    (code, code_stride), (sc, scale_stride) = out
    return backend.mx4(len(packed), 2 * packed.shape[1], code, sc, code_stride, scale_stride)


# ---- rows ----------------------------------------------------------------------

@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("rows,cols,pad,scale_pad,extra", [(1, 32, 0, 0, 0), (3, 96, 16, 1, 5), (17, 544, 0, 3, 1),
                                                            (40, 2048, 32, 0, 0), (301, 64, 0, 0, 3)])
def test_lay_and_read(backend, kind, rows, cols, pad, scale_pad, extra):
    rng = np.random.default_rng(rows * cols)
    total, first = rows + 4, 2
    x = special_rows(rng, rows, cols)
    if kind == BF16:
        x = mx.bf16(x)
    wide = np.full((rows, cols + extra), 7.5, np.float32)
    wide[:, :cols] = x
    old = rng.integers(0, 256, size=(total, cols // 2), dtype=np.uint8), rng.integers(1, 255, size=(total, cols // 32)).astype(np.uint8)
    store = hold(backend, *old, pad, scale_pad)
    src = put(backend, wide, kind)
    backend.mx4_lay_dev(store, first, rows, src, kind, cols + extra)
    code, scale = mx.quantise(x)
    got_code = store.buffers[0].get(np.uint8, total * (cols // 2 + pad)).reshape(total, -1)
    got_scale = store.buffers[1].get(np.uint8, total * (cols // 32 + scale_pad)).reshape(total, -1)
    want_code, want_scale = old[0].copy(), old[1].copy()
    want_code[first:first + rows], want_scale[first:first + rows] = mx.pack(code), scale
    assert np.array_equal(got_scale[:, :cols // 32], want_scale)
    assert np.array_equal(got_code[:, :cols // 2], want_code)
    assert (got_code[:, cols // 2:] == 0xEE).all() and (got_scale[:, cols // 32:] == 0xEE).all()
    for out_kind in (F32, BF16):
        out = put(backend, np.full((rows + 1, cols + extra), 7.5, np.float32), out_kind)
        backend.mx4_read_dev(store, first, rows, out, out_kind, cols + extra)
        got = get(out, (rows + 1, cols + extra), out_kind)
        want = mx.values(mx.pack(code), scale).astype(np.float32)
        want = mx.bf16(want) if out_kind == BF16 else want
        assert np.array_equal(got[:rows, :cols], want, equal_nan=True)
        assert (got[rows] == 7.5).all() and (got[:, cols:] == 7.5).all()
        close(out)
    close(store, src)


def test_read_every_code_and_scale(backend):
    code = np.tile(np.arange(32, dtype=np.uint8) % 16, (256, 1))
    scale = np.arange(256, dtype=np.uint8)[:, None]
    store = hold(backend, mx.pack(code), scale)
    out = backend.alloc(256 * 32 * 4)
    backend.mx4_read_dev(store, 0, 256, out, F32, 32)
    got = out.get(np.float32, 256 * 32).reshape(256, 32)
    with np.errstate(over="ignore"):
        want = mx.values(mx.pack(code), scale).astype(np.float32)  # 6 * 2^127 is past the largest float
    assert np.array_equal(got, want, equal_nan=True)
    close(store, out)


# ---- products ------------------------------------------------------------------

def bar(x, w, kind, out_kind, want):
    """How far outputs may be off."""
    top = np.repeat(np.abs(x).reshape(len(x), -1, 32).max(-1), 32, 1)
    if kind is None:
        held, adds = 0.0, 16 * (-(-x.shape[1] // 128))
    else:
        held, adds = HELD[kind] * (top @ np.abs(w).T), 16 * TERMS[kind] * (-(-x.shape[1] // 128))
    tol = held + adds * 2.0 ** -24 * 1.1 * (np.abs(x) @ np.abs(w).T)
    return tol + 2.0 ** -8 * (np.abs(want) + tol) if out_kind == BF16 else tol


SHAPES = [(1, 16, 32), (1, 1, 64), (1, 6144, 1536), (2, 50, 96), (3, 33, 128), (4, 200, 160), (5, 1000, 2080),
          (6, 77, 8192), (7, 130, 544), (8, 64, 256), (13, 17, 1536), (16, 48, 384), (17, 47, 416), (31, 300, 224),
          (37, 257, 8192), (63, 129, 704), (64, 256, 512), (65, 100, 1056), (100, 520, 768), (129, 1030, 96),
          (300, 1537, 1536), (517, 272, 320), (1000, 300, 2048),
          # a head; tiles of many lanes and rows, the last of either not full
          (4, 32776, 1760), (16, 40001, 1408), (2, 65540, 96), (500, 6150, 64), (1000, 6201, 96), (1540, 7690, 160),
          # columns in slices, the last one short
          (70, 2100, 8192), (21, 4100, 4128)]


@pytest.mark.parametrize("lanes,rows,cols", SHAPES)
@pytest.mark.parametrize("kind,out_kind", [(F32, F32), (BF16, BF16), (BF16, F32), (F32, BF16)])
def test_product(backend, lanes, rows, cols, kind, out_kind):
    rng = np.random.default_rng(lanes * 7 + rows * 3 + cols)
    x = (rng.normal(size=(lanes, cols)) * np.exp(0.5 * rng.normal(size=(1, cols)))).astype(np.float32)
    x = mx.bf16(x) if kind == BF16 else x
    w = sheet(rng, rows, cols)
    lane_pad, out_pad = (0, 0) if lanes % 2 else (3, 5)
    wide = np.full((lanes, cols + lane_pad), 9.0, np.float32)
    wide[:, :cols] = x
    held = hold(backend, *w, 16 * (rows % 2), rows % 3)
    act = put(backend, wide, kind)
    out = put(backend, np.full((lanes + 1, rows + out_pad), 7.5, np.float32), out_kind)
    print("product", lanes, rows, cols, kind, out_kind, flush=True)
    backend.mx4_mat_mat_dev(held, act, kind, cols + lane_pad, lanes, out, out_kind, rows + out_pad)
    got = get(out, (lanes + 1, rows + out_pad), out_kind)
    wv = mx.values(*w)
    want = x.astype(np.float64) @ wv.T
    assert (np.abs(got[:lanes, :rows] - want) <= bar(x, wv, kind, out_kind, want)).all()
    assert (got[lanes] == 7.5).all() and (got[:, rows:] == 7.5).all()
    # what the worst-case bar allows is far more than what sums of random signs are off by
    rms = np.sqrt(np.mean(want ** 2))
    if out_kind == F32:
        assert np.sqrt(np.mean((got[:lanes, :rows] - want) ** 2)) <= (2.0 ** -19 if kind == F32 else 2.0 ** -12) * rms
    close(held, act, out)


@pytest.mark.parametrize("lanes,rows,cols", SHAPES)
@pytest.mark.parametrize("out_kind", [F32, BF16])
def test_product_of_microscaled_lanes(backend, lanes, rows, cols, out_kind):
    rng = np.random.default_rng(lanes * 5 + rows * 3 + cols)
    w, a = sheet(rng, rows, cols), sheet(rng, lanes + 3, cols)
    held, act = hold(backend, *w, 16 * (rows % 2), rows % 3), hold(backend, *a, 16 * (lanes % 2), lanes % 3)
    out = put(backend, np.full((lanes + 1, rows + 2), 7.5, np.float32), out_kind)
    print("microscaled product", lanes, rows, cols, out_kind, flush=True)
    backend.mx4_mat_mx4_dev(held, act, 2, lanes, out, out_kind, rows + 2)
    got = get(out, (lanes + 1, rows + 2), out_kind)
    x, wv = mx.values(*a)[2:2 + lanes], mx.values(*w)
    want = x @ wv.T
    assert (np.abs(got[:lanes, :rows] - want) <= bar(x, wv, None, out_kind, want)).all()
    assert (got[lanes] == 7.5).all() and (got[:, rows:] == 7.5).all()
    close(held, act, out)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("lanes", [1, 3, 9, 40, 150])
@pytest.mark.parametrize("spread", [0.0, 3.0])
def test_every_value_is_held(backend, kind, lanes, spread):
    """A sheet with one code a row passes every value through: each is held to its bar, which a term less
    would pass (2^-19 and 2^-9 of a group's largest)."""
    cols = 416
    rng = np.random.default_rng(lanes)
    x = (rng.normal(size=(lanes, cols)) * np.exp(spread * rng.normal(size=(lanes, cols)))).astype(np.float32)
    x = mx.bf16(x) if kind == BF16 else x
    code = 2 * np.eye(cols, dtype=np.uint8)
    held, act = hold(backend, mx.pack(code), np.full((cols, cols // 32), 127, np.uint8)), put(backend, x, kind)
    out = backend.alloc(4 * lanes * cols)
    backend.mx4_mat_mat_dev(held, act, kind, cols, lanes, out, F32, cols)
    got = out.get(np.float32, lanes * cols).reshape(lanes, cols)
    top = np.repeat(np.abs(x).reshape(lanes, -1, 32).max(-1), 32, 1)
    # and an fp32 rounding as each term is added
    assert (np.abs(got - x.astype(np.float64)) <= HELD[kind] * top + TERMS[kind] * 2.0 ** -24 * 1.1 * np.abs(x)).all()
    close(held, act, out)


@pytest.mark.parametrize("lanes", [1, 4, 20, 130])
def test_range(backend, lanes):
    """Lanes and sheets of every size: the smallest floats count as zero, the largest pass infinity as sums do."""
    cols, rows = 160, 40
    rng = np.random.default_rng(3)
    for power in (-140, -126, -100, -20, 40, 100, 120):
        x = np.ldexp(rng.normal(size=(lanes, cols)), power).astype(np.float32)
        x[:, 32:64] = 0
        for low in (1, 60, 127, 180, 240):
            w = sheet(rng, rows, cols, low, low + 4)
            held, act, out = hold(backend, *w), put(backend, x, F32), backend.alloc(4 * lanes * rows)
            backend.mx4_mat_mat_dev(held, act, F32, cols, lanes, out, F32, rows)
            got = out.get(np.float32, lanes * rows).reshape(lanes, rows).astype(np.float64)
            wv = mx.values(*w)
            want = x.astype(np.float64) @ wv.T
            reach = np.abs(x.astype(np.float64)) @ np.abs(wv).T
            # beside the product's bar: what lies below 2^-130 of lanes, and fp32's smallest step
            tol = bar(x.astype(np.float64), wv, F32, F32, want) + 2.0 ** -130 * np.abs(wv).sum(1) + 200 * 2.0 ** -126
            sure = reach < 2.0 ** 126
            assert (np.abs(got - want) <= tol)[sure].all(), (power, low)
            over = np.abs(want) > 2.0 ** 129
            assert (~np.isfinite(got))[over].all()
            close(held, act, out)


@pytest.mark.parametrize("lanes", [1, 5, 30, 700])
@pytest.mark.parametrize("kind", [F32, BF16])
def test_the_largest_lanes(backend, lanes, kind):
    """Values up to the largest of their type, whose group's scale is the largest byte that is none's."""
    cols, rows = 96, 200
    rng = np.random.default_rng(lanes)
    top = np.float32(3.4028234663852886e38)
    x = (top * rng.uniform(0.2, 1, size=(lanes, cols)) * rng.choice([-1, 1], size=(lanes, cols))).astype(np.float32)
    x[:, ::7] = top
    if kind == BF16:
        x = mx.bits_float(x.view(np.uint32) >> 16)  # towards zero: the largest stays finite
    w = sheet(rng, rows, cols, 40, 44)
    held, act, out = hold(backend, *w), put(backend, x, kind), backend.alloc(4 * lanes * rows)
    backend.mx4_mat_mat_dev(held, act, kind, cols, lanes, out, F32, rows)
    wv = mx.values(*w)
    want = x.astype(np.float64) @ wv.T
    assert (np.abs(get(out, (lanes, rows), F32) - want) <= bar(x.astype(np.float64), wv, kind, F32, want)).all()
    close(held, act, out)


@pytest.mark.parametrize("lanes", [1, 5, 30, 140])
@pytest.mark.parametrize("kind", [F32, BF16])
def test_what_is_no_number(backend, lanes, kind):
    """A lane with an infinity or a NaN has NaN outputs, the others theirs; a sheet's group of scale 255 too."""
    cols, rows = 288, 50
    rng = np.random.default_rng(lanes)
    x = mx.bf16(rng.normal(size=(lanes, cols)))
    w = sheet(rng, rows, cols)
    w[1][7, 3] = 255
    bad = list(range(0, lanes, 3))
    for i, m in enumerate(bad):
        x[m, (i * 37) % cols] = [np.nan, np.inf, -np.inf][i % 3]
    held, act, out = hold(backend, *w), put(backend, x, kind), backend.alloc(4 * lanes * rows)
    backend.mx4_mat_mat_dev(held, act, kind, cols, lanes, out, F32, rows)
    got = out.get(np.float32, lanes * rows).reshape(lanes, rows)
    assert np.isnan(got[bad]).all() and np.isnan(got[:, 7]).all()
    good = [m for m in range(lanes) if m not in bad]
    rest = [n for n in range(rows) if n != 7]
    assert np.isfinite(got[good][:, rest]).all()
    clean = np.where(np.isfinite(x), x, 0)
    want = clean.astype(np.float64) @ np.nan_to_num(mx.values(*w)).T
    assert (np.abs(got - want) <= bar(clean, np.nan_to_num(mx.values(*w)), kind, F32, want))[np.ix_(good, rest)].all()
    close(held, act, out)


def test_a_lane_alone_and_among_others(backend):
    """What a lane's neighbours hold does not change it, in any form: each to its own bar."""
    cols, rows, lanes = 1536, 512, 200
    rng = np.random.default_rng(9)
    x = rng.normal(size=(lanes, cols)).astype(np.float32)
    w = sheet(rng, rows, cols)
    held = hold(backend, *w)
    act, out, again = put(backend, x, F32), backend.alloc(4 * lanes * rows), backend.alloc(4 * lanes * rows)
    backend.mx4_mat_mat_dev(held, act, F32, cols, lanes, out, F32, rows)
    first = out.get(np.float32, lanes * rows).reshape(lanes, rows)
    x2 = x.copy()
    x2[1::2] = 1e30
    other = put(backend, x2, F32)
    backend.mx4_mat_mat_dev(held, other, F32, cols, lanes, again, F32, rows)
    assert np.array_equal(again.get(np.float32, lanes * rows).reshape(lanes, rows)[0::2], first[0::2])
    for _ in range(3):
        backend.mx4_mat_mat_dev(held, act, F32, cols, lanes, again, F32, rows)
        assert np.array_equal(again.get(np.float32, lanes * rows).reshape(lanes, rows), first)
    close(held, act, other, out, again)


@pytest.mark.parametrize("lanes", [1, 6, 33, 140])
def test_recorded(backend, lanes):
    """Laid, read back and multiplied in a recording, replayed over new inputs among eager calls."""
    cols, rows = 352, 90
    rng = np.random.default_rng(lanes)
    w = sheet(rng, rows, cols)
    held, store = hold(backend, *w), backend.mx4(lanes, cols)
    x = backend.alloc(4 * lanes * cols)
    outs = [backend.alloc(4 * lanes * rows) for _ in range(2)]
    back = backend.alloc(4 * lanes * cols)

    def calls():
        backend.mx4_lay_dev(store, 0, lanes, x, F32, cols)
        backend.mx4_read_dev(store, 0, lanes, back, F32, cols)
        backend.mx4_mat_mat_dev(held, back, F32, cols, lanes, outs[0], F32, rows)
        backend.mx4_mat_mx4_dev(held, store, 0, lanes, outs[1], F32, rows)

    def result():
        backend.sync()
        return [o.get(np.float32, lanes * rows) for o in outs]

    x.put(rng.normal(size=(lanes, cols)).astype(np.float32))
    calls()
    backend.record_begin()
    calls()
    replay = backend.record_end()
    try:
        for _ in range(4):
            x.put(rng.normal(size=(lanes, cols)).astype(np.float32))
            calls()
            want = result()
            for o in outs:
                o.put(np.zeros(lanes * rows, np.float32))
            backend.replay_run(replay)
            got = result()
            assert all(np.array_equal(a, b) for a, b in zip(want, got))
            assert np.abs(got[0] - got[1]).max() <= 1e-4 * np.abs(got[1]).max()
    finally:
        backend.replay_free(replay)
    close(held, store, x, back, *outs)


@pytest.mark.parametrize("lanes", [1, 5, 16])
def test_a_head_recorded(backend, lanes):
    """A sheet past the caches' reach, replayed over new lanes among eager calls of others."""
    cols, rows = 1760, 32776
    rng = np.random.default_rng(lanes)
    w = sheet(rng, rows, cols)
    held, x, out = hold(backend, *w), backend.alloc(4 * lanes * cols), backend.alloc(4 * lanes * rows)
    small = hold(backend, w[0][:40], w[1][:40])

    def call():
        backend.mx4_mat_mat_dev(held, x, F32, cols, lanes, out, F32, rows)

    x.put(rng.normal(size=(lanes, cols)).astype(np.float32))
    call()
    backend.record_begin()
    call()
    replay = backend.record_end()
    try:
        for _ in range(3):
            host = rng.normal(size=(lanes, cols)).astype(np.float32)
            x.put(host)
            call()
            want = out.get(np.float32, lanes * rows)
            backend.mx4_mat_mat_dev(small, x, F32, cols, 1, out, F32, 40)
            backend.replay_run(replay)
            assert np.array_equal(out.get(np.float32, lanes * rows), want)
        exact = host.astype(np.float64) @ mx.values(w[0][:200], w[1][:200]).T
        got = want.reshape(lanes, rows)[:, :200]
        assert (np.abs(got - exact) <= bar(host.astype(np.float64), mx.values(w[0][:200], w[1][:200]), F32, F32, exact)).all()
    finally:
        backend.replay_free(replay)
    close(held, small, x, out)


def test_quantised_round_trip_of_what_was_read(backend):
    """Rows read back lie where they lay: laying them again changes nothing."""
    rng = np.random.default_rng(1)
    rows, cols = 60, 640
    x = put(backend, rng.normal(size=(rows, cols)), F32)
    a, b, back = backend.mx4(rows, cols), backend.mx4(rows, cols), backend.alloc(4 * rows * cols)
    backend.mx4_lay_dev(a, 0, rows, x, F32, cols)
    backend.mx4_read_dev(a, 0, rows, back, F32, cols)
    backend.mx4_lay_dev(b, 0, rows, back, F32, cols)
    values = []
    for s in (a, b):
        code, scale = s.buffers[0].get(np.uint8, rows * cols // 2), s.buffers[1].get(np.uint8, rows * cols // 32)
        values.append(mx.values(code.reshape(rows, -1), scale.reshape(rows, -1)))
    assert np.array_equal(*values)
    close(a, b, x, back)


@pytest.mark.parametrize("lanes", [1, 5, 40])
def test_rows_past_32_bits(backend, lanes):
    """Rows 16 MiB apart, the last beyond 4 GiB, of a sheet, of lanes and of outputs."""
    rows, cols, far = 272, 96, 1 << 24
    rng = np.random.default_rng(lanes)
    w, a = sheet(rng, rows, cols), sheet(rng, rows, cols)
    code, scale = backend.alloc(rows * far), backend.upload(w[1])
    for n in range(rows):
        code.put(w[0][n], n * far)
    held = backend.mx4(rows, cols, code, scale, far, cols // 32)
    x, wv = mx.bf16(rng.normal(size=(rows, cols))), mx.values(*w)
    at = rows - lanes  # the last rows
    # the sheet's, and as microscaled lanes
    act, out = put(backend, x[:lanes], F32), backend.alloc(4 * lanes * rows)
    backend.mx4_mat_mat_dev(held, act, F32, cols, lanes, out, F32, rows)
    want = x[:lanes].astype(np.float64) @ wv.T
    assert (np.abs(get(out, (lanes, rows), F32) - want) <= bar(x[:lanes], wv, F32, F32, want)).all()
    other = hold(backend, *a)
    backend.mx4_mat_mx4_dev(other, held, at, lanes, out, F32, rows)
    av = mx.values(*a)
    want = wv[at:] @ av.T
    assert (np.abs(get(out, (lanes, rows), F32) - want) <= bar(wv[at:], av, None, F32, want)).all()
    # laid and read there
    backend.mx4_lay_dev(held, at, lanes, act, F32, cols)
    back = backend.alloc(4 * lanes * cols)
    backend.mx4_read_dev(held, at, lanes, back, F32, cols)
    laid = mx.quantise(x[:lanes])
    assert np.array_equal(get(back, (lanes, cols), F32), mx.values(mx.pack(laid[0]), laid[1]).astype(np.float32))
    close(out, back, act, scale)
    # lanes and outputs as far apart: the same memory, as floats
    wide = far // 4
    for n in range(rows):
        code.put(x[n], n * far)
    backend.mx4_mat_mat_dev(other, At(code, at * far), F32, wide, lanes, At(code, at * far + (1 << 20)), F32, wide)
    want = x[at:].astype(np.float64) @ av.T
    got = np.stack([code.get(np.float32, rows, (at + m) * far + (1 << 20)) for m in range(lanes)])
    assert (np.abs(got - want) <= bar(x[at:], av, F32, F32, want)).all()
    close(code, other)


def test_unaligned_lanes(backend):
    """Lanes and outputs at the least alignment of their types."""
    rng = np.random.default_rng(2)
    lanes, rows, cols = 21, 70, 320
    w = sheet(rng, rows, cols)
    held = hold(backend, *w)
    x = mx.bf16(rng.normal(size=(lanes, cols)))
    wv = mx.values(*w)
    want = x.astype(np.float64) @ wv.T
    for kind, width in ((F32, 4), (BF16, 2)):
        for shift in (1, 2, 3):
            act, out = backend.alloc(width * (lanes * cols + 8)), backend.alloc(width * (lanes * rows + 8))
            act.put(mx.bf16_bits(x) if kind == BF16 else x, shift * width)
            backend.mx4_mat_mat_dev(held, At(act, shift * width), kind, cols, lanes, At(out, shift * width), kind, rows)
            got = get(out, (lanes, rows), kind, shift * width)
            assert (np.abs(got - want) <= bar(x, wv, kind, kind, want)).all()
            close(act, out)
    close(held)


def test_refused_on_the_gpu(backend):
    lib, desk = backend.lib, ctypes.byref(backend.desk)
    s = backend.mx4(4, 64)
    assert lib.igl_mx4_lay_dev(desk, ctypes.byref(s.rows), 0, 5, s.buffers[0].ptr, F32, 64) == native.IGL_FAIL_ARGUMENT
    assert lib.igl_desk_error_take(desk) == native.IGL_FAIL_ARGUMENT
    assert lib.igl_mx4_lay_dev(desk, ctypes.byref(s.rows), 0, 4, s.buffers[0].ptr, native.IGL_STORE_F16, 64) == native.IGL_FAIL_SUPPORT
    assert lib.igl_desk_error_take(desk) == native.IGL_FAIL_SUPPORT
    close(s)
