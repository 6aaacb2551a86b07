"""GPU: what a product has to hold whatever form it takes (mx4_held.FORMS, whose forms test_mx4_held counts on the CPU):
ranges, neighbours, far rows, odd addresses, recordings; and experts' blocks of many slots and many choices.  Bars as
test_gpu_mx4's and test_gpu_experts', at a few of the rows where a sheet has many."""
import numpy as np
import pytest

import mx4_held as held
import mx4_oracle as mx
from test_gpu_experts import Block, picks, run
from test_gpu_mx4 import BF16, F32, At, bar, close, get, hold, put, sheet

pytestmark = pytest.mark.gpu

MX4 = "mx4"  # microscaled lanes
KINDS = pytest.mark.parametrize("kind", [F32, BF16, MX4])


def some(rows):
    return np.unique(np.concatenate([np.arange(min(rows, 40)), np.arange(max(rows - 20, 0), rows)]))


def near(got, x, w, rows, kind):
    """Outputs of the few rows against 64 bits; bf16 lanes to fp32 ones' bar."""
    at = some(rows)
    wv, v = mx.values(w[0][at], w[1][at]), x.astype(np.float64)
    want = v @ wv.T
    return (np.abs(got[:, at].astype(np.float64) - want) <= bar(v, wv, None if kind == MX4 else F32, F32, want)).all()


class Lanes:
    """Lanes of a kind on the device."""

    def __init__(self, backend, lanes, cols, kind):
        self.backend, self.kind, self.lanes, self.cols = backend, kind, lanes, cols
        self.buf = backend.mx4(lanes, cols) if kind == MX4 else backend.alloc((2 if kind == BF16 else 4) * lanes * cols)

    def new(self, rng):
        """Other values, as 64 bits have them."""
        if self.kind == MX4:
            code, scale = sheet(rng, self.lanes, self.cols)
            self.buf.buffers[0].put(code)
            self.buf.buffers[1].put(scale)
            return mx.values(code, scale)
        x = rng.normal(size=(self.lanes, self.cols)).astype(np.float32)
        self.set(x)
        return mx.bf16(x) if self.kind == BF16 else x

    def set(self, x):
        self.buf.put(mx.bf16_bits(mx.bf16(x)) if self.kind == BF16 else np.ascontiguousarray(x, np.float32))

    def product(self, rows_held, rows, out, out_kind=F32):
        if self.kind == MX4:
            self.backend.mx4_mat_mx4_dev(rows_held, self.buf, 0, self.lanes, out, out_kind, rows)
        else:
            self.backend.mx4_mat_mat_dev(rows_held, self.buf, self.kind, self.cols, self.lanes, out, out_kind, rows)


@pytest.mark.parametrize("case", held.FORMS)
@pytest.mark.parametrize("kind", [F32, BF16])
def test_range(backend, case, kind):
    """Lanes and sheets of every size: the smallest floats count as zero, the largest pass infinity as sums do."""
    lanes, rows, cols = case[:3]
    rng = np.random.default_rng(3)
    out = backend.alloc(4 * lanes * rows)
    for power, low in ((-140, 240), (-126, 180), (-126, 1), (-20, 60), (40, 127), (100, 127), (120, 1), (120, 60), (120, 140)):
        x = np.ldexp(rng.normal(size=(lanes, cols)), power).astype(np.float32)
        x[:, 32:64] = 0
        x = mx.bf16(x) if kind == BF16 else x
        w = sheet(rng, rows, cols, low, low + 4)
        rows_held, act = hold(backend, *w), put(backend, x, kind)
        print("range", case, kind, power, low, flush=True)
        backend.mx4_mat_mat_dev(rows_held, act, kind, cols, lanes, out, F32, rows)
        got = get(out, (lanes, rows), F32)
        at = some(rows)
        wv = np.abs(mx.values(w[0][at], w[1][at]))
        reach = np.abs(x.astype(np.float64)) @ wv.T
        want = x.astype(np.float64) @ mx.values(w[0][at], w[1][at]).T
        # beside the bar what lies below 2^-130 of lanes, and what an instruction's sums may lose below 2^-126
        tol = bar(x.astype(np.float64), mx.values(w[0][at], w[1][at]), F32, F32, want)
        tol = tol + 2.0 ** -130 * wv.sum(1) + 16 * 5 * -(-cols // 128) * 2.0 ** -126
        sure = reach < 2.0 ** 126
        assert (np.abs(got[:, at].astype(np.float64) - want) <= tol)[sure].all(), (power, low)
        assert (~np.isfinite(got[:, at]))[np.abs(want) > 2.0 ** 129].all()
        close(rows_held, act)
    close(out)


@pytest.mark.parametrize("case", held.FORMS)
@KINDS
def test_a_lane_among_others(backend, case, kind):
    """What a lane's neighbours hold does not change its bits, nor does calling again."""
    lanes, rows, cols = case[:3]
    rng = np.random.default_rng(lanes + rows)
    w = sheet(rng, rows, cols)
    rows_held, act = hold(backend, *w), Lanes(backend, lanes, cols, kind)
    out, again = backend.alloc(4 * lanes * rows), backend.alloc(4 * lanes * rows)
    x = act.new(rng)
    act.product(rows_held, rows, out)
    first = get(out, (lanes, rows), F32)
    assert near(first, x, w, rows, kind)
    for _ in range(3):
        act.product(rows_held, rows, again)
        assert np.array_equal(get(again, (lanes, rows), F32), first)
    if kind == MX4:
        scale = act.buf.buffers[1].get(np.uint8, lanes * cols // 32).reshape(lanes, -1)
        scale[1::2] = 220
        act.buf.buffers[1].put(scale)
    else:
        loud = x.copy()
        loud[1::2] = 1e30
        act.set(loud)
    act.product(rows_held, rows, again)
    assert np.array_equal(get(again, (lanes, rows), F32)[0::2], first[0::2])
    close(rows_held, act.buf, out, again)


@pytest.mark.parametrize("case", held.FORMS)
@pytest.mark.parametrize("kind,out_kind", [(F32, F32), (BF16, BF16), (BF16, F32), (F32, BF16)])
def test_odd_addresses(backend, case, kind, out_kind):
    """Lanes and outputs at the least alignment of their types, rows of odd strides; nothing else written."""
    lanes, rows, cols = case[:3]
    rng = np.random.default_rng(rows)
    w, wide, far = sheet(rng, rows, cols), cols + 3, rows + 1
    rows_held = hold(backend, *w, 16, 1)
    x = mx.bf16(rng.normal(size=(lanes, cols)))
    size, out_size = (2 if kind == BF16 else 4), (2 if out_kind == BF16 else 4)
    host = np.full((lanes, wide), 9.0, np.float32)
    host[:, :cols] = x
    act = backend.alloc(size * (lanes * wide + 8))
    for shift in (1, 3):
        act.put(mx.bf16_bits(host) if kind == BF16 else host, shift * size)
        out = put(backend, np.full(lanes * far + 16, 7.5, np.float32), out_kind)
        print("odd addresses", case, kind, out_kind, shift, flush=True)
        backend.mx4_mat_mat_dev(rows_held, At(act, shift * size), kind, wide, lanes, At(out, shift * out_size), out_kind, far)
        raw = get(out, (lanes * far + 16,), out_kind)
        got = raw[shift:shift + lanes * far].reshape(lanes, far)
        assert (raw[:shift] == 7.5).all() and (raw[shift + lanes * far:] == 7.5).all() and (got[:, rows:] == 7.5).all()
        at = some(rows)
        wv = mx.values(w[0][at], w[1][at])
        want = x.astype(np.float64) @ wv.T
        assert (np.abs(got[:, at] - want) <= bar(x.astype(np.float64), wv, F32, out_kind, want)).all()
        close(out)
    close(rows_held, act)


@pytest.mark.parametrize("case", held.FORMS)
@KINDS
def test_recorded(backend, case, kind):
    """Replayed over new lanes among eager calls of others, which take the workspace between."""
    lanes, rows, cols = case[:3]
    rng = np.random.default_rng(lanes * 3 + rows)
    w = sheet(rng, rows, cols)
    rows_held, act = hold(backend, *w), Lanes(backend, lanes, cols, kind)
    other = Lanes(backend, max(lanes // 2, 1), cols, F32)
    out, between = backend.alloc(4 * lanes * rows), backend.alloc(4 * lanes * rows)
    other.new(rng)
    act.new(rng)
    other.product(rows_held, rows, between)
    act.product(rows_held, rows, out)
    backend.record_begin()
    act.product(rows_held, rows, out)
    replay = backend.record_end()
    try:
        for _ in range(3):
            x = act.new(rng)
            act.product(rows_held, rows, out)
            want = get(out, (lanes, rows), F32)
            assert near(want, x, w, rows, kind)
            out.put(np.zeros(lanes * rows, np.float32))
            other.product(rows_held, rows, between)
            backend.replay_run(replay)
            backend.sync()
            assert np.array_equal(get(out, (lanes, rows), F32), want)
    finally:
        backend.replay_free(replay)
    close(rows_held, act.buf, other.buf, out, between)


@pytest.mark.parametrize("lanes,rows,cols,stride", [(*f[:3], s) for f, s in zip(held.FAR, held.STRIDES)])
@KINDS
def test_rows_past_32_bits(backend, lanes, rows, cols, stride, kind):
    """A sheet, its lanes and its outputs that each reach past 4 GiB."""
    rng = np.random.default_rng(lanes)
    reach = 9 << 29

    def apart(count, least, unit):
        return max(-(-reach // count // unit) * unit, -(-least // unit) * unit)

    far = stride or min(apart(rows, cols // 2, 16), 1 << 24)
    w = sheet(rng, rows, cols)
    code, scale = backend.alloc(rows * far), backend.upload(w[1])
    for n in range(rows):
        code.put(w[0][n], n * far)
    rows_held = backend.mx4(rows, cols, code, scale, far, cols // 32)
    out_far = apart(lanes, 4 * rows, 16)
    out = backend.alloc(lanes * out_far)
    print("past 32 bits", lanes, rows, cols, kind, far, out_far, flush=True)
    if kind == MX4:
        a = sheet(rng, lanes, cols)
        act_far = min(apart(lanes, cols // 2, 16), 1 << 24)
        act, act_scale = backend.alloc(lanes * act_far), backend.upload(a[1])
        for m in range(lanes):
            act.put(a[0][m], m * act_far)
        x = mx.values(*a)
        backend.mx4_mat_mx4_dev(rows_held, backend.mx4(lanes, cols, act, act_scale, act_far, cols // 32), 0, lanes, out, F32,
                                out_far // 4)
        close(act_scale)
    else:
        x, size = mx.bf16(rng.normal(size=(lanes, cols))), 2 if kind == BF16 else 4
        act_far = apart(lanes, size * cols, 16)
        act = backend.alloc(lanes * act_far)
        for m in range(lanes):
            act.put(mx.bf16_bits(x[m:m + 1]) if kind == BF16 else x[m], m * act_far)
        backend.mx4_mat_mat_dev(rows_held, act, kind, act_far // size, lanes, out, F32, out_far // 4)
    got = np.stack([out.get(np.float32, rows, m * out_far) for m in range(lanes)])
    assert near(got, x, w, rows, kind)
    close(code, scale, act, out)


# ---- experts ---------------------------------------------------------------------

@pytest.mark.parametrize("count,hidden,inner,top,lanes", [c[:5] for c in held.SLOTS])
@pytest.mark.parametrize("kind", [F32, BF16])
def test_many_slots(backend, count, hidden, inner, top, lanes, kind):
    """Slots past a wave's round (4096 of a workgroup) and past what a workgroup keeps (16384), in tiles of each size; a
    lane's experts unevenly liked, some lanes without."""
    rng = np.random.default_rng(count + lanes)
    block = Block(backend, rng, count, hidden, inner)
    x = mx.bf16(rng.normal(size=(lanes, hidden)))
    pick, weight = picks(rng, lanes, count, top)
    pick[rng.random(lanes) < 0.05] = -1
    print("slots", count, hidden, inner, top, lanes, kind, flush=True)
    got = run(backend, block, x, pick, weight, kind, F32)
    want, reach = block.want(x, pick, weight)
    assert (np.abs(got - want) <= block.tol(reach, F32, F32, want)).all()
    assert np.array_equal(run(backend, block, x, pick, weight, kind, F32), got)
    close(*block.held)


@pytest.mark.parametrize("count,hidden,inner,top,lanes", [c[:5] for c in held.CHOICES])
@pytest.mark.parametrize("kind", [F32, BF16])
def test_many_choices(backend, count, hidden, inner, top, lanes, kind):
    """More than eight experts a lane: a token's waves and the rows' sum take a second turn."""
    rng = np.random.default_rng(count + top)
    block = Block(backend, rng, count, hidden, inner)
    x = mx.bf16(rng.normal(size=(lanes, hidden)))
    pick, weight = picks(rng, lanes, count, top)
    pick[:, 3] = -1
    print("choices", count, hidden, inner, top, lanes, kind, flush=True)
    for out_kind in (F32, BF16):
        got = run(backend, block, x, pick, weight, kind, out_kind)
        want, reach = block.want(x, pick, weight)
        assert (np.abs(got - want) <= block.tol(reach, F32, out_kind, want)).all()
    close(*block.held)


BLOCKS = pytest.mark.parametrize("count,hidden,inner,top,lanes", [(16, 96, 160, 4, 1), (8, 224, 96, 3, 37), (5, 64, 2080, 2, 800)])


@BLOCKS
@pytest.mark.parametrize("kind,out_kind", [(F32, F32), (BF16, BF16), (BF16, F32), (F32, BF16)])
def test_experts_at_odd_addresses(backend, count, hidden, inner, top, lanes, kind, out_kind):
    """Lanes and outputs at the least alignment of their types, rows of odd strides; nothing else written."""
    rng = np.random.default_rng(lanes)
    block = Block(backend, rng, count, hidden, inner)
    wide, far = hidden + 3, hidden + 1
    x = mx.bf16(rng.normal(size=(lanes, hidden)))
    host = np.full((lanes, wide), 9.0, np.float32)
    host[:, :hidden] = x
    pick, weight = picks(rng, lanes, count, top)
    p, w = backend.upload(pick), backend.upload(weight.astype(np.float32))
    size, out_size = (2 if kind == BF16 else 4), (2 if out_kind == BF16 else 4)
    act = backend.alloc(size * (lanes * wide + 8))
    want, reach = block.want(x, pick, weight.astype(np.float32))
    for shift in (1, 3):
        act.put(mx.bf16_bits(host) if kind == BF16 else host, shift * size)
        out = put(backend, np.full(lanes * far + 16, 7.5, np.float32), out_kind)
        backend.experts_dev(block.set, At(act, shift * size), kind, wide, lanes, p, w, top, At(out, shift * out_size), out_kind, far)
        raw = get(out, (lanes * far + 16,), out_kind)
        got = raw[shift:shift + lanes * far].reshape(lanes, far)
        assert (raw[:shift] == 7.5).all() and (raw[shift + lanes * far:] == 7.5).all() and (got[:, hidden:] == 7.5).all()
        assert (np.abs(got[:, :hidden] - want) <= block.tol(reach, F32, out_kind, want)).all()
        close(out)
    close(*block.held, act, p, w)


@BLOCKS
@pytest.mark.parametrize("kind", [F32, BF16])
def test_two_recordings(backend, count, hidden, inner, top, lanes, kind):
    """An experts' call and a product, recorded apart over one workspace and replayed in turns over new lanes."""
    rng = np.random.default_rng(lanes + 1)
    block, w = Block(backend, rng, count, hidden, inner), sheet(rng, 2500, hidden)
    rows_held, act = hold(backend, *w), Lanes(backend, lanes, hidden, kind)
    out, sums = backend.alloc(4 * lanes * hidden), backend.alloc(4 * lanes * 2500)
    pick, weight = picks(rng, lanes, count, top)
    p, q = backend.upload(pick), backend.upload(weight.astype(np.float32))
    calls = (lambda: backend.experts_dev(block.set, act.buf, kind, hidden, lanes, p, q, top, out, F32, hidden),
             lambda: act.product(rows_held, 2500, sums))
    act.new(rng)
    for call in calls:
        call()
    replays = []
    for call in calls:
        backend.record_begin()
        call()
        replays.append(backend.record_end())
    try:
        for _ in range(3):
            x = act.new(rng)
            for call in calls:
                call()
            want = get(out, (lanes, hidden), F32), get(sums, (lanes, 2500), F32)
            exact, reach = block.want(x, pick, weight.astype(np.float32))
            assert (np.abs(want[0] - exact) <= block.tol(reach, F32, F32, exact)).all()
            out.put(np.zeros(lanes * hidden, np.float32))
            sums.put(np.zeros(lanes * 2500, np.float32))
            for replay in replays[::-1]:
                backend.replay_run(replay)
            backend.sync()
            assert np.array_equal(get(out, (lanes, hidden), F32), want[0]) and np.array_equal(get(sums, (lanes, 2500), F32), want[1])
    finally:
        for replay in replays:
            backend.replay_free(replay)
    close(*block.held, rows_held, act.buf, out, sums, p, q)


@BLOCKS
@pytest.mark.parametrize("kind", [F32, BF16])
def test_experts_of_no_numbers(backend, count, hidden, inner, top, lanes, kind):
    """A lane with an infinity or a NaN has NaN outputs, and so has one whose hidden values pass the largest float; the
    others have theirs."""
    rng = np.random.default_rng(lanes + 2)
    block = Block(backend, rng, count, hidden, inner)
    x = mx.bf16(rng.normal(size=(lanes, hidden)))
    pick, weight = picks(rng, lanes, count, top)
    want, reach = block.want(x, pick, weight)
    bad = np.arange(0, lanes, 4)
    x[bad[::3], hidden // 2], x[bad[1::3], 0] = np.inf, np.nan
    x[bad[2::3]] = mx.bf16(1e30 * x[bad[2::3]])
    got = run(backend, block, x, pick, weight, kind, F32)
    good = np.setdiff1d(np.arange(lanes), bad)
    assert np.isnan(got[bad]).all()
    assert (np.abs(got - want) <= block.tol(reach, F32, F32, want))[good].all()
    close(*block.held)
