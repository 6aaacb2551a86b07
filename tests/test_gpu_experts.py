"""GPU parity of the choice of experts and of the experts' feed-forward blocks,
against their definitions in 64 bits (mx4_oracle).

Picks are equal.  A weight is formed in 64 bits and rounded once: 2^-24 of it, and
2^-48 for the 64-bit exponentials.

Bar of an output: a product over `cols` columns is off by
p = (held + 16 adds an instruction) of its sum of magnitudes (test_gpu_mx4); the
gate's exponential and quotient by 2^-20 of its result; so h by p of gate_up times
|gate'| and the other factor, the down product by p of its own, weight and sum over
`top` choices by 2^-24 each.  With `reach` the sum of the magnitudes all of that
passes through (mx4_oracle.experts), the output is off by (p1 + p2 + 2^-19) reach;
bf16 lanes keep h to 2^-14 of a group's largest, and an output in bf16 adds 2^-8.
"""
import numpy as np
import pytest

import mx4_oracle as mx
from igllm_amd import native
from test_gpu_mx4 import BF16, F32, TERMS, At, close, get, hold, put, sheet

pytestmark = pytest.mark.gpu


# ---- the choice ----------------------------------------------------------------

def rule_of(count, r):
    return native.Route(count, r["top"], native.IGL_ROUTE_SOFTMAX if r["score"] == "softmax" else native.IGL_ROUTE_SIGMOID,
                        r.get("groups", 1), r.get("kept", 1), r.get("best", 1), r.get("renorm", 1), r.get("scale", 1.0))


def check_route(backend, logits, r, bias=None, gain=None, pad=0):
    lanes, count = logits.shape
    wide = np.full((lanes, count + pad), 1e9, np.float32)
    wide[:, :count] = logits
    bufs = [backend.upload(wide)] + [backend.upload(v) if v is not None else None for v in (bias, gain)]
    pick = backend.upload(np.full((lanes + 1, r["top"]), -7, np.int32))
    weight = backend.upload(np.full((lanes + 1, r["top"]), 7.5, np.float32))
    backend.route_dev(rule_of(count, r), bufs[0], count + pad, lanes, bufs[1], bufs[2], pick, weight)
    got = pick.get(np.int32, (lanes + 1) * r["top"]).reshape(lanes + 1, -1)
    gw = weight.get(np.float32, (lanes + 1) * r["top"]).reshape(lanes + 1, -1)
    assert (got[lanes] == -7).all() and (gw[lanes] == 7.5).all()
    want, ww = mx.route(logits, r, bias, gain)
    assert np.array_equal(got[:lanes], want)
    assert (np.abs(gw[:lanes] - ww) <= (2.0 ** -24 + 2.0 ** -48) * np.abs(ww) + 2.0 ** -149).all()
    close(*[b for b in bufs if b], pick, weight)


RULES = [({"top": 1, "score": "softmax"}, 1), ({"top": 1, "score": "softmax"}, 7), ({"top": 8, "score": "softmax"}, 128),
         ({"top": 5, "score": "softmax", "renorm": 0, "scale": 2.5}, 63), ({"top": 6, "score": "sigmoid"}, 65),
         ({"top": 8, "score": "sigmoid", "groups": 8, "kept": 4, "best": 2, "scale": 2.5}, 256),
         ({"top": 6, "score": "softmax", "groups": 8, "kept": 3, "best": 1, "renorm": 0}, 160),
         ({"top": 3, "score": "softmax", "groups": 5, "kept": 2, "best": 2}, 35),
         ({"top": 20, "score": "sigmoid", "groups": 3, "kept": 1, "best": 2}, 36),  # more than the kept group has
         ({"top": 64, "score": "sigmoid"}, 300), ({"top": 9, "score": "softmax"}, 1024),
         ({"top": 10, "score": "sigmoid", "groups": 64, "kept": 10, "best": 2}, 1024),
         ({"top": 4, "score": "softmax", "groups": 4, "kept": 4, "best": 2}, 4),  # groups of one
         ({"top": 30, "score": "softmax"}, 30), ({"top": 2, "score": "sigmoid", "groups": 2, "kept": 1}, 510)]


@pytest.mark.parametrize("r,count", RULES)
@pytest.mark.parametrize("lanes", [1, 3, 130])
@pytest.mark.parametrize("biased", [False, True])
def test_route(backend, r, count, lanes, biased):
    rng = np.random.default_rng(count + lanes)
    logits = (1.5 * rng.normal(size=(lanes, count))).astype(np.float32)
    bias = (0.1 * rng.normal(size=count)).astype(np.float32) if biased else None
    gain = rng.uniform(0.5, 2, size=count).astype(np.float32) if biased else None
    check_route(backend, logits, r, bias, gain, lanes % 2)


# four lanes of a batch a wave: up to 256 experts, a multiple of four, and sixteen choices and groups
MANY = RULES + [({"top": 16, "score": "sigmoid", "groups": 16, "kept": 9, "best": 2}, 256), ({"top": 1, "score": "sigmoid"}, 4),
                ({"top": 7, "score": "softmax", "groups": 7, "kept": 3, "best": 2}, 84),
                ({"top": 9, "score": "softmax", "groups": 2, "kept": 1, "best": 1, "renorm": 0}, 20)]


@pytest.mark.parametrize("r,count", MANY)
@pytest.mark.parametrize("biased", [False, True])
def test_route_of_many_lanes(backend, r, count, biased):
    rng = np.random.default_rng(count + 1)
    logits = (1.5 * rng.normal(size=(2051, count))).astype(np.float32)
    bias = (0.1 * rng.normal(size=count)).astype(np.float32) if biased else None
    gain = rng.uniform(0.5, 2, size=count).astype(np.float32) if biased else None
    check_route(backend, logits, r, bias, gain, 1)


@pytest.mark.parametrize("r,count", MANY)
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("times", [1, 35])
def test_route_of_equal_and_of_no_numbers(backend, r, count, biased, times):
    """Equal scores, masked experts, infinities and NaN: few values, many ties."""
    rng = np.random.default_rng(count)
    logits = rng.integers(-2, 3, size=(60, count)).astype(np.float32)
    masked = rng.random((60, count)) < np.linspace(0, 1, 60)[:, None]
    logits[masked] = -np.inf
    logits[20:30][rng.random((10, count)) < 0.3] = np.nan
    logits[30:34][rng.random((4, count)) < 0.1] = np.inf
    logits[34] = -np.inf
    logits[35] = np.nan
    logits[36] = np.inf
    logits[37] = 0
    logits[38] = -3.4e38
    bias = None
    if biased:
        bias = (0.25 * rng.integers(-1, 2, size=count)).astype(np.float32)
        bias[rng.random(count) < 0.1] = -np.inf
        bias[rng.random(count) < 0.1] = np.nan
    if r["score"] == "softmax":  # sums of unequal scores can be equal in one order of adding and not in another
        logits = np.where(np.isfinite(logits) & (logits > -3e38), 0, logits).astype(np.float32) if biased or r.get("groups", 1) > 1 else logits
    check_route(backend, np.tile(logits, (times, 1)), r, bias)


@pytest.mark.parametrize("lanes", [3, 2100])
@pytest.mark.parametrize("count", [9, 64, 200])
def test_route_of_zeros_of_both_signs(backend, count, lanes):
    """Equal numbers, the lowest index first."""
    rng = np.random.default_rng(count)
    logits = np.where(rng.random((lanes, count)) < 0.5, np.float32(-0.0), np.float32(0.0))
    bias = np.where(rng.random(count) < 0.5, np.float32(-0.0), np.float32(0.0))
    for score in ("softmax", "sigmoid"):
        check_route(backend, logits, {"top": 5, "score": score})
        check_route(backend, logits, {"top": 5, "score": score}, bias)


def test_route_next_to_each_other(backend):
    """Logits and biases one float apart fall as the reals do."""
    rng = np.random.default_rng(4)
    base = rng.uniform(0.5, 1.5, size=(100, 1)).astype(np.float32)
    logits = (base.view(np.int32) + rng.permuted(np.tile(np.arange(48, dtype=np.int32), (100, 1)), axis=1)).view(np.float32)
    for score, times in (("softmax", 1), ("sigmoid", 1), ("softmax", 21), ("sigmoid", 21)):
        logits = np.tile(logits[:100], (times, 1))
        check_route(backend, logits, {"top": 8, "score": score})
        bias = (np.float32(0.125).view(np.int32) + rng.permutation(48).astype(np.int32)).view(np.float32)
        check_route(backend, logits, {"top": 8, "score": score}, bias)
        check_route(backend, logits, {"top": 8, "score": score, "groups": 6, "kept": 2, "best": 2}, bias)


# ---- the blocks ----------------------------------------------------------------

class Block:
    """A layer's experts on the device and in 64 bits."""

    def __init__(self, backend, rng, count, hidden, inner, gate=native.IGL_GATE_GELU):
        # scales that keep outputs near one: levels have a variance of about 8
        low = [int(127 - round(np.log2(np.sqrt(8 * k)))) for k in (hidden, inner)]
        self.w = [sheet(rng, rows, cols, b - 1, b + 2)
                  for rows, cols, b in ((count * 2 * inner, hidden, low[0]), (count * hidden, inner, low[1]))]
        self.held = [hold(backend, *w) for w in self.w]
        self.set = backend.experts(*self.held, count, hidden, inner, gate)
        self.values = [mx.values(*w) for w in self.w]
        self.count, self.hidden, self.inner = count, hidden, inner
        self.gate = mx.gelu if gate == native.IGL_GATE_GELU else mx.silu

    def want(self, x, pick, weight):
        return mx.experts(x.astype(np.float64), *self.values, pick, weight, self.inner, self.gate)

    def tol(self, reach, kind, out_kind, want):
        held = 2.0 ** -23 if kind == F32 else 2.0 ** -12.5  # of a group's largest, in magnitudes of its values
        steps = -(-self.hidden // 128) + -(-self.inner // 128)
        tol = (2 * held + 16 * TERMS[kind] * steps * 2.0 ** -24 * 1.1 + 2.0 ** -19) * 8 * reach
        return tol + 2.0 ** -8 * (np.abs(want) + tol) if out_kind == BF16 else tol


def picks(rng, lanes, count, top, skew=1.0):
    score = rng.normal(size=(lanes, count)) + skew * rng.normal(size=(1, count))
    pick = np.argsort(-score, 1)[:, :top].astype(np.int32)
    weight = rng.uniform(0.1, 1, size=(lanes, top)).astype(np.float32)
    return pick, weight / weight.sum(1, keepdims=True)


def run(backend, block, x, pick, weight, kind, out_kind, pad=0):
    lanes, top = pick.shape
    hidden = block.hidden
    wide = np.full((lanes, hidden + pad), 9.0, np.float32)
    wide[:, :hidden] = x
    act = put(backend, wide, kind)
    out = put(backend, np.full((lanes + 1, hidden + pad), 7.5, np.float32), out_kind)
    p, w = backend.upload(pick), backend.upload(weight.astype(np.float32))
    backend.experts_dev(block.set, act, kind, hidden + pad, lanes, p, w, top, out, out_kind, hidden + pad)
    got = get(out, (lanes + 1, hidden + pad), out_kind)
    assert (got[lanes] == 7.5).all() and (got[:, hidden:] == 7.5).all()
    close(act, out, p, w)
    return got[:lanes, :hidden]


@pytest.mark.parametrize("count,hidden,inner,top,lanes", [
    (1, 32, 32, 1, 1), (4, 64, 96, 2, 1), (16, 256, 160, 4, 1), (32, 1536, 704, 8, 1), (8, 128, 64, 3, 2),
    (16, 320, 224, 2, 5), (8, 96, 128, 8, 7), (64, 160, 96, 6, 17), (5, 544, 288, 3, 40), (32, 256, 128, 4, 64),
    (3, 128, 160, 2, 150), (12, 288, 352, 4, 300), (2, 64, 32, 1, 700),
    # a token's longest rows; tiles of 32 and of 64 places
    (3, 64, 4096, 2, 2), (64, 96, 512, 4, 300), (40, 96, 1024, 3, 600)])
@pytest.mark.parametrize("kind,out_kind", [(F32, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("gate", [native.IGL_GATE_GELU, native.IGL_GATE_SILU])
def test_experts(backend, count, hidden, inner, top, lanes, kind, out_kind, gate):
    rng = np.random.default_rng(count + hidden + lanes)
    block = Block(backend, rng, count, hidden, inner, gate)
    x = rng.normal(size=(lanes, hidden)).astype(np.float32)
    x = mx.bf16(x) if kind == BF16 else x
    pick, weight = picks(rng, lanes, count, top)
    print("experts", count, hidden, inner, top, lanes, kind, out_kind, gate, flush=True)
    got = run(backend, block, x, pick, weight, kind, out_kind, lanes % 3)
    want, reach = block.want(x, pick, weight)
    assert (np.abs(got - want) <= block.tol(reach, kind, out_kind, want)).all()
    if out_kind == F32:  # the worst case is far from what random signs give
        rms = np.sqrt(np.mean(want ** 2))
        assert np.sqrt(np.mean((got - want) ** 2)) <= (2.0 ** -18 if kind == F32 else 2.0 ** -8) * rms
    close(*block.held)


@pytest.mark.parametrize("lanes", [2, 30, 150, 600])
def test_rows_apart(backend, lanes):
    """Weights whose rows have bytes between them, at odd places of scales."""
    count, hidden, inner, top = 5, 224, 160, 2
    rng = np.random.default_rng(lanes)
    block = Block(backend, rng, count, hidden, inner)
    apart = [hold(backend, *w, 16 * (i + 1), 3 - i) for i, w in enumerate(block.w)]
    x = mx.bf16(rng.normal(size=(lanes, hidden)))
    pick, weight = picks(rng, lanes, count, top)
    for kind in (F32, BF16):
        close_by = run(backend, block, x, pick, weight, kind, F32)
        own, block.set = block.set, backend.experts(*apart, count, hidden, inner)
        assert np.array_equal(run(backend, block, x, pick, weight, kind, F32), close_by)
        block.set = own
        want, reach = block.want(x, pick, weight)
        assert (np.abs(close_by - want) <= block.tol(reach, kind, F32, want)).all()
    close(*block.held, *apart)


@pytest.mark.parametrize("lanes", [1, 3, 30, 200])
def test_picks_of_every_kind(backend, lanes):
    """None, out of range, the same expert twice in a lane, all lanes at one expert."""
    count, hidden, inner, top = 6, 96, 64, 3
    rng = np.random.default_rng(lanes)
    block = Block(backend, rng, count, hidden, inner)
    x = rng.normal(size=(lanes, hidden)).astype(np.float32)
    for pick in (np.full((lanes, top), -1), np.full((lanes, top), 4), np.tile([2, -1, 2], (lanes, 1)),
                 np.tile([count, -2 ** 31, 2 ** 31 - 1], (lanes, 1)), rng.integers(-2, count + 2, size=(lanes, top))):
        pick = np.ascontiguousarray(pick, np.int32)
        weight = rng.normal(size=pick.shape).astype(np.float32)
        got = run(backend, block, x, pick, weight, F32, F32)
        want, reach = block.want(x, pick, weight)
        assert (np.abs(got - want) <= block.tol(reach, F32, F32, want)).all()
        none = ((pick < 0) | (pick >= count)).all(1)
        assert (got[none] == 0).all()
    close(*block.held)


@pytest.mark.parametrize("lanes", [2, 9, 100])
def test_lanes_that_hold_no_number(backend, lanes):
    """A lane with an infinity or a NaN, or such a weight, is one in its own row only."""
    count, hidden, inner, top = 4, 128, 96, 2
    rng = np.random.default_rng(lanes)
    block = Block(backend, rng, count, hidden, inner)
    x = rng.normal(size=(lanes, hidden)).astype(np.float32)
    pick, weight = picks(rng, lanes, count, top)
    want, reach = block.want(x, pick, weight)
    x[0, 5], weight[1, 1] = np.inf, np.nan
    got = run(backend, block, x, pick, weight, F32, F32)
    assert np.isnan(got[:2]).all()
    assert (np.abs(got - want) <= block.tol(reach, F32, F32, want))[2:].all()
    close(*block.held)


@pytest.mark.parametrize("lanes", [1, 4, 40, 130])
def test_a_layer_recorded(backend, lanes):
    """Router product, choice and experts together, recorded and replayed over new lanes among eager calls."""
    count, hidden, inner, top = 16, 256, 96, 4
    rng = np.random.default_rng(lanes)
    block = Block(backend, rng, count, hidden, inner)
    router = sheet(rng, count, hidden, 121, 124)
    held = hold(backend, *router)
    rule = rule_of(count, {"top": top, "score": "sigmoid", "groups": 4, "kept": 2, "best": 2})
    bias = (0.1 * rng.normal(size=count)).astype(np.float32)
    x, logits, b = backend.alloc(4 * lanes * hidden), backend.alloc(4 * lanes * count), backend.upload(bias)
    pick, weight, out = backend.alloc(4 * lanes * top), backend.alloc(4 * lanes * top), backend.alloc(4 * lanes * hidden)

    def calls():
        backend.mx4_mat_mat_dev(held, x, F32, hidden, lanes, logits, F32, count)
        backend.route_dev(rule, logits, count, lanes, b, None, pick, weight)
        backend.experts_dev(block.set, x, F32, hidden, lanes, pick, weight, top, out, F32, hidden)

    def result():
        backend.sync()
        return (logits.get(np.float32, lanes * count).reshape(lanes, -1), pick.get(np.int32, lanes * top).reshape(lanes, -1),
                weight.get(np.float32, lanes * top).reshape(lanes, -1), out.get(np.float32, lanes * hidden).reshape(lanes, -1))

    host = rng.normal(size=(lanes, hidden)).astype(np.float32)
    x.put(host)
    calls()
    backend.record_begin()
    calls()
    replay = backend.record_end()
    try:
        for _ in range(4):
            host = rng.normal(size=(lanes, hidden)).astype(np.float32)
            x.put(host)
            calls()
            eager = result()
            want_pick, want_weight = mx.route(eager[0], {"top": top, "score": "sigmoid", "groups": 4, "kept": 2, "best": 2}, bias)
            assert np.array_equal(eager[1], want_pick)
            assert (np.abs(eager[2] - want_weight) <= 2.0 ** -23 * np.abs(want_weight)).all()
            want, reach = block.want(host, eager[1], eager[2])
            assert (np.abs(eager[3] - want) <= block.tol(reach, F32, F32, want)).all()
            out.put(np.zeros(lanes * hidden, np.float32))
            pick.put(np.zeros(lanes * top, np.int32))
            backend.replay_run(replay)
            assert all(np.array_equal(a, c) for a, c in zip(eager, result()))
    finally:
        backend.replay_free(replay)
    close(*block.held, held, x, logits, b, pick, weight, out)


def test_two_desks_at_once(backend):
    """Two desks have their own workspaces."""
    from igllm_amd.backend import Backend

    count, hidden, inner, top, lanes = 8, 256, 128, 2, 50
    rng = np.random.default_rng(5)
    block = Block(backend, rng, count, hidden, inner)
    other = Backend(device=0)
    try:
        sides = []
        for be in (backend, other):
            x = rng.normal(size=(lanes, hidden)).astype(np.float32)
            pick, weight = picks(rng, lanes, count, top)
            bufs = [be.upload(v) for v in (x, pick, weight)] + [be.alloc(4 * lanes * hidden)]
            sides.append((be, x, pick, weight, bufs))
        for _ in range(10):
            for be, _, _, _, (x, p, w, out) in sides:
                be.experts_dev(block.set, x, F32, hidden, lanes, p, w, top, out, F32, hidden)
        for be, x, pick, weight, bufs in sides:
            be.sync()
            want, reach = block.want(x, pick, weight)
            got = bufs[3].get(np.float32, lanes * hidden).reshape(lanes, hidden)
            assert (np.abs(got - want) <= block.tol(reach, F32, F32, want)).all()
            close(*bufs)
    finally:
        other.close()
    close(*block.held)


def test_workspace_is_frozen_while_a_replay_lives(backend):
    """A call that needs more room than there is fails while a replay lives, and leaves its output."""
    from igllm_amd.backend import Backend, BackendError

    be = Backend(device=0)
    count, hidden, inner, top = 4, 64, 64, 2
    rng = np.random.default_rng(6)
    block = Block(be, rng, count, hidden, inner)
    try:
        x = rng.normal(size=(40, hidden)).astype(np.float32)
        pick, weight = picks(rng, 40, count, top)
        bufs = [be.upload(v) for v in (x, pick, weight)] + [be.upload(np.full((40, hidden), 7.5, np.float32))]
        args = bufs[0], F32, hidden
        be.experts_dev(block.set, *args, 2, bufs[1], bufs[2], top, bufs[3], F32, hidden)
        be.record_begin()
        be.experts_dev(block.set, *args, 2, bufs[1], bufs[2], top, bufs[3], F32, hidden)
        replay = be.record_end()
        with pytest.raises(BackendError):
            be.experts_dev(block.set, *args, 40, bufs[1], bufs[2], top, bufs[3], F32, hidden)
        be.sync()
        assert (bufs[3].get(np.float32, 40 * hidden).reshape(40, -1)[2:] == 7.5).all()
        be.replay_free(replay)
        be.experts_dev(block.set, *args, 40, bufs[1], bufs[2], top, bufs[3], F32, hidden)
        be.sync()
        got = bufs[3].get(np.float32, 40 * hidden).reshape(40, hidden)
        want, reach = block.want(x, pick, weight)
        assert (np.abs(got - want) <= block.tol(reach, F32, F32, want)).all()
        close(*bufs, *block.held)
    finally:
        be.close()
