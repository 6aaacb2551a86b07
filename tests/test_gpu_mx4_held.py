"""GPU: every value is held, through every form of a product and of the experts' blocks.  Sheets with one code a row
pass values through (mx4_held); their bars fail with a term less (test_mx4_held)."""
import numpy as np
import pytest

import mx4_held as held
import mx4_oracle as mx
from igllm_amd import native
from test_gpu_mx4 import BF16, F32, close, get, hold, put, sheet

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lanes,width", [b[:2] for b in held.BLOCKS])
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("gate", [native.IGL_GATE_GELU, native.IGL_GATE_SILU])
def test_hidden_values(backend, lanes, width, kind, gate):
    """gate(x_a) x_b passed through the down product, whatever the lanes' type."""
    x, a, b, h = held.hidden_case(lanes, width, mx.gelu if gate == native.IGL_GATE_GELU else mx.silu)
    gate_up = hold(backend, *held.passing(np.concatenate([a, b]), width))
    down = hold(backend, *held.passing(np.arange(width), width))
    experts = backend.experts(gate_up, down, 1, width, width, gate)
    act, out = put(backend, x, kind), backend.alloc(4 * lanes * width)
    pick, weight = backend.upload(np.zeros(lanes, np.int32)), backend.upload(np.ones(lanes, np.float32))
    backend.experts_dev(experts, act, kind, width, lanes, pick, weight, 1, out, F32, width)
    got = get(out, (lanes, width), F32)
    assert (np.abs(got - h) <= held.hidden_bar(h)).all()
    close(gate_up, down, act, out, pick, weight)


@pytest.mark.parametrize("case", held.FORMS)
@pytest.mark.parametrize("kind", [F32, BF16])
def test_values(backend, case, kind):
    lanes, rows, cols = case[:3]
    x = held.wide_lanes(lanes, cols, kind == BF16)
    at = np.random.default_rng(rows).permutation(np.arange(rows) % cols)
    rows_held, act, out = hold(backend, *held.passing(at, cols)), put(backend, x, kind), backend.alloc(4 * lanes * rows)
    print("values", case, kind, flush=True)
    backend.mx4_mat_mat_dev(rows_held, act, kind, cols, lanes, out, F32, rows)
    got = get(out, (lanes, rows), F32)
    assert (np.abs(got - x.astype(np.float64)[:, at]) <= held.value_bar(x, kind == BF16)[:, at]).all()
    close(rows_held, act, out)


@pytest.mark.parametrize("case", held.FORMS)
def test_microscaled_values(backend, case):
    lanes, rows, cols = case[:3]
    code, scale = sheet(np.random.default_rng(lanes), lanes, cols, 1, 250)
    at = np.random.default_rng(rows).permutation(np.arange(rows) % cols)
    rows_held, act, out = hold(backend, *held.passing(at, cols)), hold(backend, code, scale), backend.alloc(4 * lanes * rows)
    print("microscaled values", case, flush=True)
    backend.mx4_mat_mx4_dev(rows_held, act, 0, lanes, out, F32, rows)
    assert np.array_equal(get(out, (lanes, rows), F32), mx.values(code, scale)[:, at])
    close(rows_held, act, out)


@pytest.mark.parametrize("lanes,width", [b[:2] for b in held.UPS])
@pytest.mark.parametrize("kind", [F32, BF16])
def test_up_values(backend, lanes, width, kind):
    """What the experts' up products pass through."""
    x, a, b = held.up_case(lanes, width, kind == BF16)
    inner = width // 2
    gate_up = hold(backend, *held.passing(np.concatenate([a, b]), width))
    down = hold(backend, *held.passing(np.arange(width) % inner, inner))
    experts = backend.experts(gate_up, down, 1, width, inner)
    act, out = put(backend, x, kind), backend.alloc(4 * lanes * width)
    pick, weight = backend.upload(np.zeros(lanes, np.int32)), backend.upload(np.ones(lanes, np.float32))
    backend.experts_dev(experts, act, kind, width, lanes, pick, weight, 1, out, F32, width)
    want = mx.gelu(x.astype(np.float64)[:, a]) * x.astype(np.float64)[:, b]
    bar = held.up_bar(x, a, b, kind == BF16, mx.gelu)
    got = get(out, (lanes, width), F32)
    assert (np.abs(got - np.tile(want, 2)) <= np.tile(bar, 2)).all()
    close(gate_up, down, act, out, pick, weight)


@pytest.mark.parametrize("case", held.FORMS)
@pytest.mark.parametrize("times", [1000, 4096])
def test_outliers(backend, case, times):
    """bf16 lanes with a channel in 32 far above the others, at which the sheet's codes are zero: off by a small part
    of what the rows do read.  A lane of 2^-16 of the largest and more is exact, less is held to 2^-23 / 1.875 of the
    largest; sums are 16 adds an instruction of 32 or 128 columns and term (test_gpu_mx4)."""
    lanes, rows, cols = case[:3]
    x, loud = held.outlier_lanes(lanes, cols, True, times)
    code, scale = sheet(np.random.default_rng(rows), rows, cols)
    levels = mx.unpack(code)
    levels[:, loud] = 0
    code = mx.pack(levels)
    rows_held, act, out = hold(backend, code, scale), put(backend, x, BF16), backend.alloc(4 * lanes * rows)
    print("outliers", case, times, flush=True)
    backend.mx4_mat_mat_dev(rows_held, act, BF16, cols, lanes, out, F32, rows)
    got = get(out, (lanes, rows), F32)
    some = np.unique(np.concatenate([np.arange(min(rows, 40)), np.arange(max(rows - 20, 0), rows)]))
    w, v = mx.values(code[some], scale[some]), x.astype(np.float64)
    reach = np.abs(v) @ np.abs(w).T
    tol = held.value_bar(x, True) @ np.abs(w).T + 16 * 5 * -(-cols // 128) * 2.0 ** -24 * 1.1 * reach
    assert (np.abs(got[:, some] - v @ w.T) <= tol).all()
    close(rows_held, act, out)


@pytest.mark.parametrize("case", held.FORMS)
@pytest.mark.parametrize("kind", [F32, BF16])
def test_what_is_no_number(backend, case, kind):
    """A lane with an infinity or a NaN has NaN outputs and no other lane has; so has a sheet's group of scale 255."""
    lanes, rows, cols = case[:3]
    rng = np.random.default_rng(lanes)
    x = mx.bf16(rng.normal(size=(lanes, cols)))
    w = sheet(rng, rows, cols)
    w[1][rows // 2, cols // 64] = 255
    bad = np.arange(0, lanes, 3) if lanes > 1 else np.arange(0)
    x[bad, (37 * bad) % cols] = np.array([np.nan, np.inf, -np.inf], np.float32)[bad % 3 if lanes < 6 else (bad // 3) % 3]
    rows_held, act, out = hold(backend, *w), put(backend, x, kind), backend.alloc(4 * lanes * rows)
    print("no number", case, kind, flush=True)
    backend.mx4_mat_mat_dev(rows_held, act, kind, cols, lanes, out, F32, rows)
    got = get(out, (lanes, rows), F32)
    want = np.zeros((lanes, rows), bool)
    want[bad], want[:, rows // 2] = True, True
    assert np.array_equal(np.isnan(got), want) and np.isfinite(got[~want]).all()
    close(rows_held, act, out)
