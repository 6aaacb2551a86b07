"""The bars of the tests that every value is held, on the CPU: what the model of the terms gives passes them, and
with a term less it does not; and that those tests reach every form of a product."""
import numpy as np
import pytest

import mx4_held as held
import mx4_oracle as mx
from test_mx4_host import lib, so  # noqa: F401
from test_mx4_terms import cut


def model(x, terms):
    return cut(x.astype(np.float64).reshape(-1, 32), terms)[0].reshape(x.shape)


@pytest.mark.parametrize("gate", [mx.gelu, mx.silu])
@pytest.mark.parametrize("lanes", [1, 40])
def test_hidden_values(lanes, gate):
    x, _, _, h = held.hidden_case(lanes, 512, gate)
    assert np.array_equal(model(x, 3), x)  # the lanes are not what is seen here: three terms hold them
    for terms in (5, 4, 3):
        assert (np.abs(model(h.astype(np.float32), terms) - h) <= held.hidden_bar(h)).all() == (terms == 5)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("lanes,cols", sorted({(f[0], f[2]) for f in held.FORMS if f[0] * f[2] < 1 << 18}))
def test_values(lanes, cols, bf16):
    x = held.wide_lanes(lanes, cols, bf16)
    for terms in (5, 4, 3):
        assert (np.abs(model(x, terms) - x) <= held.value_bar(x, bf16)).all() == (terms == 5)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("gate", [mx.gelu, mx.silu])
@pytest.mark.parametrize("lanes,width", [(1, 512), (40, 512)])
def test_up_values(lanes, width, bf16, gate):
    x, a, b = held.up_case(lanes, width, bf16)
    g = gate(x.astype(np.float64))[:, a]
    for terms in (5, 4, 3):
        got = model((g * model(x, terms)[:, b]).astype(np.float32), 5)
        assert (np.abs(got - g * x[:, b]) <= held.up_bar(x, a, b, bf16, gate)).all() == (terms == 5)


def test_outliers():
    """bf16 lanes beside channels 4000 times theirs, as three, four and five terms hold them: a bar of the sums that
    the row reads, 2^-16 of them, sees either of the first."""
    x, loud = held.outlier_lanes(40, 512, True, 4096)
    rest = np.setdiff1d(np.arange(512), loud)
    for terms in (5, 4, 3):
        off = np.abs(model(x, terms) - x)[:, rest].sum(1)
        assert (off <= 2.0 ** -16 * np.abs(x[:, rest]).sum(1)).all() == (terms == 5)


@pytest.mark.parametrize("case", held.FORMS + held.FAR)
def test_forms(lib, case):  # noqa: F811
    """Which form every case takes, so that a change of the rule cannot leave one without tests."""
    lanes, rows, cols = case[:3]
    for kind, form in zip((5, 3, 0), case[3:]):
        single = lib.planmx_single(rows, cols, lanes, kind)
        assert single if form == held.STEP else not single and lib.planmx_form(rows, cols, lanes, kind) == form


def test_experts_forms(lib):  # noqa: F811
    for lanes, hidden, inner, places in held.BLOCKS + held.UPS:
        assert {lib.planmx_experts(1, hidden, inner, lanes, 1, bf16) for bf16 in (0, 1)} == {places}
    for case in held.SLOTS + held.CHOICES:
        assert [lib.planmx_experts(*case[:3], case[4], case[3], bf16) for bf16 in (0, 1)] == list(case[5:]), case


def test_every_form_is_there(lib):  # noqa: F811
    for i, forms in enumerate(({-1, 0, 1, 2, 3, 5}, {-1, 0, 1, 2, 3, 4, 5}, {0, 2, 3})):
        assert {f[3 + i] for f in held.FORMS} == forms
        slices = {lib.planmx_slices(f[1], f[2], f[0], 64 if i == 2 else 32, 256) > 1 for f in held.FORMS if f[3 + i] == held.SMALL}
        assert slices == {False, True}
