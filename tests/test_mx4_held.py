"""The bars of the tests that every value is held, on the CPU: what the model of the terms gives passes them, and
with a term less it does not."""
import numpy as np
import pytest

import mx4_held as held
import mx4_oracle as mx
from test_mx4_terms import cut


@pytest.mark.parametrize("gate", [mx.gelu, mx.silu])
@pytest.mark.parametrize("lanes", [1, 40])
def test_hidden_values(lanes, gate):
    x, _, _, h = held.hidden_case(lanes, 512, gate)
    # the lanes are not what is seen here: three terms hold them
    assert np.array_equal(cut(x.astype(np.float64).reshape(-1, 32), 3)[0].reshape(x.shape), x)
    h32 = h.astype(np.float32).astype(np.float64)
    for terms in (5, 4, 3):
        got = cut(h32.reshape(-1, 32), terms)[0].reshape(h.shape)
        assert (np.abs(got - h) <= held.hidden_bar(h)).all() == (terms == 5)
