"""GPU: every value is held, through every form of a product and of the experts' blocks.  Sheets with one code a row
pass values through (mx4_held); their bars fail with a term less (test_mx4_held)."""
import numpy as np
import pytest

import mx4_held as held
import mx4_oracle as mx
from igllm_amd import native
from test_gpu_mx4 import BF16, F32, close, get, hold, put

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lanes,width", [(1, 512), (5, 96), (40, 512), (600, 2048), (1200, 2048)])  # a step; tiles of 16, 32, 64
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
