"""GPU attention over the 4-bit ring at the ends of its numbers: scales, scores
and weights far from one another, against 64 bits."""
import numpy as np
import pytest

import cache4_oracle as c4
from test_gpu_cache4 import SCALE, attend, check, close, open_ring, ring_bytes

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
