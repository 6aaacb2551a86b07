"""GPU: which of two experts comes first where their scores are one number in 64 bits and their logits are not: without
a bias and groups the larger logit, with either the lower index."""
import numpy as np
import pytest

from test_gpu_experts import check_route

pytestmark = pytest.mark.gpu


def saturated(lanes, count):
    """Sigmoid scores that are all 1."""
    rng = np.random.default_rng(count)
    return rng.permuted(np.tile(40 + 0.25 * np.arange(count, dtype=np.float32), (lanes, 1)), axis=1)


def vanished(lanes, count):
    """Softmax scores that are all 0, but for the largest's 1."""
    x = -1000 - saturated(lanes, count)
    x[np.arange(lanes), np.arange(lanes) % count] = 0
    return x


@pytest.mark.parametrize("lanes", [1, 3, 2100])
@pytest.mark.parametrize("count", [12, 64, 160, 256, 1000])
@pytest.mark.parametrize("score,logits", [("sigmoid", saturated), ("softmax", vanished)])
def test_scores_that_are_equal(backend, lanes, count, score, logits):
    x = logits(lanes, count)
    check_route(backend, x, {"top": 6, "score": score})
    check_route(backend, x, {"top": 6, "score": score}, np.zeros(count, np.float32))
    check_route(backend, x, {"top": 6, "score": score, "groups": 4, "kept": 2, "best": 2})


def test_the_two_orders_differ():
    """As the oracle has them."""
    import mx4_oracle as mx

    x = np.array([[40, 41, 3, 42]], np.float32)
    assert mx.route(x, {"top": 3, "score": "sigmoid"})[0].tolist() == [[3, 1, 0]]
    assert mx.route(x, {"top": 3, "score": "sigmoid"}, np.zeros(4, np.float32))[0].tolist() == [[0, 1, 3]]
