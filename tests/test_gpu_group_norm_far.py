"""Group norm's gradients where a value of 0 would lie infinitely far from the mean
in standard deviations: rows behind a tile's last batch are not values."""
import numpy as np
import pytest

from tests.test_gpu_dense import arr

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def J():
    import jax4j_b200 as j
    return j


@pytest.mark.parametrize("act", ["none", "tanh", "sigmoid", "silu", "gelu"])
@pytest.mark.parametrize("S,C,G", [(1001, 24, 2), (130, 200, 1), (9000, 3, 3), (4, 5000, 2)])
def test_constant_groups(J, act, S, C, G):
    """x = 2^100 everywhere: its mean is exact, every xhat is 0, and eps = 1e-20
    makes one standard deviation 1e10 of x's own units away from 0 overflow.
    act'(0) is 1, 1, 1/4, 1/2 and 1/2, dy one value: sums of a few thousand equal
    numbers of few bits are exact, so all three gradients are."""
    slope = {"none": 1.0, "tanh": 1.0, "sigmoid": 0.25, "silu": 0.5, "gelu": 0.5}[act]
    x = np.full((2, S, C), 2.0 ** 100, np.float32)
    X, GM, BT, DY = arr(J, x), arr(J, np.ones(C, np.float32)), arr(J, np.zeros(C, np.float32)), arr(J, np.ones_like(x))
    y, pull = J.JAX.vjp(lambda a, g, b: J.Nn.groupNorm(a, G, g, b, eps=1e-20, activation=act), X, GM, BT)
    assert np.array_equal(y.numpy(), np.full_like(x, 0.5 if act == "sigmoid" else 0.0))
    dx, dg, db = (g.numpy() for g in pull(DY))
    np.testing.assert_array_equal(db, np.full(C, 2 * S * slope, np.float32))
    np.testing.assert_array_equal(dg, np.zeros(C, np.float32))
    np.testing.assert_array_equal(dx, np.zeros_like(x))
