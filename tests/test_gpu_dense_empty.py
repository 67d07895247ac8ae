"""Gradients of Nn.dense, each wanted alone, where an extent is 0."""
import numpy as np
import pytest

from tests.test_gpu_dense import arr, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def J():
    import jax4j_b200 as j
    return j


@pytest.mark.parametrize("shape,N", [((0, 3), 4), ((2, 0), 4), ((2, 3), 0), ((0, 0), 4), ((0, 3), 0), ((2, 0, 3), 5)],
                         ids=str)
@pytest.mark.parametrize("name", ["none", "tanh", "gelu"])
@pytest.mark.parametrize("dt", [np.float32, np.float64])
def test_each_gradient_alone(J, shape, N, name, dt):
    x, w, b, res, dy = make(1, shape, N, dt)
    X, W, B, R, DY = (arr(J, a) for a in (x, w, b, res, dy))
    for f, a in ((lambda a: J.Nn.dense(a, W, B, name, R), X), (lambda a: J.Nn.dense(X, a, B, name, R), W),
                 (lambda a: J.Nn.dense(X, W, a, name, R), B), (lambda a: J.Nn.dense(X, W, B, name, a), R)):
        y, pull = J.JAX.vjp(f, a)
        g, = pull(DY)
        assert g.shape() == a.shape() and g.dtype() == a.dtype()
        assert y.shape().dimensions() == dy.shape
        if a is R:
            np.testing.assert_array_equal(g.numpy(), dy)
        elif a is not B or not (len(dy) and shape[-1] == 0):  # a sum of no terms
            assert not g.numpy().any()
