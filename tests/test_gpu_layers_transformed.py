"""Nn.dense and Nn.groupNorm under transformations of transformations, loops and
branches, against the same computation without them."""
import numpy as np
import pytest

from tests.test_gpu_dense import arr

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def J():
    import jax4j_b200 as j
    return j


def layers(J):
    r = np.random.default_rng(5)
    W, B = arr(J, (r.standard_normal((32, 32)) / 6).astype(np.float32)), arr(J, r.standard_normal(32).astype(np.float32))
    G = arr(J, (1 + 0.2 * r.standard_normal(32)).astype(np.float32))
    return {"dense": lambda a: J.Nn.dense(a, W, B, "silu", a),
            "group norm": lambda a: J.Nn.groupNorm(a, 4, G, B, activation="gelu")}


@pytest.mark.parametrize("small", [True, False])
@pytest.mark.parametrize("name", ["dense", "group norm"])
def test_mapped_layers_under_jit_grad_and_vmap(J, monkeypatch, name, small):
    from jax4j_b200 import layers as L
    monkeypatch.setattr(L, "SMALL_PRODUCT", L.SMALL_PRODUCT if small else 0)
    f = layers(J)[name]
    x = np.random.default_rng(6).standard_normal((6, 8, 32)).astype(np.float32)
    X, X4 = arr(J, x), arr(J, x.reshape(2, 3, 8, 32))
    direct = f(X).numpy()
    loss = lambda g: lambda a: g(a).tanh().sum()  # noqa: E731
    want = J.JAX.grad(loss(f))(X).numpy()
    one, two = J.JAX.vmap(f), J.JAX.vmap(J.JAX.vmap(f))
    np.testing.assert_array_equal(one(X4).numpy().reshape(x.shape), direct)
    np.testing.assert_array_equal(J.JAX.jit(lambda a: one(a))(X4).numpy().reshape(x.shape), direct)
    np.testing.assert_array_equal(J.JAX.grad(loss(one))(X4).numpy().reshape(x.shape), want)
    X5 = arr(J, x.reshape(2, 3, 2, 4, 32))
    if name == "dense":
        np.testing.assert_array_equal(two(X5).numpy().reshape(x.shape), direct)
        np.testing.assert_array_equal(J.JAX.grad(loss(two))(X5).numpy().reshape(x.shape), want)
    else:  # samples of four positions
        halves = f(arr(J, x.reshape(12, 4, 32)))
        np.testing.assert_array_equal(two(X5).numpy().reshape(12, 4, 32), halves.numpy())
        np.testing.assert_array_equal(J.JAX.grad(loss(two))(X5).numpy().reshape(12, 4, 32),
                                      J.JAX.grad(loss(f))(arr(J, x.reshape(12, 4, 32))).numpy())
