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


@pytest.mark.parametrize("small", [True, False])
@pytest.mark.parametrize("name", ["dense", "group norm"])
def test_scan_and_its_gradients(J, monkeypatch, name, small):
    """A carry through five steps of a layer: eager, traced and recorded scans, and
    both gradients, are those of the steps written out."""
    from jax4j_b200 import layers as L
    monkeypatch.setattr(L, "SMALL_PRODUCT", L.SMALL_PRODUCT if small else 0)
    f = layers(J)[name]
    r = np.random.default_rng(7)
    x, c = r.standard_normal((5, 20, 32)).astype(np.float32), r.standard_normal((20, 32)).astype(np.float32)
    X, C = arr(J, x), arr(J, c)
    X1 = arr(J, x, 1)  # its slices lie off every 16-byte boundary

    def step(carry, xt):
        h = f(carry.add(xt))
        return h, h.tanh()

    def steps(carry, xs):
        ys = []
        for t in range(5):
            carry, y = step(carry, arr(J, xs.numpy()[t]))
            ys.append(y.numpy())
        return carry.numpy(), np.stack(ys)

    carry, ys = steps(C, X)
    for xs in (X, X1):
        out = J.Lax.scan(step, C, xs)
        np.testing.assert_array_equal(out.carry().numpy(), carry)
        np.testing.assert_array_equal(out.ys().numpy(), ys)
        traced = J.JAX.jit(lambda a: J.Lax.scan(step, C, a).ys())
        np.testing.assert_array_equal(traced(xs).numpy(), ys)
    loss = lambda cc, xx: J.Lax.scan(step, cc, xx).ys().sum()  # noqa: E731
    gc, gx = J.JAX.gradBoth(loss)(C, X)
    parts = [arr(J, x[t]) for t in range(5)]

    def written_out(*a):
        carry, total = a[0], None
        for t in range(5):
            carry, y = step(carry, a[1 + t])
            total = y.sum() if total is None else total.add(y.sum())
        return total

    _, pull = J.JAX.vjp(written_out, C, *parts)
    grads = pull(J.ConcreteNDArray.scalar(1.0))
    # the same products; a carry's two cotangents are added in either order
    np.testing.assert_allclose(gc.numpy(), grads[0].numpy(), rtol=1e-5, atol=1e-6)
    np.testing.assert_allclose(gx.numpy(), np.stack([g.numpy() for g in grads[1:]]), rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("name", ["dense", "group norm"])
def test_cond_takes_the_branch_and_its_gradient(J, name):
    f = layers(J)[name]
    x = arr(J, np.random.default_rng(8).standard_normal((3, 4, 32)).astype(np.float32))
    other = lambda a: a.mul(a)  # noqa: E731
    for yes in (1.0, 0.0):
        pred = J.ConcreteNDArray.scalar(yes)
        branch = f if yes else other
        net = lambda a: J.Lax.cond(pred, f, other, a)  # noqa: E731,B023
        np.testing.assert_array_equal(J.JAX.jit(net)(x).numpy(), branch(x).numpy())
        np.testing.assert_array_equal(J.JAX.grad(lambda a: net(a).tanh().sum())(x).numpy(),  # noqa: B023
                                      J.JAX.grad(lambda a: branch(a).tanh().sum())(x).numpy())  # noqa: B023


@pytest.mark.parametrize("name", ["dense", "group norm"])
def test_vjp_of_a_layer(J, name):
    """JAX.vjp of one layer -- its arguments once and in order, in another order,
    one of them twice, a closed-over weight, two outputs, an argument left out --
    against the gradient of the same loss; and inside a pmap."""
    r = np.random.default_rng(9)
    x, w = r.standard_normal((8, 32)).astype(np.float32), (r.standard_normal((32, 32)) / 6).astype(np.float32)
    v, dy = r.standard_normal(32).astype(np.float32), r.standard_normal((8, 32)).astype(np.float32)
    X, W, V, DY = (arr(J, a) for a in (x, w, v, dy))
    if name == "dense":
        f, args = (lambda a, b, c: J.Nn.dense(a, b, c, "silu")), (X, W, V)
    else:
        f, args = (lambda a, b, c: J.Nn.groupNorm(a, 4, b, c, activation="silu")), (X, V, V)

    def grads_of(fn, *at):  # through a longer Jaxpr
        return J.JAX.vjp(lambda *a: fn(*a).mul(DY).sum(), *at)[1](J.ConcreteNDArray.scalar(1.0))

    y, pull = J.JAX.vjp(f, *args)
    np.testing.assert_array_equal(y.numpy(), f(*args).numpy())
    want = [g.numpy() for g in grads_of(f, *args)]
    for _ in range(2):
        for g, e in zip(pull(DY), want):
            np.testing.assert_array_equal(g.numpy(), e)
    swapped = J.JAX.vjp(lambda c, b, a: f(a, b, c), *args[::-1])[1](DY)
    for g, e in zip(swapped, want[::-1]):
        np.testing.assert_array_equal(g.numpy(), e)
    np.testing.assert_array_equal(J.JAX.vjp(lambda a: f(a, *args[1:]), X)[1](DY)[0].numpy(), want[0])
    extra = J.JAX.vjp(lambda a, q, b, c: f(a, b, c), X, DY, *args[1:])[1](DY)
    assert not extra[1].numpy().any()
    np.testing.assert_array_equal(extra[2].numpy(), want[1])
    two, pull2 = J.JAX.vjp(lambda a, b, c: (f(a, b, c), a), *args)
    np.testing.assert_array_equal(two[1].numpy(), x)
    np.testing.assert_array_equal(pull2(DY, DY)[0].numpy(), (want[0] + dy))
    if name == "dense":
        twice = J.JAX.vjp(lambda a, b: J.Nn.dense(a, b, None, "silu", a), X, W)[1](DY)
        res = J.JAX.vjp(lambda a, b, c: J.Nn.dense(a, b, None, "silu", c), X, W, X)[1](DY)
        np.testing.assert_array_equal(twice[0].numpy(), res[0].numpy() + res[2].numpy())
        np.testing.assert_array_equal(twice[1].numpy(), res[1].numpy())
    for bad in ((), (X, X), (V,)):
        with pytest.raises(J.IllegalArgumentException, match="cotangent"):
            pull(*bad)

    def body(xs):
        local = [J.ConcreteNDArray(a.tensor(), a.shape()).to(xs.device()) for a in args[1:]]
        d = J.ConcreteNDArray(DY.tensor(), DY.shape()).to(xs.device())
        return J.Lax.psum(J.JAX.vjp(f, xs, *local)[1](d)[1])

    both = J.JAX.pmap(body, [J.Device(None), J.Device(None)])(arr(J, np.stack([x, x]))).numpy()
    np.testing.assert_array_equal(both, np.stack([want[1] + want[1]] * 2))
