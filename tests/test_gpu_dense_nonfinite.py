"""Infinities and NaN through the gradients of Nn.dense: they reach exactly the
values that depend on them, on the CUDA cores and on the tensor cores (where such
operands take the exact path), single CTAs and pairs."""
import numpy as np
import pytest

from tests.test_gpu_dense import arr, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def J():
    import jax4j_b200 as j
    return j


@pytest.mark.parametrize("small", [True, False])
@pytest.mark.parametrize("rows", [40, 300])
@pytest.mark.parametrize("where", ["x", "w", "dy", "all"])
def test_gradients(J, monkeypatch, small, rows, where):
    from jax4j_b200 import layers
    monkeypatch.setattr(layers, "SMALL_PRODUCT", layers.SMALL_PRODUCT if small else 0)
    x, w, b, _, dy = make(rows, (rows, 50), 60, residual=False)
    if where in ("x", "all"):
        x[3, 4], x[9, 0] = np.inf, np.nan
    if where in ("w", "all"):
        w[7, 11], w[20, 59] = -np.inf, np.nan
    if where in ("dy", "all"):
        dy[5, 6], dy[rows - 1, 30], dy[0, 6] = np.inf, np.nan, -np.inf
    _, pull = J.JAX.vjp(lambda p, q, c: J.Nn.dense(p, q, c), arr(J, x), arr(J, w), arr(J, b))
    got = [g.numpy().astype(np.float64) for g in pull(arr(J, dy))]
    x, w, dy = (a.astype(np.float64) for a in (x, w, dy))
    with np.errstate(invalid="ignore"):
        want = [dy @ w.T, x.T @ dy, dy.sum(0)]
        sizes = [np.abs(dy) @ np.abs(w).T, np.abs(x).T @ np.abs(dy), np.abs(dy).sum(0)]
    for g, v, size in zip(got, want, sizes):
        assert np.array_equal(np.isnan(g), np.isnan(v))
        inf = np.isinf(v)
        assert np.array_equal(np.isinf(g), inf) and np.array_equal(g[inf], v[inf])
        fin = np.isfinite(v)
        # sums of at most 300 terms: 300 roundings of half a step and the splits'
        assert np.all(np.abs(g[fin] - v[fin]) <= 310 * 2.0 ** -24 * size[fin])
