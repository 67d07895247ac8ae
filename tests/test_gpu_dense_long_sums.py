"""Nn.dense where one of its sums has more terms than one cluster of CTAs adds in
short rows: the sum comes in parts, forward and in either gradient."""
import numpy as np
import pytest

from tests.layers_ref import U
from tests.test_gpu_dense import arr, check, make, reference, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def J():
    import jax4j_b200 as j
    return j


@pytest.mark.parametrize("M,K,N", [(1000000, 8, 8), (64, 1000000, 8), (16, 2000000, 4), (64, 8, 1000000)],
                         ids=["dw", "y", "y of 16 rows", "dx"])
def test_sums_of_one_value(J, M, K, N):
    """The worst sums there are: equal terms round the same way at every addition.
    A thread adds at most 1024 of them in a row and under 76 sums follow (16 CTAs
    or 8 warps and 16, a thirty-second of the parts, the shuffles), each within
    half a step of a running sum that is at most the result: 1100 U.  Rows of
    15625 terms and more lose 7.7e-5 (1300 U) and more here."""
    c = np.float32(1.1)
    X, W, DY = arr(J, np.full((M, K), c)), arr(J, np.full((K, N), c)), arr(J, np.ones((M, N), np.float32))
    y, pull = J.JAX.vjp(lambda a, b: J.Nn.dense(a, b), X, W)
    dx, dw = pull(DY)
    for got, terms, value in ((y, K, float(c) ** 2), (dx, N, float(c)), (dw, M, float(c))):
        want = terms * value
        assert np.abs(got.numpy().astype(np.float64) - want).max() <= 1100 * U * want, (terms, value)


LONG = [((100003, 24), 30), ((70, 150001), 33), ((5, 300000), 9), ((20, 7), 200001), ((40001, 130), 3)]


@pytest.mark.parametrize("shape,N", LONG, ids=[f"{'x'.join(map(str, s))}x{n}" for s, n in LONG])
@pytest.mark.parametrize("f64", [False, True], ids=["f32", "f64"])
def test_against_64_bits(J, shape, N, f64):
    x, w, b, res, dy = make(sum(shape) + N, shape, N, np.float64 if f64 else np.float32)
    check(run(J, x, w, b, "silu", res, dy), reference(x, w, b, "silu", res, dy, 2.0 ** -53 if f64 else U, False))


def test_only_one_gradient(J):
    x, w, _, _, dy = make(9, (50000, 20), 12, bias=False, residual=False)
    X, W, DY = arr(J, x), arr(J, w), arr(J, dy)
    both = J.JAX.vjp(lambda a, b: J.Nn.dense(a, b), X, W)[1](DY)
    dx = J.JAX.vjp(lambda a: J.Nn.dense(a, W), X)[1](DY)
    dw = J.JAX.vjp(lambda b: J.Nn.dense(X, b), W)[1](DY)
    np.testing.assert_array_equal(both[0].numpy(), dx[0].numpy())
    np.testing.assert_array_equal(both[1].numpy(), dw[0].numpy())


@pytest.mark.parametrize("shape,N", [((40000, 20), 12), ((30, 50000), 12)])
def test_recorded_and_on_another_stream(J, shape, N):
    """Two recorded steps with sums in parts, replayed one after the other on other values, and a side stream."""
    import torch
    from jax4j_b200.graphs import CapturedStep
    x, w, b, res, dy = make(12, shape, N)
    r = np.random.default_rng(13)

    def step(*a):
        y, pull = J.JAX.vjp(lambda p, q, s, t: J.Nn.dense(p, q, s, "gelu", t), *a[:4])
        return [y, *pull(a[4])[:3]]

    args = [arr(J, a) for a in (x, w, b, res, dy)]
    graphs = [CapturedStep(step, [J.ConcreteNDArray(a.tensor().clone(), a.shape()) for a in args]) for _ in range(2)]
    for _ in range(2):
        args = [arr(J, r.standard_normal(a.shape().dimensions()).astype(np.float32)) for a in args]
        want = [a.numpy() for a in step(*args)]
        for gr in graphs:
            for i, a in enumerate(args):
                gr.set_input(i, a)
        for out in [gr() for gr in graphs]:
            for a, v in zip(out, want):
                np.testing.assert_array_equal(a.numpy(), v)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step(*args)
        side.synchronize()
        for a, v in zip(other, want):
            np.testing.assert_array_equal(a.numpy(), v)
    for gr in graphs:
        gr.release()


@pytest.mark.parametrize("K", [1024, 4096, 8192])
def test_product_bias(J, K):
    """Positive operands, where the tensor cores' truncation cannot cancel: it is
    a chunk's (the adds of chunks round to nearest), and a layer's chunks are no
    longer than the plain product's, so its mean error is no larger either (5 % for
    the mean's own noise)."""
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(K)
    x, w = (torch.rand(*s, generator=g, device="cuda") for s in ((1024, K), (K, 1024)))
    want = x.double() @ w.double()
    arrays = [J.ConcreteNDArray(t, J.Shape(tuple(t.shape))) for t in (x, w)]
    bias = lambda y: abs(((y.tensor().view(1024, 1024).double() - want) / want).mean().item())  # noqa: E731
    assert bias(J.Nn.dense(*arrays)) <= 1.05 * bias(arrays[0].dot(arrays[1]))


def test_product_bias_under_3xtf32():
    import os
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-x", "tests/test_gpu_dense_long_sums.py", "-k",
                        "test_product_bias and not tf32"], env={**os.environ, "J4C_GEMM_SPLIT": "tf32"},
                       capture_output=True, text=True, timeout=600,
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-2000:]
