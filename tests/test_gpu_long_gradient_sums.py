"""The sums of the bias's, gamma's and beta's gradients over many rows: equal terms,
which round the same way at every addition, so a long row of additions shows.
The terms are values whose sum of so many in one FP32 row is off by thousands of
half steps U = 2^-24 (10174, 7383 and 2016 U)."""
import numpy as np
import pytest

U = 2.0 ** -24
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def J():
    import jax4j_b200 as j
    return j


def full(J, shape, value):
    import torch
    return J.ConcreteNDArray(torch.full(shape, float(value), device="cuda"), shape)


def off(got, want):
    return (got.tensor().double() / want - 1).abs().max().item()


def test_bias_of_a_long_column(J):
    """A warp adds at most 1024 rows, then 8 warps, a thirty-second of the 24415
    groups of rows and 32 lanes: under 1024 + 8 + 764 + 5 additions."""
    M, c = 200_000_000, np.float32(1.4160400)
    X, W, B = full(J, (M, 1), 0.5), full(J, (1, 1), 1.0), full(J, (1,), 1.0)
    _, pull = J.JAX.vjp(lambda b: J.Nn.dense(X, W, b), B)
    assert off(pull(full(J, (M, 1), c))[0], M * float(c)) <= 1801 * U


@pytest.mark.parametrize("D", [1, 4])
def test_parameters_over_many_samples(J, D):
    """A set of warps adds at most 1024 samples of its group; its sums then go over a
    thirty-second of the sets and 32 lanes."""
    B, C, c = 30000, 4800, np.float32(1.0751879)
    X = full(J, (B, C), 0.0)
    _, pull = J.JAX.vjp(lambda g, b: J.Nn.groupNorm(X, C // D, g, b), full(J, (C,), 1.0), full(J, (C,), 0.0))
    dg, db = pull(full(J, (B, C), c))
    assert off(db, B * float(c)) <= (1024 + 30 + 5) * U
    assert not dg.numpy().any()


def test_parameters_over_many_positions(J):
    """Groups held in registers: 64 positions in a row, then 128 such sums."""
    S, C, c = 8192, 8, np.float32(1.9624060)
    X = full(J, (1, S, C), 0.0)
    _, pull = J.JAX.vjp(lambda g, b: J.Nn.groupNorm(X, C, g, b), full(J, (C,), 1.0), full(J, (C,), 0.0))
    dg, db = pull(full(J, (1, S, C), c))
    assert off(db, S * float(c)) <= (64 + 128 + 8) * U
    assert not dg.numpy().any()
