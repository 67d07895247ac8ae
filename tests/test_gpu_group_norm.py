"""Nn.groupNorm and its gradients against their formulas in 64 bits."""
import numpy as np
import pytest

from tests.layers_ref import ACTS, U, act

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def J():
    import jax4j_b200 as j
    return j


def arr(J, x, offset=0):
    import torch
    x = np.ascontiguousarray(x)
    buf = torch.empty(x.size + offset, dtype=torch.from_numpy(x).dtype, device="cuda")
    buf[offset:] = torch.from_numpy(x.reshape(-1))
    return J.ConcreteNDArray(buf[offset:], J.Shape(x.shape))


DEPTH = 300  # additions that a value of any sum passes through, at most, at these sizes


def reference(x, G, gamma, beta, eps, name, dy, unit):
    """{name: (value, error bound of an evaluation with half step `unit`)}.
    unit scales the FLOAT32 bounds; FLOAT64 activations are CUDA's own, which
    are closer to their values than jmath's."""
    k = unit / U
    shape = x.shape
    B, C = shape[0], shape[-1]
    x, dy = x.astype(np.float64).reshape(B, -1, C), dy.astype(np.float64).reshape(B, -1, C)
    S = x.shape[1]
    gm = np.ones(C) if gamma is None else gamma.astype(np.float64)
    bt = np.zeros(C) if beta is None else beta.astype(np.float64)
    g = lambda t: t.reshape(B, S, G, C // G)  # noqa: E731
    over = lambda t, f: np.broadcast_to(f(g(t), axis=(1, 3), keepdims=True), (B, S, G, C // G)).reshape(B, S, C)  # noqa: E731
    mean = over(x, np.mean)
    d = x - mean
    var = over(d * d, np.mean)
    rstd = 1 / np.sqrt(var + eps)
    xhat = d * rstd
    # the mean is off by DEPTH units of mean |x|, a difference by that and one of its own rounding
    ed = unit * (DEPTH * over(np.abs(x), np.mean) + np.abs(d))
    # sum of squares: each difference's error twice, DEPTH of the sum; a root halves it
    erel = unit * (DEPTH + 6) / 2 + over(np.abs(d) * ed + ed * ed, np.mean) / (var + eps)
    ex = rstd * ed + np.abs(xhat) * (erel + 3 * unit)
    u = xhat * gm + bt
    eu = np.abs(gm) * ex + unit * (2 * np.abs(gm * xhat) + np.abs(u))
    y, slope, curve, ey, es = act(u, name)
    top = 1.2  # |act'| is at most 1.13
    out = {"y": (y, top * eu + k * ey + unit * np.abs(y))}
    du = dy * slope
    edu = np.abs(dy) * (curve * eu + k * es) + unit * np.abs(du)
    h = du * gm
    eh = np.abs(gm) * edu + unit * np.abs(h)
    m1, m2 = over(h, np.mean), over(h * xhat, np.mean)
    e1 = over(eh, np.mean) + unit * DEPTH * over(np.abs(h), np.mean)
    ehx = eh * np.abs(xhat) + np.abs(h) * ex + unit * np.abs(h * xhat)
    e2 = over(ehx, np.mean) + unit * DEPTH * over(np.abs(h * xhat), np.mean)
    dx = rstd * (h - m1 - xhat * m2)
    edx = rstd * (eh + e1 + np.abs(xhat) * e2 + np.abs(m2) * ex + 3 * unit * (np.abs(h) + np.abs(m1) + np.abs(xhat * m2))) \
        + np.abs(dx) * (erel + 3 * unit)
    out["dx"] = (dx, edx)
    out["dgamma"] = ((du * xhat).sum((0, 1)), (edu * np.abs(xhat) + np.abs(du) * ex).sum((0, 1))
                     + unit * DEPTH * np.abs(du * xhat).sum((0, 1)))
    out["dbeta"] = (du.sum((0, 1)), edu.sum((0, 1)) + unit * DEPTH * np.abs(du).sum((0, 1)))
    full = {"y": shape, "dx": shape, "dgamma": (C,), "dbeta": (C,)}
    return {n: (v.reshape(full[n]), 1.01 * e.reshape(full[n]) + 1e-37) for n, (v, e) in out.items()}


def run(J, x, G, gamma, beta, eps, name, dy, offset=0):
    args = [a for a in (x, gamma, beta) if a is not None]
    names = [n for n, a in (("dx", x), ("dgamma", gamma), ("dbeta", beta)) if a is not None]

    def f(*a):
        a = dict(zip(names, a))
        return J.Nn.groupNorm(a["dx"], G, a.get("dgamma"), a.get("dbeta"), eps=eps, activation=name)

    arrays = [arr(J, a, offset if i == 0 else 0) for i, a in enumerate(args)]
    y, pull = J.JAX.vjp(f, *arrays)
    eager = f(*arrays)
    np.testing.assert_array_equal(eager.numpy(), y.numpy())
    grads = pull(arr(J, dy, offset))
    again = pull(arr(J, dy, offset))
    for a, b in zip(grads, again):
        np.testing.assert_array_equal(a.numpy(), b.numpy())  # sums in a fixed order
    return {"y": y.numpy(), **{n: v.numpy() for n, v in zip(names, grads)}}


def check(got, ref):
    for n, v in got.items():
        value, tol = ref[n]
        assert v.shape == value.shape, n
        off = np.abs(v.astype(np.float64) - value) - tol
        assert np.all(off <= 0), (n, float(off.max()), int((off > 0).sum()), v.size)


# (shape, groups): held in registers by 1 to 32 warps, and cut into tiles (whole
# groups of a row, part of a row, parts of a group)
SHAPES = [((1, 1), 1), ((3, 7), 7), ((2, 16), 4), ((5, 3, 10), 5), ((4, 17, 24), 3), ((300, 2, 12), 2), ((2, 31, 48), 4),
          ((2, 8, 8, 64), 8), ((2, 100, 96), 6), ((3, 127, 32), 1), ((600, 4096), 1), ((3, 4095), 1), ((2, 5, 5000), 4),
          ((5, 8192), 1),
          ((1, 8193, 1), 1), ((2, 1000, 20), 2), ((3, 700, 250), 10), ((1, 9000), 1), ((2, 5, 12300), 3),
          ((2, 3, 40000), 4), ((1, 20000, 6), 2), ((2, 33, 33, 320), 32), ((1, 4097, 2052), 1), ((2, 9000, 40), 40), ((2, 100, 4096), 32), ((41, 1024, 512), 8)]


@pytest.mark.parametrize("shape,G", SHAPES, ids=[f"{'x'.join(map(str, s))}g{g}" for s, g in SHAPES])
@pytest.mark.parametrize("f64", [False, True], ids=["f32", "f64"])
def test_matches_the_formulas(J, shape, G, f64):
    if f64 and int(np.prod(shape)) > 4_000_000:
        pytest.skip("FLOAT64 at the smaller sizes")
    r = np.random.default_rng(sum(shape) + G)
    dt = np.float64 if f64 else np.float32
    C = shape[-1]
    name = ACTS[(sum(shape) + f64) % 6]
    x = (r.standard_normal(shape) * (0.5 + r.random(C)) + r.standard_normal(C)).astype(dt)
    gamma, beta = (1 + 0.3 * r.standard_normal(C)).astype(dt), (0.3 * r.standard_normal(C)).astype(dt)
    dy = r.standard_normal(shape).astype(dt)
    if name == "relu":  # away from the jump of its slope
        name = "silu"
    check(run(J, x, G, gamma, beta, 1e-5, name, dy), reference(x, G, gamma, beta, 1e-5, name, dy, 2.0 ** -53 if f64 else U))


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("shape,G", [((6, 5, 24), 3), ((2, 1500, 24), 3)])
@pytest.mark.parametrize("affine", ["both", "gamma", "beta", "none"])
def test_activations_and_optional_parameters(J, name, shape, G, affine):
    r = np.random.default_rng(7)
    C = shape[-1]
    x, dy = r.standard_normal(shape).astype(np.float32), r.standard_normal(shape).astype(np.float32)
    gamma = (1 + 0.3 * r.standard_normal(C)).astype(np.float32) if affine in ("both", "gamma") else None
    beta = (0.3 * r.standard_normal(C)).astype(np.float32) if affine in ("both", "beta") else None
    if name == "relu":
        # no pre-activation within rounding of 0, where either slope is right: dy is 0 there
        u = reference(x, G, gamma, beta, 1e-5, "none", dy, U)["y"]
        dy[np.abs(u[0]) <= u[1]] = 0
    check(run(J, x, G, gamma, beta, 1e-5, name, dy), reference(x, G, gamma, beta, 1e-5, name, dy, U))


@pytest.mark.parametrize("shape,G", [((6, 5, 24), 3), ((2, 1500, 24), 3), ((9, 4096), 1)])
@pytest.mark.parametrize("offset", [1, 2])
def test_unaligned_arrays(J, shape, G, offset):
    r = np.random.default_rng(8)
    C = shape[-1]
    x, dy = r.standard_normal(shape).astype(np.float32), r.standard_normal(shape).astype(np.float32)
    gamma, beta = r.standard_normal(C).astype(np.float32), r.standard_normal(C).astype(np.float32)
    check(run(J, x, G, gamma, beta, 1e-3, "gelu", dy, offset), reference(x, G, gamma, beta, 1e-3, "gelu", dy, U))


@pytest.mark.parametrize("shape,G", [((3, 40, 16), 4), ((2, 4000, 16), 4)])
def test_a_mean_far_from_zero(J, shape, G):
    """1000 standard deviations off: the bound grows only by the input's own rounding."""
    r = np.random.default_rng(9)
    x = (1000.0 + r.standard_normal(shape)).astype(np.float32)
    dy = r.standard_normal(shape).astype(np.float32)
    ref = reference(x, G, None, None, 0.0, "none", dy, U)
    got = run(J, x, G, None, None, 0.0, "none", dy)
    check(got, ref)
    # and the variance is right, not a difference of squares (1e6 * 2^-24 would be its error)
    assert abs(float(got["y"].reshape(shape[0], -1, G, 4).std((1, 3)).mean()) - 1) < 1e-3


@pytest.mark.parametrize("shape", [(2, 30, 8), (2, 5000, 8)])
def test_constant_groups_and_non_finite_values_stay_in_their_group(J, shape):
    r = np.random.default_rng(10)
    x = r.standard_normal(shape).astype(np.float32)
    x[0, :, :4] = 3.0
    clean = J.Nn.groupNorm(arr(J, x), 2, activation="tanh").numpy()
    assert np.all(clean[0, :, :4] == 0)
    x[1, 7, 1], x[1, 9, 2] = np.inf, np.nan
    y = J.Nn.groupNorm(arr(J, x), 2, activation="tanh").numpy()
    assert np.isnan(y[1, :, :4]).all()
    np.testing.assert_array_equal(y[0], clean[0])
    np.testing.assert_array_equal(y[1, :, 4:], clean[1, :, 4:])


def test_empty_batches(J):
    for shape in ((0, 4, 8), (3, 0, 8)):
        x, gamma = arr(J, np.zeros(shape, np.float32)), arr(J, np.ones(8, np.float32))
        y, pull = J.JAX.vjp(lambda a, b: J.Nn.groupNorm(a, 2, b), x, gamma)
        dx, dg = pull(arr(J, np.zeros(shape, np.float32)))
        assert y.numpy().shape == dx.numpy().shape == shape
        np.testing.assert_array_equal(dg.numpy(), np.zeros(8, np.float32))


@pytest.mark.parametrize("name", ACTS)
def test_gradients_against_differences(J, name):
    """FLOAT64 central differences: error eps^2 f'''/6 + 2^-53 |f| / eps."""
    r = np.random.default_rng(11)
    x, gamma, beta = r.standard_normal((2, 3, 8)), 1 + 0.3 * r.standard_normal(8), 0.3 * r.standard_normal(8)
    dy = r.standard_normal((2, 3, 8))

    def f(*a):
        return float((J.Nn.groupNorm(arr(J, a[0]), 2, arr(J, a[1]), arr(J, a[2]), activation=name).numpy() * dy).sum())

    got = run(J, x, 2, gamma, beta, 1e-5, name, dy)
    step = 1e-5
    for i, n in enumerate(("dx", "dgamma", "dbeta")):
        args = [x, gamma, beta]
        for at in np.ndindex(args[i].shape):
            up, down = ([a.copy() for a in args] for _ in range(2))
            up[i][at] += step
            down[i][at] -= step
            assert abs((f(*up) - f(*down)) / (2 * step) - got[n][at]) <= 1e-7, (n, at)


def test_inside_transformations(J):
    """grad, jit, checkpoint, pmap and vmap of chains with the layer agree with
    the layer called by itself."""
    r = np.random.default_rng(12)
    x, w = r.standard_normal((4, 6, 32)).astype(np.float32), r.standard_normal((32, 32)).astype(np.float32)
    gamma = (1 + 0.1 * r.standard_normal(32)).astype(np.float32)
    X, G = arr(J, x), arr(J, gamma)
    direct = J.Nn.groupNorm(X, 4, G, activation="silu")
    chain = lambda a: J.Nn.groupNorm(a.mul(a), 4, G, activation="silu").tanh().sum()  # noqa: E731
    np.testing.assert_array_equal(J.JAX.jit(lambda a: J.Nn.groupNorm(a, 4, G, activation="silu"))(X).numpy(), direct.numpy())
    g = J.JAX.grad(chain)(X).numpy()
    np.testing.assert_array_equal(J.JAX.grad(J.JAX.checkpoint(chain))(X).numpy(), g)
    ones = J.ConcreteNDArray.full(J.Shape(4, 6, 32), 1.0)
    t = J.Nn.groupNorm(X.mul(X), 4, G, activation="silu").tanh()
    dt = ones.sub(t.mul(t))
    _, pull = J.JAX.vjp(lambda a: J.Nn.groupNorm(a, 4, G, activation="silu"), X.mul(X))
    want = pull(dt)[0].mul(X).numpy() * 2
    np.testing.assert_allclose(g, want, rtol=1e-5, atol=1e-5 * np.abs(want).max())
    np.testing.assert_array_equal(J.JAX.vmap(lambda a: J.Nn.groupNorm(a, 4, G, activation="silu"))(
        X.reshape(J.Shape(2, 2, 6, 32))).numpy().reshape(4, 6, 32), direct.numpy())
    devs = [J.Device(None), J.Device(None)]
    halves = J.JAX.pmap(lambda a: J.Nn.groupNorm(a, 4, G.to(a.device()), activation="silu"), devs)(
        X.reshape(J.Shape(2, 2, 6, 32)))
    np.testing.assert_array_equal(halves.numpy().reshape(4, 6, 32), direct.numpy())
    gp = J.JAX.grad(lambda a: J.JAX.pmap(lambda b: J.Nn.groupNorm(b.mul(b), 4, activation="silu"), devs)(a).sum())(
        X.reshape(J.Shape(2, 2, 6, 32)))
    g1 = J.JAX.grad(lambda b: J.Nn.groupNorm(b.mul(b), 4, activation="silu").sum())(X)
    np.testing.assert_allclose(gp.numpy().reshape(4, 6, 32), g1.numpy(), rtol=1e-5, atol=1e-5)
    with pytest.raises(J.UnsupportedOperationException, match="forward-mode"):
        J.JAX.jvp(chain, X, X)


@pytest.mark.parametrize("shape", [(8, 4096), (2, 3000, 16)])
def test_recorded_and_on_another_stream(J, shape):
    """A captured forward and backward replays the eager results on new
    inputs while an eager pullback of the same arrays lives; two captures
    share no workspace."""
    import torch
    from jax4j_b200.graphs import CapturedStep
    r = np.random.default_rng(13)
    C = shape[-1]
    G = 1 if C > 100 else 2
    mk = lambda: arr(J, r.standard_normal(shape).astype(np.float32))  # noqa: E731
    gamma = arr(J, r.standard_normal(C).astype(np.float32))
    X, DY = mk(), mk()

    def step(x, gm, dy):
        y, pull = J.JAX.vjp(lambda a, b: J.Nn.groupNorm(a, G, b, activation="gelu"), x, gm)
        return [y, *pull(dy)]

    y, pull = J.JAX.vjp(lambda a, b: J.Nn.groupNorm(a, G, b, activation="gelu"), X, gamma)
    graphs = [CapturedStep(step, [mk(), gamma, mk()]) for _ in range(2)]
    for x, dy in ((X, DY), (mk(), mk())):
        want = [a.numpy() for a in step(x, gamma, dy)]
        outs = []
        for gr in graphs:
            gr.set_input(0, x)
            gr.set_input(2, dy)
        for gr in graphs:
            outs.append(gr())
        for out in outs:
            for a, b in zip(out, want):
                np.testing.assert_array_equal(a.numpy(), b)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step(x, gamma, dy)
        side.synchronize()
        for a, b in zip(other, want):
            np.testing.assert_array_equal(a.numpy(), b)
    first = [a.numpy() for a in pull(DY)]
    for a, b in zip(first, [v.numpy() for v in step(X, gamma, DY)[1:]]):
        np.testing.assert_array_equal(a, b)
    for gr in graphs:
        gr.release()
