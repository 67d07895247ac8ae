"""Nn.dense and its gradients against their formulas in 64 bits: the products
straight from the arrays (FLOAT32 and FLOAT64) and those from splits."""
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


def steps(K, tensor):
    """Error of a K-term product, in half steps of sum |a||b|.  CUDA cores: K
    roundings of mean zero, 8 standard deviations of their sum.  Tensor cores:
    48 truncating MMAs of a 256-deep chunk at 3.6e-8 (29 U; 3xTF32: 96 of them),
    the splits' 2^-22 (4 U) and K / 128 additions of chunks."""
    from jax4j_b200 import core
    return (29 if core.split_kind() == 1 else 58) + 4 + K / 128 + 8 if tensor else 8 * np.sqrt(K) + 8


def reference(x, w, bias, name, residual, dy, unit, tensor):
    k = unit / U
    x, w = x.astype(np.float64), w.astype(np.float64)
    lead = x.shape[:-1]
    x = x.reshape(int(np.prod(lead)), x.shape[-1])
    M, K = x.shape
    N = w.shape[1]
    dy = dy.astype(np.float64).reshape(M, N)
    b = np.zeros(N) if bias is None else bias.astype(np.float64)
    z = x @ w + b
    ez = unit * (steps(K, tensor) * (np.abs(x) @ np.abs(w)) + np.abs(z))
    y, slope, curve, ey, es = act(z, name)
    ey = 1.2 * ez + k * ey + unit * np.abs(y)
    out = y if residual is None else y + residual.astype(np.float64).reshape(M, N)
    res = {"y": (out, ey + unit * np.abs(out))}
    if residual is None and name in ("tanh", "sigmoid"):
        # the slope comes from the stored output: 1 - y^2, y (1 - y)
        es = (2 * np.abs(y) if name == "tanh" else 1.0) * ey / k + 2 * U
    dz = dy * slope
    edz = np.abs(dy) * (curve * ez + k * es) + unit * np.abs(dz)
    res["dx"] = (dz @ w.T, edz @ np.abs(w).T + unit * steps(N, tensor) * (np.abs(dz) @ np.abs(w).T))
    res["dw"] = (x.T @ dz, np.abs(x).T @ edz + unit * steps(M, tensor) * (np.abs(x).T @ np.abs(dz)))
    # column sums: a warp's rows, eight warps, the groups: under 32 + M / 8 additions
    res["dbias"] = (dz.sum(0), edz.sum(0) + unit * (32 + M / 8) * np.abs(dz).sum(0))
    res["dresidual"] = (dy.reshape(lead + (N,)), 0 * dy.reshape(lead + (N,)))
    res["y"] = tuple(a.reshape(lead + (N,)) for a in res["y"])
    res["dx"] = tuple(a.reshape(lead + (K,)) for a in res["dx"])
    return {n: (v, 1.01 * e + 1e-37) for n, (v, e) in res.items()}


def run(J, x, w, bias, name, residual, dy, offset=0):
    parts = {"dx": x, "dw": w, "dbias": bias, "dresidual": residual}
    names = [n for n, a in parts.items() if a is not None]
    arrays = [arr(J, parts[n], offset) for n in names]

    def f(*a):
        a = dict(zip(names, a))
        return J.Nn.dense(a["dx"], a["dw"], a.get("dbias"), name, a.get("dresidual"))

    y, pull = J.JAX.vjp(f, *arrays)
    np.testing.assert_array_equal(f(*arrays).numpy(), y.numpy())
    DY = arr(J, dy, offset)
    grads = pull(DY)
    for a, b in zip(grads, pull(DY)):
        np.testing.assert_array_equal(a.numpy(), b.numpy())
    return {"y": y.numpy(), **{n: v.numpy() for n, v in zip(names, grads)}}


def check(got, ref):
    for n, v in got.items():
        value, tol = ref[n]
        assert v.shape == value.shape, n
        if not v.size:
            continue
        off = np.abs(v.astype(np.float64) - value) - tol
        assert np.all(off <= 0), (n, float(off.max()), int((off > 0).sum()), v.size)


def make(seed, x_shape, N, dt=np.float32, bias=True, residual=True):
    r = np.random.default_rng(seed)
    K = x_shape[-1]
    x = r.standard_normal(x_shape).astype(dt)
    w = (r.standard_normal((K, N)) / np.sqrt(max(K, 1))).astype(dt)
    b = (0.3 * r.standard_normal(N)).astype(dt) if bias else None
    res = r.standard_normal(x_shape[:-1] + (N,)).astype(dt) if residual else None
    return x, w, b, res, r.standard_normal(x_shape[:-1] + (N,)).astype(dt)


SMALL = [((1, 1), 1), ((7,), 5), ((1, 784), 512), ((2, 333), 2400), ((3, 100), 10), ((4, 64), 4736), ((7, 50), 1184),
         ((16, 257), 130), ((17, 33), 65), ((2, 3, 20), 9), ((64, 64), 64), ((100, 1), 7), ((65, 1025), 66), ((5, 0), 4),
         ((0, 3), 4), ((3, 4), 0), ((256, 784), 512), ((700, 16), 300)]


@pytest.mark.parametrize("shape,N", SMALL, ids=[f"{'x'.join(map(str, s))}x{n}" for s, n in SMALL])
@pytest.mark.parametrize("f64", [False, True], ids=["f32", "f64"])
def test_small_products(J, shape, N, f64):
    name = ACTS[2 + (sum(shape) + N) % 4]
    x, w, b, res, dy = make(sum(shape) + N, shape, N, np.float64 if f64 else np.float32, bias=N % 2 == 0,
                            residual=sum(shape) % 2 == 0)
    check(run(J, x, w, b, name, res, dy), reference(x, w, b, name, res, dy, 2.0 ** -53 if f64 else U, False))


# Few tiles and a long sum, whose K goes over 16 CTAs, and gradients of which one
# has a long sum and the other many tiles: a launch each.
LONG = [((40, 4100), 70), ((5000, 24), 30), ((1200, 1500), 5), ((1100, 5), 900), ((2500, 700), 33)]


@pytest.mark.parametrize("shape,N", LONG, ids=[f"{'x'.join(map(str, s))}x{n}" for s, n in LONG])
@pytest.mark.parametrize("f64", [False, True], ids=["f32", "f64"])
def test_long_sums(J, shape, N, f64):
    x, w, b, res, dy = make(sum(shape) + N, shape, N, np.float64 if f64 else np.float32)
    check(run(J, x, w, b, "silu", res, dy), reference(x, w, b, "silu", res, dy, 2.0 ** -53 if f64 else U, False))


def test_only_one_gradient_of_long_sums(J):
    x, w, _, _, dy = make(9, (1200, 1500), 5, bias=False, residual=False)
    X, W, DY = arr(J, x), arr(J, w), arr(J, dy)
    both = J.JAX.vjp(lambda a, b: J.Nn.dense(a, b), X, W)[1](DY)
    dx = J.JAX.vjp(lambda a: J.Nn.dense(a, W), X)[1](DY)
    dw = J.JAX.vjp(lambda b: J.Nn.dense(X, b), W)[1](DY)
    np.testing.assert_array_equal(both[0].numpy(), dx[0].numpy())
    np.testing.assert_array_equal(both[1].numpy(), dw[0].numpy())


LARGE = [((17, 5), 3), ((128, 64), 256), ((130, 64), 260), ((257, 1000), 513), ((300, 513), 1000), ((3, 100, 48), 77),
         ((1024, 300), 1000), ((600, 2048), 512)]


@pytest.mark.parametrize("shape,N", LARGE, ids=[f"{'x'.join(map(str, s))}x{n}" for s, n in LARGE])
@pytest.mark.parametrize("name", ["none", "tanh", "gelu"])
@pytest.mark.parametrize("extras", [True, False])
def test_tensor_core_products(J, monkeypatch, shape, N, name, extras):
    from jax4j_b200 import layers
    monkeypatch.setattr(layers, "SMALL_PRODUCT", 0)
    x, w, b, res, dy = make(sum(shape) + N, shape, N, bias=extras, residual=extras)
    check(run(J, x, w, b, name, res, dy), reference(x, w, b, name, res, dy, U, True))


# Wide tiles of a CTA pair, one wave of them and a wave and a half whose last
# tiles are split along K (the shapes above mostly take narrow ones).
@pytest.mark.parametrize("shape,N", [((2048, 40), 2048), ((3840, 704), 1790)], ids=["2048x40x2048", "3840x704x1790"])
def test_wide_tiles(J, monkeypatch, shape, N):
    from jax4j_b200 import layers
    monkeypatch.setattr(layers, "SMALL_PRODUCT", 0)
    x, w, b, res, dy = make(N, shape, N)
    check(run(J, x, w, b, "silu", res, dy), reference(x, w, b, "silu", res, dy, U, True))


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("extras", ["both", "bias", "residual", "none"])
@pytest.mark.parametrize("small", [True, False])
def test_activations_and_optional_inputs(J, monkeypatch, name, extras, small):
    from jax4j_b200 import layers
    monkeypatch.setattr(layers, "SMALL_PRODUCT", layers.SMALL_PRODUCT if small else 0)
    x, w, b, res, dy = make(3, (70, 40), 96, bias=extras in ("both", "bias"), residual=extras in ("both", "residual"))
    if name == "relu":  # where either slope is right: dy is 0 there
        z, ez = reference(x, w, b, "none", None, dy, U, not small)["y"]
        dy[np.abs(z) <= ez] = 0
    check(run(J, x, w, b, name, res, dy), reference(x, w, b, name, res, dy, U, not small))


@pytest.mark.parametrize("small", [True, False])
@pytest.mark.parametrize("offset", [1, 2])
def test_unaligned_arrays(J, monkeypatch, small, offset):
    from jax4j_b200 import layers
    monkeypatch.setattr(layers, "SMALL_PRODUCT", layers.SMALL_PRODUCT if small else 0)
    for shape, N in (((70, 40), 96), ((2, 64), 4736)):
        x, w, b, res, dy = make(5, shape, N)
        check(run(J, x, w, b, "silu", res, dy, offset), reference(x, w, b, "silu", res, dy, U, not small))


def test_at_the_border_between_the_products(J):
    """K = 1024: 1024 x 512 outputs are the last on the CUDA cores, 1025 x 512 the first beyond."""
    from jax4j_b200 import layers
    assert layers.SMALL_PRODUCT == 1024 * 1024 * 512
    for M in (1024, 1025):
        x, w, b, res, dy = make(M, (M, 1024), 512)
        check(run(J, x, w, b, "gelu", res, dy), reference(x, w, b, "gelu", res, dy, U, M == 1025))


def test_few_rows_of_a_large_weight(J):
    """Up to 16 rows stay on the CUDA cores forward, whatever the weight; their
    gradients take the tensor cores beyond SMALL_PRODUCT."""
    from jax4j_b200 import layers
    assert layers.FEW_ROWS == 16
    x, w, b, res, dy = make(14, (16, 6000), 6004)
    assert 16 * 6000 * 6004 > layers.SMALL_PRODUCT
    ref = reference(x, w, b, "silu", res, dy, U, True)
    small = reference(x, w, b, "silu", res, dy, U, False)["y"]
    got = run(J, x, w, b, "silu", res, dy)
    check({"y": got.pop("y")}, {"y": small})
    # the pre-activation's error is the larger of the two forms'
    check(got, {n: (v, np.maximum(e, reference(x, w, b, "silu", res, dy, U, False)[n][1])) for n, (v, e) in ref.items()})


@pytest.mark.parametrize("env", [{"J4C_GEMM_SPLIT": "tf32"}, {"J4C_GEMM_PAIR": "0"}])
def test_other_gemm_variants(env):
    """The tensor-core layers under 3xTF32 and with single-CTA tiles (both are fixed for a process)."""
    import os
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-x", "tests/test_gpu_dense.py", "-k",
                        "tensor_core or line_words or non_finite or border or unaligned"], env={**os.environ, **env},
                       capture_output=True, text=True, timeout=600,
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-2000:]


@pytest.mark.parametrize("rows,cols", [(1, 1), (7, 100), (33, 1024), (40, 1028), (5, 4097), (9, 8192), (300, 512), (3, 8195)])
def test_row_splits_without_a_max_pass(J, rows, cols):
    """The split that takes its maxima on the way is, bit for bit, the one that is given them."""
    import torch
    from jax4j_b200 import _lib
    r = np.random.default_rng(rows + cols)
    x = (r.standard_normal((rows, cols)) * 10.0 ** r.integers(-30, 30, (rows, 1))).astype(np.float32)
    for special in (False, True):
        if special:
            x[rows // 2, cols // 2] = np.nan
            x[0, 0] = -np.inf
        for offset in (0, 1):
            X = arr(J, x, offset)
            n = _lib.lib().j4c_split_floats(rows, cols)
            out = [torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(4)]
            lines = torch.empty(rows + cols + 1, dtype=torch.int32, device="cuda")
            s = X._stream()
            _lib.call("j4c_split_lines", X.data_ptr(), rows, cols, lines.data_ptr(), s)
            _lib.call("j4c_split_f32_ex", X.data_ptr(), rows, cols, out[0].data_ptr(), out[1].data_ptr(), None, None, None,
                      None, lines.data_ptr(), s)
            _lib.call("j4c_split_f32_ex", X.data_ptr(), rows, cols, out[2].data_ptr(), out[3].data_ptr(), None, None, None,
                      None, None, s)
            for a, b in ((out[0], out[2]), (out[1], out[3])):
                np.testing.assert_array_equal(a.cpu().numpy(), b.cpu().numpy())


@pytest.mark.parametrize("small", [True, False])
def test_non_finite_values(J, monkeypatch, small):
    """Infinities and NaN reach exactly the outputs that depend on them."""
    from jax4j_b200 import layers
    monkeypatch.setattr(layers, "SMALL_PRODUCT", layers.SMALL_PRODUCT if small else 0)
    x, w, b, res, dy = make(6, (40, 50), 60)
    x[3, 4], x[9, 0] = np.inf, np.nan
    w[7, 11] = -np.inf
    y = J.Nn.dense(arr(J, x), arr(J, w), arr(J, b), "sigmoid", arr(J, res)).numpy()
    with np.errstate(invalid="ignore"):
        z = x.astype(np.float64) @ w.astype(np.float64) + b
    bad = np.isnan(z)
    assert np.array_equal(np.isnan(y), bad) and bad.any()
    np.testing.assert_allclose(y[~bad], (1 / (1 + np.exp(-z)) + res)[~bad], rtol=1e-5, atol=1e-5)


def test_gradient_line_words(J):
    import torch
    from jax4j_b200 import _lib
    r = np.random.default_rng(8)
    for M, N in ((1, 1), (33, 255), (100, 257), (700, 1028)):
        dy, z = (r.standard_normal((M, N)).astype(np.float32) for _ in range(2))
        if M == 100:
            dy[50, 100] = np.nan
        DY, Z = arr(J, dy), arr(J, z)
        dz = torch.empty(M * N, device="cuda")
        db = torch.empty(N, device="cuda")
        lines, want = (torch.empty(M + N + 1, dtype=torch.int32, device="cuda") for _ in range(2))
        need = _lib.lib().j4c_dense_grad_workspace(0, M, N)
        ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
        s = DY._stream()
        _lib.call("j4c_dense_grad", 0, M, N, DY.data_ptr(), Z.data_ptr(), 5, 0, dz.data_ptr(), db.data_ptr(),
                  lines.data_ptr(), ws.data_ptr(), need, s)
        _lib.call("j4c_split_lines", dz.data_ptr(), M, N, want.data_ptr(), s)
        np.testing.assert_array_equal(lines.cpu().numpy()[:-1], want.cpu().numpy()[:-1])
        assert bool(lines[-1].item()) == bool(want[-1].item()) == (M == 100)


@pytest.mark.parametrize("name", ACTS)
def test_gradients_against_differences(J, name):
    x, w, b, res, dy = make(9, (3, 5), 4, np.float64)
    got = run(J, x, w, b, name, res, dy)

    def f(*a):
        return float((J.Nn.dense(*[arr(J, t) for t in a[:3]], name, arr(J, a[3])).numpy() * dy).sum())

    step = 1e-5
    for i, n in enumerate(("dx", "dw", "dbias", "dresidual")):
        args = [x, w, b, res]
        for at in np.ndindex(args[i].shape):
            up, down = ([a.copy() for a in args] for _ in range(2))
            up[i][at] += step
            down[i][at] -= step
            assert abs((f(*up) - f(*down)) / (2 * step) - got[n][at]) <= 1e-7, (n, at)


@pytest.mark.parametrize("small", [True, False])
def test_inside_transformations(J, monkeypatch, small):
    from jax4j_b200 import layers
    monkeypatch.setattr(layers, "SMALL_PRODUCT", layers.SMALL_PRODUCT if small else 0)
    x, w, b, res, _ = make(10, (6, 8, 32), 32)
    X, W, B, R = (arr(J, a) for a in (x, w, b, res))
    layer = lambda a: J.Nn.dense(a, W, B, "silu", a)  # noqa: E731
    direct = layer(X).numpy()
    np.testing.assert_array_equal(J.JAX.jit(layer)(X).numpy(), direct)
    loss = lambda a: layer(layer(a)).tanh().sum()  # noqa: E731
    g = J.JAX.grad(loss)(X).numpy()
    np.testing.assert_array_equal(J.JAX.grad(J.JAX.checkpoint(loss))(X).numpy(), g)
    np.testing.assert_array_equal(J.JAX.vmap(layer)(X.reshape(J.Shape(2, 3, 8, 32))).numpy().reshape(6, 8, 32), direct)
    # the same chain of the framework's own operations
    two = X.reshape(J.Shape(48, 32))
    chain = lambda a: [a.dot(W).add(B)][0]  # noqa: E731

    def plain(a):
        for _ in range(2):
            z = chain(a)
            a = z.mul(z.sigmoid()).add(a)
        return a.tanh().sum()

    np.testing.assert_allclose(g.reshape(48, 32), J.JAX.grad(plain)(two).numpy(), rtol=1e-4, atol=1e-5)
    devs = [J.Device(None), J.Device(None)]
    gp = J.JAX.grad(lambda a: J.JAX.pmap(lambda p: loss(p), devs)(a).sum())(X.reshape(J.Shape(2, 3, 8, 32)))
    np.testing.assert_allclose(gp.numpy().reshape(6, 8, 32), g, rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("small", [True, False])
def test_only_the_wanted_gradients(J, monkeypatch, small):
    from jax4j_b200 import layers
    monkeypatch.setattr(layers, "SMALL_PRODUCT", layers.SMALL_PRODUCT if small else 0)
    x, w, b, _, dy = make(11, (600, 700), 800, residual=False)
    X, W, B = arr(J, x), arr(J, w), arr(J, b)
    full = run(J, x, w, b, "gelu", None, dy)
    DY = arr(J, dy)
    for f, arg, n in ((lambda a: J.Nn.dense(a, W, B, "gelu"), X, "dx"), (lambda a: J.Nn.dense(X, a, B, "gelu"), W, "dw"),
                      (lambda a: J.Nn.dense(X, W, a, "gelu"), B, "dbias")):
        np.testing.assert_array_equal(J.JAX.vjp(f, arg)[1](DY)[0].numpy(), full[n])


@pytest.mark.parametrize("shape,N,small,dt", [((64, 200), 100, True, np.float32), ((512, 1024), 600, False, np.float32),
                                              ((40, 4100), 70, True, np.float64), ((1200, 1500), 5, True, np.float32),
                                              ((3840, 704), 1790, False, np.float32)])
def test_recorded_and_on_another_stream(J, monkeypatch, shape, N, small, dt):
    import torch
    from jax4j_b200 import layers
    monkeypatch.setattr(layers, "SMALL_PRODUCT", layers.SMALL_PRODUCT if small else 0)
    from jax4j_b200.graphs import CapturedStep
    x, w, b, res, dy = make(12, shape, N, dt)
    r = np.random.default_rng(13)

    def step(*a):
        y, pull = J.JAX.vjp(lambda p, q, s, t: J.Nn.dense(p, q, s, "gelu", t), *a[:4])
        return [y, *pull(a[4])[:3]]

    args = [arr(J, a) for a in (x, w, b, res, dy)]
    y, pull = J.JAX.vjp(lambda p, q: J.Nn.dense(p, q, args[2], "gelu"), args[0], args[1])
    graphs = [CapturedStep(step, [J.ConcreteNDArray(a.tensor().clone(), a.shape()) for a in args]) for _ in range(2)]
    for _ in range(2):
        args = [arr(J, r.standard_normal(a.shape().dimensions()).astype(dt)) for a in args]
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
    assert np.isfinite(pull(arr(J, dy))[0].numpy()).all()
    for gr in graphs:
        gr.release()
