"""Optim.adamW against its formulas in 64 bits: both moment formats, leaves of
every awkward size and alignment, trees of more leaves than one launch takes,
non-finite gradients, recorded steps and other streams."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a step of FLOAT32, relative


@pytest.fixture(scope="module")
def J():
    import jax4j_b200 as j
    return j


def tree(J, arrays):
    return J.PyTree.list(*[J.PyTree.leaf(a) for a in arrays])


def arr(J, x, shape=None, offset=0):
    """x on the GPU, `offset` elements behind a 256-byte boundary."""
    import torch
    x = np.ascontiguousarray(x)
    buf = torch.empty(x.size + offset, dtype=torch.from_numpy(x).dtype, device="cuda")
    buf[offset:] = torch.from_numpy(x.reshape(-1))
    return J.ConcreteNDArray(buf[offset:], J.Shape(shape or x.shape))


def host(tree_, J):
    return [a.numpy() for a in J.PyTrees.flatten(tree_)]


def ref_step(w, g, m, v, t, lr, b1, b2, eps, wd, scale):
    """The formulas in 64 bits, and bounds of the FLOAT32 evaluation's error:
    every product, sum, root and quotient is off by at most U of its result,
    and every coefficient by U of its value."""
    w, m, v = (x.astype(np.float64) for x in (w, m, v))
    g = g.astype(np.float64) * scale
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    # m: g' one rounding and scale's; per product one rounding and a coefficient's; one sum
    em = U * (3 * np.abs(b1 * m) + 5 * np.abs((1 - b1) * g))
    ev = U * (3 * b2 * v + 8 * (1 - b2) * g * g)
    a, b = 1 / (1 - b1 ** t), 1 / np.sqrt(1 - b2 ** t)
    root = np.sqrt(v1)
    den = root * b + eps
    up = m1 * a / den
    # numerator: em and two roundings; denominator: ev / 2 (the root halves it), root, coefficient, product, eps, sum
    with np.errstate(divide="ignore", invalid="ignore"):
        rel_v = np.where(v1 > 0, ev / v1, 0.0)
    eup = em * a / den + np.abs(up) * (2 * U + rel_v / 2 + 5 * U + U)
    w1 = w - lr * wd * w - lr * up
    # lr * wd * w: two roundings; lr * up: two; two differences
    ew = U * (2 * np.abs(lr * wd * w) + 2 * np.abs(lr * up) + 2 * (np.abs(w) + np.abs(lr * up))) + lr * eup
    tiny = 1e-44  # subnormal steps
    return (w1, 1.01 * ew + tiny), (m1, 1.01 * em + tiny), (v1, 1.01 * ev + tiny)


SIZES = [1, 3, 4, 127, 128, 129, 1023, 4096, 4100, 70001]


def make(seed, sizes, dtype=np.float32):
    r = np.random.default_rng(seed)
    w = [r.standard_normal(n).astype(dtype) for n in sizes]
    g = [(r.standard_normal(n) * np.exp(r.standard_normal(n))).astype(dtype) for n in sizes]
    return w, g


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("scale", [1.0, 0.125])
def test_steps_match_the_formulas(J, dtype, offset, scale):
    w, _ = make(1, SIZES, dtype)
    wd = [0.0 if i % 3 == 0 else 0.01 * i for i in range(len(w))]
    params = tree(J, [arr(J, x, offset=offset) for x in w])
    state = J.Optim.adamWInit(params)
    m, v = [np.zeros_like(x) for x in w], [np.zeros_like(x) for x in w]
    for t in range(1, 4):
        _, g = make(10 + t, SIZES, dtype)
        lr = 0.01 / t
        params, state = J.Optim.adamW(params, tree(J, [arr(J, x, offset=offset) for x in g]), state, lr, beta1=0.8,
                                      beta2=0.95, eps=1e-6, weightDecay=wd, scale=scale)
        new_w, (mt, vt) = host(params, J), state.moments()
        new_m, new_v = host(mt, J), host(vt, J)
        for i in range(len(w)):
            refs = ref_step(w[i], g[i], m[i], v[i], t, lr, 0.8, 0.95, 1e-6, wd[i], scale)
            for got, (ref, tol) in zip((new_w[i], new_m[i], new_v[i]), refs):
                assert got.dtype == dtype
                if dtype == np.float64:
                    tol = tol * 2.0 ** -28 + 1e-300  # a FLOAT64 half step is 2^-53
                assert np.all(np.abs(got.astype(np.float64) - ref) <= tol), (i, t)
        w, m, v = new_w, new_m, new_v
        np.testing.assert_allclose(state.step().numpy(), [t, 0.8 ** t, 0.95 ** t], rtol=1e-15)


def test_bits_equal_the_rounded_expressions(J):
    """The FLOAT32 step is the elementwise evaluation of its expressions, each
    operation rounded (torch's elementwise kernels round the same way)."""
    import torch
    w, g = make(2, [5000])
    W, G = torch.from_numpy(w[0]).cuda(), torch.from_numpy(g[0]).cuda()
    params = tree(J, [arr(J, w[0])])
    state = J.Optim.adamWInit(params)
    M = V = torch.zeros_like(W)
    p1 = p2 = 1.0
    for _ in range(3):
        params, state = J.Optim.adamW(params, tree(J, [arr(J, g[0])]), state, 1e-3)
        p1, p2 = p1 * 0.9, p2 * 0.999
        M = M.mul(0.9).add(G.mul(1.0 - 0.9))
        V = V.mul(0.999).add(G.mul(G).mul(1.0 - 0.999))
        a, b = np.float32(1 / (1 - p1)), np.float32(1 / np.sqrt(1 - p2))
        up = M.mul(float(a)).div(V.sqrt().mul(float(b)).add(1e-8))
        W = W.sub(W.mul(1e-3 * 0.01)).sub(up.mul(1e-3))
    np.testing.assert_array_equal(host(params, J)[0].view(np.uint32), W.cpu().numpy().view(np.uint32))
    m, v = state.moments()
    np.testing.assert_array_equal(host(m, J)[0], M.cpu().numpy())
    np.testing.assert_array_equal(host(v, J)[0], V.cpu().numpy())


def unpack(words, n):
    """The packed words' values in 64 bits, and each value's block step."""
    nb = (n + 127) // 128
    b = words.view(np.uint8)
    cm, cr = b[:128 * nb].astype(np.int64), b[128 * nb:256 * nb].astype(np.int64)
    steps = words[64 * nb:].view(np.float32).astype(np.float64)
    e, f = (cm >> 3) & 15, cm & 7
    mag = np.where(e > 0, (8 + f) * 2.0 ** (e - 10.0), f * 2.0 ** -9)
    m = np.where((cm & 127) == 127, np.nan, np.where(cm > 127, -mag, mag))
    e, f = cr >> 4, cr & 15
    r = np.where(cr == 255, np.nan, np.where(e > 0, (16 + f) * 2.0 ** (e - 11.0), f * 2.0 ** -10))
    sm, sr = np.repeat(steps[:nb], 128), np.repeat(steps[nb:], 128)
    return (m * sm)[:n], (r * sr)[:n], sm[:n], sr[:n]


@pytest.mark.parametrize("offset", [0, 3])
def test_eight_bit_steps(J, offset):
    sizes = [0] + SIZES
    w, _ = make(3, sizes)
    params = tree(J, [arr(J, x, offset=offset) for x in w])
    state = J.Optim.adamWInit(params, stateBits=8)
    for t in range(1, 5):
        _, g = make(30 + t, sizes)
        before = [unpack(a.numpy(), n) for a, n in zip(state.arrays()[1:], sizes)]
        params, state = J.Optim.adamW(params, tree(J, [arr(J, x, offset=offset) for x in g]), state, 1e-2)
        after = [unpack(a.numpy(), n) for a, n in zip(state.arrays()[1:], sizes)]
        got_w, (mt, vt) = host(params, J), state.moments()
        for i, n in enumerate(sizes):
            # the held root is decoded (one rounding) and squared (one): 3 U of v
            m0, r0 = before[i][0], before[i][1]
            (w1, ew), (m1, em), (v1, ev) = ref_step(w[i], g[i], m0, r0 * r0, t, 1e-2, 0.9, 0.999, 1e-8, 0.01, 1.0)
            em, ev = em + U * np.abs(0.9 * m0), ev + 3 * U * r0 * r0
            with np.errstate(divide="ignore", invalid="ignore"):
                up = np.abs(1e-2 * m1 / (1 - 0.9 ** t) / (np.sqrt(v1 / (1 - 0.999 ** t)) + 1e-8))
            mag = np.abs(0.9 * m0) / np.maximum(np.abs(m1), 1e-300)
            # the quotient is off by up to 2 ulp (4 U), of which ref_step counts one rounding
            assert np.all(np.abs(got_w[i] - w1) <= ew + up * U * (5 + mag)), (i, t)
            m, r, sm, sr = after[i]
            r1 = np.sqrt(v1)
            # half a step of the code (2^-4 and 2^-5 relative, 2^-10 and 2^-11 of the block's step below the
            # smallest normal; a root's smallest code takes anything above zero, hence 2^-10), and the roundings
            # of the computed value, of the scaling and of the step (4 U)
            assert np.all(np.abs(m - m1) <= np.abs(m1) * (2.0 ** -4 + 4 * U) + sm * 2.0 ** -10 + 1.07 * em), (i, t)
            er = np.where(r1 > 0, ev / np.maximum(r1, 1e-300), 0)
            assert np.all(np.abs(r - r1) <= r1 * (2.0 ** -5 + 4 * U) + sr * 2.0 ** -10 + 1.07 * er), (i, t)
            assert np.all((r > 0) == (r1 > 0)), "a root above zero is held as zero"
            np.testing.assert_allclose(host(mt, J)[i], m, rtol=U)
            np.testing.assert_allclose(host(vt, J)[i], r * r, rtol=4 * U)
        w = got_w


def test_eight_bit_moments_of_a_steady_gradient_converge(J):
    """A block whose gradient stops decays through its step: after 200 steps
    of zero gradients no moment is stuck at its value."""
    g = np.linspace(0.5, 2.0, 256).astype(np.float32)
    params = tree(J, [arr(J, np.zeros(256, np.float32))])
    state = J.Optim.adamWInit(params, stateBits=8)
    for t in range(20):
        params, state = J.Optim.adamW(params, tree(J, [arr(J, g)]), state, 1e-3, beta2=0.9)
    held = [x[0] for x in map(lambda tr: host(tr, J), state.moments())]
    zero = tree(J, [arr(J, np.zeros(256, np.float32))])
    for t in range(40):
        params, state = J.Optim.adamW(params, zero, state, 1e-3, beta2=0.9)
    for x, y in zip(held, [x[0] for x in map(lambda tr: host(tr, J), state.moments())]):
        # 0.9^40 = 0.0148; the block's largest value decays exactly (its code is the top one), the others with it
        np.testing.assert_allclose(y, x * 0.9 ** 40, rtol=2.0 ** -4)


@pytest.mark.parametrize("count", [25, 400, 900])
@pytest.mark.parametrize("bits", [8, 32])
def test_many_leaves(J, count, bits):
    """More leaves than the small table (24) and than one launch (380)."""
    sizes = [1 + (7 * i) % 300 for i in range(count)]
    w, g = make(4, sizes)
    params = tree(J, [arr(J, x) for x in w])
    state = J.Optim.adamWInit(params, stateBits=bits)
    new, state = J.Optim.adamW(params, tree(J, [arr(J, x) for x in g]), state, 1e-2)
    got = host(new, J)
    for i in range(count):
        (w1, ew), _, _ = ref_step(w[i], g[i], 0 * w[i], 0 * w[i], 1, 1e-2, 0.9, 0.999, 1e-8, 0.01, 1.0)
        assert np.all(np.abs(got[i] - w1) <= ew), i
    np.testing.assert_array_equal(host(params, J)[5], w[5])  # the arguments stay
    assert state.step().numpy()[0] == 1.0


@pytest.mark.parametrize("bits", [8, 32])
def test_empty_trees_and_leaves(J, bits):
    """Nothing to update: the count still advances."""
    for arrays in ([], [arr(J, np.zeros(0, np.float32))], [arr(J, np.zeros((0, 4), np.float32))] * 2):
        params = tree(J, arrays)
        p, s = J.Optim.adamW(params, params, J.Optim.adamWInit(params, bits), 1e-2, beta2=0.5)
        assert len(J.PyTrees.flatten(p)) == len(arrays)
        np.testing.assert_array_equal(s.step().numpy(), [1.0, 0.9, 0.5])
        m, _ = s.moments()
        assert [a.numpy().shape for a in J.PyTrees.flatten(m)] == [a.shape().dimensions() for a in arrays]


def test_mixed_dtypes_take_one_count(J):
    w32, g32 = make(5, [300])
    w64, g64 = make(6, [200], np.float64)
    params = tree(J, [arr(J, w64[0]), arr(J, w32[0])])
    state = J.Optim.adamWInit(params)
    params, state = J.Optim.adamW(params, tree(J, [arr(J, g64[0]), arr(J, g32[0])]), state, 1e-2)
    got = host(params, J)
    for x, w, g, f in ((got[0], w64[0], g64[0], 2.0 ** -28), (got[1], w32[0], g32[0], 1.0)):
        (w1, ew), _, _ = ref_step(w, g, 0 * w, 0 * w, 1, 1e-2, 0.9, 0.999, 1e-8, 0.01, 1.0)
        assert np.all(np.abs(x - w1) <= ew * f)
    assert state.step().numpy()[0] == 1.0


@pytest.mark.parametrize("bits", [8, 32])
def test_non_finite_gradients_stay_where_they_are(J, bits):
    w, g = make(7, [512])
    bad = g[0].copy()
    bad[5], bad[131], bad[260] = np.nan, np.inf, -np.inf
    params = tree(J, [arr(J, w[0])])
    s0 = J.Optim.adamWInit(params, stateBits=bits)
    p1, s1 = J.Optim.adamW(params, tree(J, [arr(J, bad)]), s0, 1e-2)
    q1, t1 = J.Optim.adamW(params, tree(J, [arr(J, g[0])]), s0, 1e-2)
    hit = np.array([5, 131, 260])
    rest = np.delete(np.arange(512), hit)
    np.testing.assert_array_equal(host(p1, J)[0][rest], host(q1, J)[0][rest])
    assert np.isnan(host(p1, J)[0][hit]).all()  # inf / inf as well
    m, v = (host(x, J)[0] for x in s1.moments())
    if bits == 8:
        assert np.isnan(m[hit]).all() and np.isnan(v[hit]).all()
        # a block with a value that is not finite takes its step from the others
        assert np.isfinite(m[rest]).all() and np.isfinite(v[rest]).all() and (v[rest] > 0).all()
    else:
        np.testing.assert_array_equal(m[rest], host(t1.moments()[0], J)[0][rest])
        assert np.isnan(v[5]) and np.isinf(v[131]) and np.isinf(v[260])


@pytest.mark.parametrize("bits", [8, 32])
def test_extreme_magnitudes(J, bits):
    """Gradients from 1e-37 to 1e18 beside each other: squares below FLOAT32
    are zeros, no value turns into NaN."""
    g = np.float32(10.0) ** np.linspace(-37, 18, 1024).astype(np.float32)
    params = tree(J, [arr(J, np.ones(1024, np.float32))])
    p, s = J.Optim.adamW(params, tree(J, [arr(J, g.astype(np.float32))]), J.Optim.adamWInit(params, bits), 1e-2)
    assert np.isfinite(host(p, J)[0]).all()
    for x in s.moments():
        assert np.isfinite(host(x, J)[0]).all()


def test_lr_as_an_array_and_in_place_at_the_c_entry(J):
    import ctypes as C

    import torch
    from jax4j_b200._lib import call
    w, g = make(8, [3000])
    params, grads = tree(J, [arr(J, w[0])]), tree(J, [arr(J, g[0])])
    s0 = J.Optim.adamWInit(params, 8)
    lr = J.ConcreteNDArray.of([0.25])
    p1, s1 = J.Optim.adamW(params, grads, s0, lr, weightDecay=0.0)
    p2, s2 = J.Optim.adamW(params, grads, s0, 0.25, weightDecay=0.0)
    np.testing.assert_array_equal(host(p1, J)[0], host(p2, J)[0])
    W, G, Q = (t.clone() for t in (J.PyTrees.flatten(params)[0].tensor(), J.PyTrees.flatten(grads)[0].tensor(),
                                   s0.arrays()[1].tensor()))
    one = lambda t: (C.c_void_p * 1)(t.data_ptr())  # noqa: E731
    steps, out = s0.step().tensor(), torch.empty(3, dtype=torch.float64, device="cuda")
    call("j4c_adamw_step", 0, 8, 1, (C.c_int64 * 1)(3000), one(W), one(G), one(Q), one(W), one(Q), (C.c_double * 1)(0.0),
         steps.data_ptr(), out.data_ptr(), None, 0.25, 1.0, 0.9, 0.999, 1e-8, torch.cuda.current_stream().cuda_stream)
    np.testing.assert_array_equal(W.cpu().numpy(), host(p2, J)[0])
    np.testing.assert_array_equal(Q.cpu().numpy(), s2.arrays()[1].numpy())
    np.testing.assert_array_equal(out.cpu().numpy(), s2.step().numpy())


@pytest.mark.parametrize("bits", [8, 32])
def test_recorded_steps_count_on(J, bits):
    """A CapturedStep that carries weights, moments and the count replays the
    eager steps bit for bit; a second recording beside it shares nothing."""
    from jax4j_b200.graphs import CapturedStep
    w, g = make(9, [700, 33])
    grads = [arr(J, x) for x in g]
    p0 = tree(J, [arr(J, x) for x in w])
    s0 = J.Optim.adamWInit(p0, bits)

    def step(*a):
        st = s0.withArrays(a[2:-1])
        p, st = J.Optim.adamW(tree(J, a[:2]), tree(J, grads), st, a[-1])
        return [*J.PyTrees.flatten(p), *st.arrays()]

    def fresh():
        return [J.ConcreteNDArray(x.tensor().clone(), x.shape(), x.dtype()) for x in [*J.PyTrees.flatten(p0), *s0.arrays()]]

    graphs = []
    for _ in range(2):
        ins = fresh() + [J.ConcreteNDArray.of([1e-2])]
        graphs.append(CapturedStep(step, ins, donate={i: i for i in range(len(ins) - 1)}))
    p, s = p0, s0
    for t in range(4):
        lr = 1e-2 if t < 2 else 5e-3
        for gr in graphs:
            gr.set_input(len(gr.inputs) - 1, J.ConcreteNDArray.of([lr]))
            gr()
        p, s = J.Optim.adamW(p, tree(J, grads), s, J.ConcreteNDArray.of([lr]))
        for gr in graphs:
            for a, b in zip(gr.inputs, [*J.PyTrees.flatten(p), *s.arrays()]):
                np.testing.assert_array_equal(a.numpy(), b.numpy())
        assert s.step().numpy()[0] == t + 1
    for gr in graphs:
        gr.release()


def test_on_another_stream(J):
    import torch
    w, g = make(11, [100000])
    params, grads = tree(J, [arr(J, w[0])]), tree(J, [arr(J, g[0])])
    state = J.Optim.adamWInit(params)
    want = host(J.Optim.adamW(params, grads, state, 1e-2)[0], J)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        p, _ = J.Optim.adamW(params, grads, state, 1e-2)
    side.synchronize()
    np.testing.assert_array_equal(host(p, J)[0], want)


def test_data_parallel_step(J):
    """Lax.psumAdamWTree on two shards: every shard ends with Optim.adamW of
    the summed gradients."""
    r = np.random.default_rng(12)
    w = r.standard_normal((33, 20)).astype(np.float32)
    x = r.standard_normal((2, 8, 33)).astype(np.float32)
    params = J.PyTree.dictOf({"w": arr(J, w)})
    state = J.Optim.adamWInit(params, 8)
    new = {}

    def loss(p, xs):
        return xs.dot(p.children["w"].value).tanh().sum()

    def body(xs):
        loc = J.PyTrees.map(lambda a: a.to(xs.device()), params)
        v, grads = J.JAX.valueAndGradTree(lambda p: loss(p, xs))(loc)
        new[id(xs.device())] = J.Lax.psumAdamWTree(loc, grads, state, 1e-2, scale=0.5, beta2=0.99)
        return v

    J.JAX.pmap(body, [J.Device(None), J.Device(None)])(arr(J, x))
    both = list(new.values())
    assert len(both) == 2
    gs = [J.JAX.gradTree(lambda p, i=i: loss(p, arr(J, x[i])))(params) for i in range(2)]
    total = J.PyTrees.map2(lambda a, b: a.add(b), *gs)
    want, ws = J.Optim.adamW(params, total, state, 1e-2, scale=0.5, beta2=0.99)
    for p, s in both:
        np.testing.assert_array_equal(host(p, J)[0], host(want, J)[0])
        np.testing.assert_array_equal(s.arrays()[1].numpy(), ws.arrays()[1].numpy())
