"""The training operators together, as a network uses them: residual blocks of
group norm and dense layers with activations, a softmax cross-entropy, gradients
through the grad interpreter and the AdamW update -- eagerly, data-parallel,
and recorded as a CUDA graph -- against the same step in FLOAT64 torch."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def J():
    import jax4j_b200 as j
    return j


WIDTHS = {"tiny": (24, 32, 10, 12), "wide": (200, 512, 100, 1600)}  # inputs, hidden, classes, batch
BLOCKS = 2


def init(seed, size):
    d, h, c, _ = WIDTHS[size]
    r = np.random.default_rng(seed)
    dense = lambda k, n: (r.standard_normal((k, n)) / np.sqrt(k)).astype(np.float32)  # noqa: E731
    p = {"w_in": dense(d, h), "b_in": (0.1 * r.standard_normal(h)).astype(np.float32)}
    for i in range(BLOCKS):
        p[f"gamma{i}"] = (1 + 0.1 * r.standard_normal(h)).astype(np.float32)
        p[f"beta{i}"] = (0.1 * r.standard_normal(h)).astype(np.float32)
        p[f"w{i}"], p[f"b{i}"] = dense(h, h), (0.1 * r.standard_normal(h)).astype(np.float32)
    p["w_out"], p["b_out"] = dense(h, c), (0.1 * r.standard_normal(c)).astype(np.float32)
    return p


def batch(seed, size):
    d, _, c, n = WIDTHS[size]
    r = np.random.default_rng(seed)
    t = np.zeros((n, c), np.float32)
    t[np.arange(n), r.integers(0, c, n)] = 1
    return r.standard_normal((n, d)).astype(np.float32), t


def loss_of(J, x, t):
    neg = J.ConcreteNDArray.scalar(-1.0, device=x.device())

    def loss(p):
        v = {k: leaf.value for k, leaf in p.children.items()}
        h = J.Nn.dense(x, v["w_in"], v["b_in"], "silu")
        for i in range(BLOCKS):
            h = J.Nn.dense(J.Nn.groupNorm(h, 4, v[f"gamma{i}"], v[f"beta{i}"]), v[f"w{i}"], v[f"b{i}"], "gelu", h)
        logits = J.Nn.dense(h, v["w_out"], v["b_out"])
        return J.Nn.softmax(logits).log().mul(t).sum(-1).mean().mul(neg)
    return loss


def torch_loss(p, x, t):
    import torch
    F = torch.nn.functional
    h = F.silu(x @ p["w_in"] + p["b_in"])
    for i in range(BLOCKS):
        n = F.group_norm(h, 4, p[f"gamma{i}"], p[f"beta{i}"], eps=1e-5)
        h = F.gelu(n @ p[f"w{i}"] + p[f"b{i}"], approximate="tanh") + h
    return -(torch.log_softmax(h @ p["w_out"] + p["b_out"], -1) * t).sum(-1).mean()


def tree(J, params):
    return J.PyTree.dictOf({k: J.ConcreteNDArray.of(v) for k, v in params.items()})


def values(tree_):
    return {k: leaf.value.numpy() for k, leaf in tree_.children.items()}


@pytest.mark.parametrize("size", ["tiny", "wide"])
def test_gradients_of_the_network(J, size):
    import torch
    params = init(1, size)
    x, t = batch(2, size)
    p64 = {k: torch.from_numpy(v.astype(np.float64)).requires_grad_() for k, v in params.items()}
    ref = torch_loss(p64, torch.from_numpy(x.astype(np.float64)), torch.from_numpy(t.astype(np.float64)))
    ref.backward()
    value, grads = J.JAX.valueAndGradTree(loss_of(J, J.ConcreteNDArray.of(x), J.ConcreteNDArray.of(t)))(tree(J, params))
    # a dozen operations of 1e-6 relative error at most, each amplified by a bounded slope
    assert abs(float(value.numpy()[0]) - ref.item()) <= 2e-5 * abs(ref.item())
    for k, g in values(grads).items():
        want = p64[k].grad.numpy()
        assert np.linalg.norm(g - want) <= 1e-4 * np.linalg.norm(want), k


@pytest.mark.parametrize("bits", [8, 32])
def test_steps_eager_and_recorded(J, bits):
    """Four steps: eager ones against FLOAT64 torch gradients fed through the
    formulas' own FLOAT64 state (32-bit moments), and a recorded step that
    carries everything against the eager ones, bit for bit."""
    import torch
    from jax4j_b200.graphs import CapturedStep
    params = init(3, "tiny")
    names = list(params)
    data = [batch(10 + i, "tiny") for i in range(4)]
    wd = [0.01 if params[k].ndim == 2 else 0.0 for k in names]
    p, s = tree(J, params), None
    s = J.Optim.adamWInit(p, bits)
    s0 = s

    def step(*a):
        n = len(names)
        pt = J.PyTree.dictOf(dict(zip(names, a[:n])))
        st = s0.withArrays(a[n:-2])
        value, g = J.JAX.valueAndGradTree(loss_of(J, a[-2], a[-1]))(pt)
        pt, st = J.Optim.adamW(pt, g, st, 1e-2, weightDecay=wd)
        return [*J.PyTrees.flatten(pt), *st.arrays(), value]

    first = [J.ConcreteNDArray.of(v) for v in data[0]]
    ins = [J.ConcreteNDArray(a.tensor().clone(), a.shape(), a.dtype())
           for a in [*J.PyTrees.flatten(p), *s.arrays(), *first]]
    graph = CapturedStep(step, ins, donate={i: i for i in range(len(ins) - 2)})
    p64 = {k: torch.from_numpy(v.astype(np.float64)) for k, v in params.items()}
    m64, v64 = ({k: torch.zeros_like(w) for k, w in p64.items()} for _ in range(2))
    losses = []
    for t, (x, y) in enumerate(data, 1):
        xs, ys = J.ConcreteNDArray.of(x), J.ConcreteNDArray.of(y)
        graph.set_input(len(ins) - 2, xs)
        graph.set_input(len(ins) - 1, ys)
        replay = graph()
        out = step(*J.PyTrees.flatten(p), *s.arrays(), xs, ys)
        p = J.PyTrees.unflatten(p, out[:len(names)])
        s = s.withArrays(out[len(names):-1])
        np.testing.assert_array_equal(replay[-1].numpy(), out[-1].numpy())
        for a, b in zip(graph.inputs, out[:-1]):
            np.testing.assert_array_equal(a.numpy(), b.numpy())
        losses.append(float(out[-1].numpy()[0]))
        lead = {k: w.clone().requires_grad_() for k, w in p64.items()}
        torch_loss(lead, torch.from_numpy(x.astype(np.float64)), torch.from_numpy(y.astype(np.float64))).backward()
        for k, d in zip(names, wd):
            g = lead[k].grad
            m64[k] = 0.9 * m64[k] + 0.1 * g
            v64[k] = 0.999 * v64[k] + 0.001 * g * g
            up = m64[k] / (1 - 0.9 ** t) / ((v64[k] / (1 - 0.999 ** t)).sqrt() + 1e-8)
            p64[k] = p64[k] - 1e-2 * (up + d * p64[k])
        if bits == 32:
            for k, w in values(p).items():
                # the first step moves every weight by lr whatever its gradient's size, so a weight whose gradient
                # is within rounding of 0 may move either way: the network's own error, not the update's; by norm
                assert np.linalg.norm(w - p64[k].numpy()) <= 2e-4 * np.linalg.norm(p64[k].numpy()), (k, t)
    assert s.step().numpy()[0] == 4 and all(np.isfinite(losses))
    graph.release()


def test_data_parallel_step(J):
    """Two shards with Lax.psumAdamWTree end where one step on the whole batch
    ends: the mean of the shards' mean losses is the batch's."""
    params = init(4, "tiny")
    x, t = batch(5, "tiny")
    p = tree(J, params)
    s = J.Optim.adamWInit(p)
    half = len(x) // 2
    new = {}

    def body(xs, ts):
        loc = J.PyTrees.map(lambda a: a.to(xs.device()), p)
        value, g = J.JAX.valueAndGradTree(loss_of(J, xs, ts))(loc)
        new[id(xs.device())] = J.Lax.psumAdamWTree(loc, g, s, 1e-2, scale=0.5)[0]
        return value

    devs = [J.Device(None), J.Device(None)]
    xs = J.ConcreteNDArray.of(x.reshape(2, half, -1))
    ts = J.ConcreteNDArray.of(t.reshape(2, half, -1))
    losses = J.JAX.pmap(body, devs)(xs, ts).numpy()
    value, g = J.JAX.valueAndGradTree(loss_of(J, J.ConcreteNDArray.of(x), J.ConcreteNDArray.of(t)))(p)
    assert abs(losses.mean() - value.numpy()[0]) <= 1e-5 * abs(value.numpy()[0])
    whole, _ = J.Optim.adamW(p, g, s, 1e-2)
    a, b = (values(v) for v in new.values())
    for k, w in values(whole).items():
        np.testing.assert_array_equal(a[k], b[k])
        # a first step is lr * sign(g): gradients that agree to rounding give the same step unless they are zero
        big = np.abs(values(g)[k]) > 1e-6
        assert np.all(np.abs(a[k] - w)[big] <= 1e-2 * 1e-2 + 1e-6)
