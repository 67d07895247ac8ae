"""What Optim.adamW and its C entries refuse, before anything reaches a GPU."""
import ctypes as C

import pytest
import torch

import jax4j_b200 as J
from jax4j_b200 import _lib


def leaf(n, dtype=J.DType.FLOAT32, shape=None):
    """An array over host memory: enough for every check that precedes a launch."""
    return J.ConcreteNDArray._wrap(torch.zeros(n, dtype=dtype.torch), J.Shape(shape or (n,)), dtype, J.Device(None))


def tree(*leaves):
    return J.PyTree.list(*[J.PyTree.leaf(a) for a in leaves])


STEP = leaf(3, J.DType.FLOAT64)


def state(params, bits=32):
    ls = J.PyTrees.flatten(params)
    arrays = ([leaf(_lib.lib().j4c_adamw_q8_words(a.shape().size()), J.DType.INT32) for a in ls] if bits == 8 else
              [leaf(a.shape().size(), a.dtype()) for a in ls for _ in range(2)])
    return J.AdamWState(params, bits, STEP, arrays)


def test_packed_sizes():
    L = _lib.lib()
    assert [L.j4c_adamw_q8_words(n) for n in (-1, 0, 1, 128, 129, 1 << 33)] == [-1, 0, 66, 66, 132, 66 << 26]
    from jax4j_b200.optim import _q8_words
    assert [_q8_words(n) for n in (0, 1, 128, 129, 1 << 33)] == [0, 66, 66, 132, 66 << 26]


def test_states_are_checked():
    p = tree(leaf(5))
    bad = J.IllegalArgumentException
    with pytest.raises(bad, match="8 or 32 bits"):
        J.AdamWState(p, 16, STEP, [])
    with pytest.raises(bad, match="FLOAT32 or FLOAT64"):
        J.AdamWState(tree(leaf(5, J.DType.INT32)), 32, STEP, [])
    with pytest.raises(bad, match="8-bit moments are for FLOAT32"):
        J.AdamWState(tree(leaf(5, J.DType.FLOAT64)), 8, STEP, [])
    with pytest.raises(bad, match="three FLOAT64"):
        J.AdamWState(p, 32, leaf(3), [leaf(5), leaf(5)])
    with pytest.raises(bad, match="take 2 arrays"):
        J.AdamWState(p, 32, STEP, [leaf(5)])
    with pytest.raises(bad, match="array 1 of the state"):
        J.AdamWState(p, 32, STEP, [leaf(5), leaf(6)])
    with pytest.raises(bad, match="array 0 of the state"):
        J.AdamWState(p, 8, STEP, [leaf(66)])
    s = state(p, 8)
    with pytest.raises(bad, match="do not match"):
        s.withArrays([STEP, leaf(65, J.DType.INT32)])
    assert s.withArrays(s.arrays()).stateBits() == 8


def test_steps_are_checked():
    p = tree(leaf(6, shape=(2, 3)), leaf(3))
    s = state(p)
    bad = J.IllegalArgumentException

    def step(params=p, grads=p, st=s, lr=0.1, **k):
        return J.Optim.adamW(params, grads, st, lr, **k)

    with pytest.raises(bad, match="2 parameters, 1 gradients"):
        step(grads=tree(leaf(6)))
    with pytest.raises(bad, match="do not match"):
        step(grads=tree(leaf(6, shape=(3, 2)), leaf(3)))
    with pytest.raises(bad, match="do not match"):
        step(st=state(tree(leaf(6, shape=(2, 3)), leaf(4))))
    with pytest.raises(bad, match="do not match"):
        step(grads=tree(leaf(6, J.DType.FLOAT64, (2, 3)), leaf(3)))
    for k in (dict(beta1=1.0), dict(beta2=-0.1), dict(beta1=float("nan"))):
        with pytest.raises(bad, match="betas"):
            step(**k)
    with pytest.raises(bad, match="eps"):
        step(eps=-1e-8)
    with pytest.raises(bad, match="weight decays"):
        step(weightDecay=[0.1])
    with pytest.raises(bad, match="lr is"):
        step(lr=leaf(2))
    with pytest.raises(bad, match="lr is"):
        step(lr=leaf(1, J.DType.FLOAT64))
    with pytest.raises(bad, match="1 gradients"):
        J.Lax.psumAdamWTree(p, tree(leaf(3)), s, 0.1)

    def traced(x):
        J.Optim.adamW(p, p, s, 0.1)
        return x

    with pytest.raises(J.UnsupportedOperationException, match="between traces"):
        J.JAX.make_jaxpr(traced, leaf(1))


def test_c_entries_refuse_bad_arguments():
    L = _lib.lib()
    fake = C.c_void_p(0x1000)
    one = (C.c_void_p * 1)(0x1000)
    null = (C.c_void_p * 1)(None)
    two = (C.c_void_p * 2)(0x1000, 0x1000)
    n, wd = (C.c_int64 * 1)(4), (C.c_double * 1)(0.0)

    def step(dtype=0, bits=32, count=1, numel=n, w=one, g=one, st=two, wo=one, so=two, decay=wd, steps=fake, out=None,
             b1=0.9, b2=0.999, eps=1e-8):
        rc = L.j4c_adamw_step(dtype, bits, count, numel, w, g, st, wo, so, decay, steps, out, None, 0.1, 1.0, b1, b2,
                              eps, None)
        return rc, L.j4c_last_error().decode()

    for kw, text in ((dict(dtype=2), "FLOAT32 or FLOAT64"), (dict(bits=16), "8 or 32"),
                     (dict(dtype=1, bits=8), "8-bit"), (dict(numel=None), "NULL table"), (dict(count=-1), "NULL table"),
                     (dict(w=null), "NULL pointer"), (dict(st=(C.c_void_p * 2)(0x1000, None)), "NULL pointer"),
                     (dict(numel=(C.c_int64 * 1)(-1)), "negative size"), (dict(steps=None), "steps"),
                     (dict(out=fake), "steps"), (dict(b1=1.0), "betas"), (dict(b2=float("nan")), "betas"),
                     (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps")):
        rc, msg = step(**kw)
        assert rc == _lib.E_INVALID and text in msg, (kw, rc, msg)
    rc = L.j4c_adamw_moments(1, n, one, null, one, None)
    assert rc == _lib.E_INVALID and "NULL pointer" in L.j4c_last_error().decode()


class GpuTensor:
    """Stands in for a tensor on GPU `gpu` where no kernel runs."""

    def __init__(self, gpu):
        self.device = torch.device("cuda", gpu)

    def get_device(self):
        return self.device.index

    def data_ptr(self):
        return 0x1000

    def to(self, device):
        return GpuTensor(device.index)


def on_gpu(gpu, n, dtype=J.DType.FLOAT32):
    return J.ConcreteNDArray._wrap(GpuTensor(gpu), J.Shape(n), dtype, J.Device.cuda(gpu))


@pytest.mark.parametrize("bits", [8, 32])
def test_moments_lie_where_the_state_does(monkeypatch, bits):
    """The moments of a state whose arrays were moved carry the arrays' device, not
    that of the parameters the state was made for."""
    from jax4j_b200 import optim
    monkeypatch.setattr(optim, "call", lambda *a: None)
    monkeypatch.setattr(optim, "stream_of", lambda ordinal: 0)
    monkeypatch.setattr(optim, "_carve", lambda sizes, dtype, device: [GpuTensor(device.index) for _ in sizes])
    p = tree(on_gpu(0, 5), on_gpu(0, 200))

    def arrays(gpu):
        moments = ([on_gpu(gpu, 66, J.DType.INT32), on_gpu(gpu, 132, J.DType.INT32)] if bits == 8 else
                   [on_gpu(gpu, n) for n in (5, 5, 200, 200)])
        return [on_gpu(gpu, 3, J.DType.FLOAT64)] + moments

    first = arrays(0)
    moved = J.AdamWState(p, bits, first[0], first[1:]).withArrays(arrays(1))
    for part in moved.moments():
        for a in J.PyTrees.flatten(part):
            assert a.device() is J.Device.cuda(1) and a.tensor().device.index == 1


@pytest.mark.parametrize("bits", [8, 32])
def test_a_shared_state_goes_where_the_shard_is(monkeypatch, bits):
    """Lax.psumAdamWTree on a shard of another GPU than the state's takes the step
    with the state beside the shard's parameters; on the state's own GPU with the
    state itself."""
    seen, lrs = [], []
    monkeypatch.setattr(J.Optim, "adamW", lambda params, grads, state, lr, **k: seen.append(state) or lrs.append(lr))
    monkeypatch.setattr(J.Lax, "psumTree", lambda grads: grads)
    p = tree(on_gpu(0, 5))
    moments = [on_gpu(0, 66, J.DType.INT32)] if bits == 8 else [on_gpu(0, 5), on_gpu(0, 5)]
    state = J.AdamWState(p, bits, on_gpu(0, 3, J.DType.FLOAT64), moments)
    lr = on_gpu(0, 1)
    J.Lax.psumAdamWTree(p, p, state, lr)
    other = tree(on_gpu(1, 5))
    J.Lax.psumAdamWTree(other, other, state, lr)
    assert seen[0] is state and lrs[0] is lr and lrs[1].tensor().device.index == 1
    for a in seen[1].arrays():
        assert a.device() is J.Device.cuda(1) and a.tensor().device.index == 1
    assert seen[1].stateBits() == bits and [a.dtype() for a in seen[1].arrays()] == [a.dtype() for a in state.arrays()]
    back = seen[1].to(J.Device.cuda(0))
    assert all(a.device() is J.Device.cuda(0) and a.tensor().device.index == 0 for a in back.arrays())


def test_eps_that_the_8_bit_quotient_does_not_take():
    """It is off beyond 2^-126 and 2^126, where a divisor may be eps alone."""
    p = tree(leaf(6))
    L = _lib.lib()
    fake, n, wd = C.c_void_p(0x1000), (C.c_int64 * 1)(0), (C.c_double * 1)(0.0)
    one = (C.c_void_p * 1)(None)
    for eps in (2.0 ** -127, 1e-40, 5e-324, 2.0 ** 126, float("inf")):
        with pytest.raises(J.IllegalArgumentException, match="8-bit moments eps"):
            J.Optim.adamW(p, p, state(p, 8), 0.1, eps=eps)
        rc = L.j4c_adamw_step(0, 8, 1, n, one, one, one, one, one, wd, fake, None, None, 0.1, 1.0, 0.9, 0.999, eps, None)
        assert rc == _lib.E_INVALID and "eps" in L.j4c_last_error().decode()
    for eps in (0.0, 2.0 ** -126, 1e-8, 2.0 ** 125):  # an empty tensor: nothing is launched
        rc = L.j4c_adamw_step(0, 8, 1, n, one, one, one, one, one, wd, fake, None, None, 0.1, 1.0, 0.9, 0.999, eps, None)
        assert rc == _lib.OK, L.j4c_last_error()
