"""What the fused layers and their C entries refuse before anything reaches a
GPU, and how they are traced."""
import ctypes as C

import pytest
import torch

import jax4j_b200 as J
from jax4j_b200 import _lib
from jax4j_b200.layers import ACTIVATIONS


def leaf(*shape, dtype=J.DType.FLOAT32):
    s = J.Shape(*shape)
    return J.ConcreteNDArray._wrap(torch.zeros(s.size(), dtype=dtype.torch), s, dtype, J.Device(None))


def test_activation_codes_match_the_header():
    import os
    import re
    src = open(os.path.join(os.path.dirname(_lib.__file__), "..", "include", "jax4j_cuda.h")).read()
    codes = {m.group(1).lower(): int(m.group(2)) for m in re.finditer(r"#define J4C_ACT_(\w+) (\d)", src)}
    assert codes == ACTIVATIONS


def test_group_norm_refusals():
    bad = J.IllegalArgumentException
    x = leaf(2, 3, 8)
    for args, text in (((x, 3), "do not divide"), ((x, 0), "do not divide"), ((x, -2), "do not divide"),
                       ((leaf(8), 2), "batch"), ((leaf(2, 0), 1), "do not divide"),
                       ((x, 2, leaf(4)), "gamma is"), ((x, 2, None, leaf(1, 8)), "beta is"),
                       ((leaf(2, 8, dtype=J.DType.INT32), 2), "FLOAT32 or FLOAT64"),
                       ((x, 2, leaf(8, dtype=J.DType.FLOAT64)), "one floating dtype")):
        with pytest.raises(bad, match=text):
            J.Nn.groupNorm(*args)
    with pytest.raises(bad, match="activation"):
        J.Nn.groupNorm(x, 2, activation="swish")
    for eps in (-1e-5, float("nan")):
        with pytest.raises(bad, match="eps"):
            J.Nn.groupNorm(x, 2, eps=eps)


def test_dense_refusals():
    bad = J.IllegalArgumentException
    x, w = leaf(2, 3, 8), leaf(8, 5)
    for args, text in (((x, leaf(7, 5)), "inner dimensions"), ((x, leaf(8)), "weight"), ((leaf(), w), "takes"),
                       ((x, w, leaf(8)), "bias is"), ((x, w, leaf(1, 5)), "bias is"),
                       ((x, w, None, "none", leaf(2, 3, 8)), "residual is"), ((x, w, None, "none", leaf(5)), "residual is"),
                       ((x, w, None, "selu"), "activation"), ((leaf(2, 8, dtype=J.DType.INT64), w), "FLOAT32 or FLOAT64"),
                       ((x, leaf(8, 5, dtype=J.DType.FLOAT64)), "one floating dtype"),
                       ((x, w, leaf(5, dtype=J.DType.FLOAT64)), "one floating dtype")):
        with pytest.raises(bad, match=text):
            J.Nn.dense(*args)


def test_vjp_refusals():
    _, pull = J.JAX.vjp(lambda a: a, leaf(3))
    for seeds, text in (((), "as many cotangents"), ((leaf(4),), "cotangent"), ((leaf(3, dtype=J.DType.FLOAT64),), "cotangent")):
        with pytest.raises(J.IllegalArgumentException, match=text):
            pull(*seeds)


def test_dense_c_entries_refuse_bad_arguments():
    L = _lib.lib()
    fake = C.c_void_p(0x1000)

    def told(rc, text, code=_lib.E_INVALID):
        assert rc == code and text in L.j4c_last_error().decode(), (rc, L.j4c_last_error())

    told(L.j4c_dot_act(0, fake, fake, -1, 2, 3, 0, 0, None, 0, None, None, fake, None), "negative")
    told(L.j4c_dot_act(0, fake, fake, 1, 2, 3, 0, 0, None, 6, None, None, fake, None), "activation")
    told(L.j4c_dot_act(0, fake, None, 1, 2, 3, 0, 0, None, 0, None, None, fake, None), "NULL")
    told(L.j4c_dot_act(0, fake, fake, 1, 2, 3, 0, 0, None, 0, None, None, None, None), "NULL")
    told(L.j4c_dot_act(0, fake, fake, 1 << 33, 2, 3, 0, 0, None, 0, None, None, fake, None), "too many", _lib.E_UNSUPPORTED)
    told(L.j4c_dot_split_act(fake, fake, fake, fake, 2, 0, 3, None, 0, None, None, fake, None), "K = 0")
    told(L.j4c_dot_split_act(fake, None, fake, fake, 2, 4, 3, None, 0, None, None, fake, None), "NULL")
    told(L.j4c_dot_split_act(fake, fake, fake, fake, 2, 4, 3, None, -1, None, None, fake, None), "activation")
    told(L.j4c_dot_act(2, fake, fake, 1, 2, 3, 0, 0, None, 0, None, None, fake, None), "FLOAT32 or FLOAT64")
    told(L.j4c_dense_backward(2, fake, fake, 2, 3, 4, fake, None, 0, 0, None, fake, fake, None, None, 0, None), "FLOAT32 or FLOAT64")
    told(L.j4c_dense_grad(0, 2, 3, fake, None, 3, 0, fake, None, None, None, 0, None), "NULL")
    told(L.j4c_dense_grad(0, 2, 3, fake, fake, 5, 1, fake, None, None, None, 0, None), "does not tell")
    told(L.j4c_dense_grad(1, 2, 3, fake, fake, 2, 1, fake, None, fake, None, 0, None), "line words")
    told(L.j4c_dense_backward(0, fake, fake, 2, 3, 4, fake, None, 0, 0, None, None, None, fake, None, 0, None), "neither product")
    told(L.j4c_dense_backward(0, fake, fake, 2, 3, 4, fake, fake, 5, 0, None, fake, fake, None, None, 0, None), "NULL")
    told(L.j4c_dense_backward(0, fake, None, 2, 3, 4, fake, None, 0, 0, None, fake, fake, None, None, 0, None), "NULL")
    told(L.j4c_dense_grad(0, 2000, 3, fake, fake, 2, 1, fake, fake, None, None, 0, None), "workspace")


def test_layers_are_one_equation():
    jaxpr = J.JAX.make_jaxpr(lambda a: J.Nn.groupNorm(a, 2, leaf(8), activation="silu").tanh(), leaf(2, 3, 8))
    kinds = [e.primitive for e in jaxpr.equations]
    assert kinds == [J.Primitive.FFI_CALL, J.Primitive.TANH]
    assert jaxpr.outVars[0].shape == J.Shape(2, 3, 8)
    assert "group_norm(groups=2" in repr(jaxpr)
    with pytest.raises(J.UnsupportedOperationException, match="inside a trace"):
        J.JAX.make_jaxpr(lambda a: J.JAX.vjp(lambda b: b, a)[0], leaf(3))


def test_c_entries_refuse_bad_arguments():
    L = _lib.lib()
    fake = C.c_void_p(0x1000)

    def norm(dtype=0, B=2, S=3, c=8, G=2, x=fake, eps=1e-5, act=0, y=fake, mean=None, rstd=None):
        rc = L.j4c_group_norm(dtype, B, S, c, G, x, None, None, eps, act, y, mean, rstd, None, 0, None)
        return rc, L.j4c_last_error().decode()

    for kw, text in ((dict(dtype=2), "FLOAT32 or FLOAT64"), (dict(B=-1), "bad extents"), (dict(c=0), "bad extents"),
                     (dict(G=3), "do not divide"), (dict(G=0), "do not divide"), (dict(eps=-1.0), "eps"),
                     (dict(eps=float("nan")), "eps"), (dict(act=6), "activation"), (dict(act=-1), "activation"),
                     (dict(x=None), "NULL"), (dict(y=None), "NULL"), (dict(mean=fake), "go together"),
                     (dict(S=1 << 31), "not supported"), (dict(S=100000), "workspace")):
        rc, msg = norm(**kw)
        assert rc == _lib.E_INVALID and text in msg, (kw, rc, msg)
    assert norm(B=0)[0] == _lib.OK
    rc = L.j4c_group_norm_grad(0, 2, 3, 8, 2, fake, None, None, 0, fake, fake, fake, fake, None, None, None, 0, None)
    assert rc == _lib.E_INVALID and "workspace" in L.j4c_last_error().decode()
    rc = L.j4c_group_norm_grad(0, 2, 3, 8, 2, fake, None, None, 0, fake, None, fake, fake, None, None, fake, 1 << 20, None)
    assert rc == _lib.E_INVALID and "NULL" in L.j4c_last_error().decode()


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("M,K,N", [(0, 3, 4), (2, 0, 4), (2, 3, 0), (0, 0, 4), (0, 3, 0)])
def test_empty_gradients_are_no_refusal(dtype, M, K, N):
    """The pointer of an empty array is NULL, as that of a gradient that is not wanted."""
    fake = C.c_void_p(0x1000)
    rc = _lib.lib().j4c_dense_backward(dtype, fake, fake, M, K, N, fake, None, 0, 0, None, None, None, None, None, 0, None)
    assert rc == _lib.OK, _lib.lib().j4c_last_error()


def _layers():
    w, b = leaf(8, 5), leaf(5)
    return {"dense": (lambda a: J.Nn.dense(a, w, b, "silu"), (8,), (5,)),
            "residual": (lambda a: J.Nn.dense(a, leaf(8, 8), None, "gelu", a), (2, 8), (2, 8)),
            "group norm": (lambda a: J.Nn.groupNorm(a, 2, leaf(8), activation="tanh"), (2, 3, 8), (2, 3, 8))}


@pytest.mark.parametrize("name", ["dense", "residual", "group norm"])
def test_vmap_inside_a_trace_is_recorded(name):
    """As vmap of elementwise operations is: jit and grad of a mapped layer, and vmap of vmap."""
    f, shape, out = _layers()[name]
    for maps in (1, 2):
        g = f
        for _ in range(maps):
            g = J.JAX.vmap(g)
        lead = (4, 6)[:maps]
        jaxpr = J.JAX.make_jaxpr(lambda a: g(a).tanh(), leaf(*lead, *shape))
        assert [e.primitive for e in jaxpr.equations] == [J.Primitive.FFI_CALL, J.Primitive.TANH]
        assert jaxpr.outVars[0].shape == J.Shape(*lead, *out)
        if name == "group norm":  # every example's samples keep their own groups
            assert jaxpr.equations[0].metadata._extents(J.Shape(*lead, *shape)) == (2 * 4 * (6 if maps == 2 else 1), 3, 8)


@pytest.mark.parametrize("name", ["dense", "residual", "group norm"])
def test_interpretation_inside_a_trace_is_recorded_and_gradients_refused(monkeypatch, name):
    from jax4j_b200 import grad
    f, shape, out = _layers()[name]
    inner = J.JAX.make_jaxpr(f, leaf(*shape))
    outer = J.JAX.make_jaxpr(lambda a: grad.forward_interpret(inner, [a])[0], leaf(*shape))
    assert [e.primitive for e in outer.equations] == [J.Primitive.FFI_CALL] and outer.outVars[0].shape == J.Shape(*out)
    monkeypatch.setattr(grad, "ones", lambda s, dtype, device=None: leaf(*s.dimensions()))
    with pytest.raises(J.UnsupportedOperationException, match="inside a trace"):
        J.JAX.make_jaxpr(lambda a: J.JAX.grad(f)(a), leaf(*shape))


def test_which_products_run_straight_from_their_arrays():
    """Whole tiles of 64 columns count, except where a sum is long."""
    from jax4j_b200 import layers
    for shape in ((1024, 1024, 512), (256, 784, 512), (8192, 1024, 10), (2048, 4096, 64), (64, 1000000, 8),
                  (1000000, 8, 8), (512, 65536, 10), (0, 1 << 20, 1 << 20), (1 << 20, 0, 1 << 20), (1 << 20, 1 << 20, 0)):
        assert layers._small(*shape), shape
    for shape in ((1025, 1024, 512), (8192, 4096, 10), (16384, 2048, 10), (8192, 4096, 1), (4096, 4096, 30),
                  (64, 1000000, 9)):
        assert not layers._small(*shape), shape


def test_group_norm_refuses_half_a_group():
    x = leaf(2, 3, 8)
    for groups in (2.5, 0.5, 1.999):
        with pytest.raises(J.IllegalArgumentException, match="do not divide"):
            J.Nn.groupNorm(x, groups)
    jaxpr = J.JAX.make_jaxpr(lambda a: J.Nn.groupNorm(a, 2.0), x)  # a whole number of another type is one
    assert "group_norm(groups=2," in repr(jaxpr)


def test_concrete_values_inside_a_trace_are_computed(monkeypatch):
    """A Jaxpr interpreted on closed-over arrays inside a trace gives arrays, and
    its gradient too; the layers' own entries record."""
    from jax4j_b200 import grad, layers
    done = []
    monkeypatch.setattr(layers, "call", lambda name, *a: done.append(name))
    monkeypatch.setattr(layers, "stream_of", lambda gpu: 0)
    monkeypatch.setattr(J.ConcreteNDArray, "_stream", lambda self: 0)
    monkeypatch.setattr(layers, "_grad_workspace", lambda *a: 0)
    x = leaf(4, 8)
    w, g = leaf(8, 5).to(x.device()), leaf(4, 5).to(x.device())
    inner = J.JAX.make_jaxpr(lambda a: J.Nn.dense(a, w, None, "tanh"), x)
    seen = []

    def outer(a):
        seen.append(grad.forward_interpret(inner, [x])[0])
        seen.append(grad.backward_interpret(inner, [x], [g])[0])
        return J.Nn.dense(x, w)  # recorded, of two constants

    jaxpr = J.JAX.make_jaxpr(outer, leaf(1))
    assert all(isinstance(s, J.ConcreteNDArray) for s in seen) and [s.shape() for s in seen] == [J.Shape(4, 5), J.Shape(4, 8)]
    assert done == ["j4c_dot_act", "j4c_dot_act", "j4c_dense_backward"]
    assert [e.primitive for e in jaxpr.equations] == [J.Primitive.FFI_CALL]
