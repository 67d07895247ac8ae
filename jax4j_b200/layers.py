"""Layers that run as single operations: group norm with an activation.

Nothing here has a counterpart in the reference, whose layers are chains of
NDArray operations (examples/MNISTFromScratch.java:103-125).  Under a trace a
layer records one FFI_CALL equation -- the reference's primitive for a
registered function with its own VJP (api/FFI.java:17-51) -- so grad, pmap,
jit, scan and checkpoint compose with it as with any other equation.
"""
from __future__ import annotations

from typing import List, Optional

import torch

from . import _lib
from ._lib import call
from .core import (ConcreteNDArray, DType, IllegalArgumentException, NDArray, Primitive, Shape,
                   UnsupportedOperationException)
from .tracing import Equation, FfiMeta, TracedNDArray, Tracer, to_var

# J4C_ACT_* (include/jax4j_cuda.h)
ACTIVATIONS = {"none": 0, "relu": 1, "tanh": 2, "sigmoid": 3, "silu": 4, "gelu": 5}


def activation_code(name: Optional[str]) -> int:
    code = ACTIVATIONS.get("none" if name is None else name)
    if code is None:
        raise IllegalArgumentException(f"unknown activation {name!r}: one of {', '.join(ACTIVATIONS)}")
    return code


def _apply(meta: FfiMeta, inputs: List[NDArray], out_shape: Shape) -> NDArray:
    """The layer on its arrays, or its equation under a trace."""
    tracer = Tracer.current()
    if tracer is None:
        return meta.forward(inputs, False)[0]
    in_vars = [to_var(x) for x in inputs]
    out = tracer.nextVar(out_shape, in_vars[0].dtype)
    tracer.addEquation(Equation(in_vars, [out], Primitive.FFI_CALL, meta))
    return TracedNDArray(out)


def _device_of(inputs: List[ConcreteNDArray]):
    """The result's device, by the rules of elementwise operations
    (core/ConcreteNDArray.java:261-267)."""
    dev = inputs[0].device()
    for x in inputs[1:]:
        if x._device is not dev:
            first = ConcreteNDArray._wrap(inputs[0]._t, inputs[0]._shape, inputs[0]._dtype, dev)
            dev = first._check_devices(x)
    return dev


def _floating(what: str, first: NDArray, others) -> None:
    if not first.dtype().is_floating():
        raise IllegalArgumentException(f"{what} requires FLOAT32 or FLOAT64 operands, got {first.dtype()}")
    for x in others:
        if x is not None and x.dtype() != first.dtype():
            raise IllegalArgumentException(f"{what} requires operands of one floating dtype, got {first.dtype()} and "
                                           f"{x.dtype()} — use .astype() to convert.")


# ---------------------------------------------------------------------------
# group norm
# ---------------------------------------------------------------------------
def group_norm(x: NDArray, groups: int, gamma: Optional[NDArray], beta: Optional[NDArray], eps: float,
               activation: Optional[str]) -> NDArray:
    d = x.shape().dimensions()
    act = activation_code(activation)
    if len(d) < 2:
        raise IllegalArgumentException(f"groupNorm takes [batch, ..., channels], got {x.shape()}")
    C = d[-1]
    _floating("groupNorm", x, (gamma, beta))
    groups = int(groups)
    if groups < 1 or C < 1 or C % groups:
        raise IllegalArgumentException(f"groupNorm: {C} channels do not divide into {groups} groups")
    for name, p in (("gamma", gamma), ("beta", beta)):
        if p is not None and p.shape().dimensions() != (C,):
            raise IllegalArgumentException(f"groupNorm: {name} is {p.shape()}, the channels are [{C}]")
    if not eps >= 0.0:
        raise IllegalArgumentException(f"groupNorm: eps is not negative, got {eps}")
    inputs = [x] + [p for p in (gamma, beta) if p is not None]
    meta = _GroupNorm(groups, gamma is not None, beta is not None, float(eps), act)
    return _apply(meta, inputs, x.shape())


class _GroupNorm(FfiMeta):
    name = "group_norm"

    def __init__(self, groups: int, has_gamma: bool, has_beta: bool, eps: float, act: int):
        self.groups, self.has_gamma, self.has_beta, self.eps, self.act = groups, has_gamma, has_beta, eps, act

    def _params(self, inputs):
        gamma = inputs[1] if self.has_gamma else None
        beta = inputs[-1] if self.has_beta else None
        return gamma, beta

    @staticmethod
    def _extents(shape: Shape):
        d = shape.dimensions()
        S = 1
        for n in d[1:-1]:
            S *= n
        return d[0], S, d[-1]

    def forward(self, inputs, keep):
        x = inputs[0]
        gamma, beta = self._params(inputs)
        dev = _device_of(inputs)
        B, S, C = self._extents(x._shape)
        t, dt = x._t, x._dtype
        stream = x._stream()
        y = torch.empty(t.numel(), dtype=t.dtype, device=t.device)
        stats = torch.empty(2 * B * self.groups, dtype=t.dtype, device=t.device) if keep else None
        L = _lib.lib()
        need = L.j4c_group_norm_workspace(dt.ordinal, B, S, C, self.groups, 0)
        ws = torch.empty(need, dtype=torch.uint8, device=t.device) if need else None
        mean = stats.data_ptr() if keep and B else None
        call("j4c_group_norm", dt.ordinal, B, S, C, self.groups, t.data_ptr(), gamma._t.data_ptr() if gamma else None,
             beta._t.data_ptr() if beta else None, self.eps, self.act, y.data_ptr(), mean,
             mean + B * self.groups * t.element_size() if mean else None, ws.data_ptr() if need else None, need, stream)
        return ConcreteNDArray._wrap(y, x._shape, dt, dev), stats

    def vjp(self, inputs, out, stats, g, wanted):
        x = inputs[0]
        gamma, beta = self._params(inputs)
        B, S, C = self._extents(x._shape)
        t, dt = x._t, x._dtype
        stream = x._stream()
        dx = torch.empty(t.numel(), dtype=t.dtype, device=t.device)
        want_gamma = self.has_gamma and wanted[1]
        want_beta = self.has_beta and wanted[-1]
        dgamma = torch.empty(C, dtype=t.dtype, device=t.device) if want_gamma else None
        dbeta = torch.empty(C, dtype=t.dtype, device=t.device) if want_beta else None
        need = _lib.lib().j4c_group_norm_workspace(dt.ordinal, B, S, C, self.groups, 1)
        ws = torch.empty(need, dtype=torch.uint8, device=t.device) if need else None
        mean = stats.data_ptr() if B else None
        call("j4c_group_norm_grad", dt.ordinal, B, S, C, self.groups, t.data_ptr(),
             gamma._t.data_ptr() if gamma else None, beta._t.data_ptr() if beta else None, self.act, mean,
             mean + B * self.groups * t.element_size() if mean else None, g._t.data_ptr(), dx.data_ptr(),
             dgamma.data_ptr() if want_gamma else None, dbeta.data_ptr() if want_beta else None,
             ws.data_ptr() if need else None, need, stream)
        grads = [ConcreteNDArray._wrap(dx, x._shape, dt, g._device)]
        if self.has_gamma:
            grads.append(ConcreteNDArray._wrap(dgamma, gamma._shape, dt, g._device) if want_gamma else None)
        if self.has_beta:
            grads.append(ConcreteNDArray._wrap(dbeta, beta._shape, dt, g._device) if want_beta else None)
        return grads

    def batch(self, inputs, batched, batch):
        if not batched[0] or any(batched[1:]):
            raise UnsupportedOperationException("vmap of groupNorm batches x alone")
        # examples are samples side by side
        x = inputs[0]
        d = x.shape().dimensions()
        y = self.forward([x.reshape(Shape((d[0] * d[1],) + d[2:]))] + list(inputs[1:]), False)[0]
        return y.reshape(x.shape())
