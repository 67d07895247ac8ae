"""Layers that run as single operations: a dense layer with its bias, activation
and residual, and group norm with an activation.

Nothing here has a counterpart in the reference, whose layers are chains of
NDArray operations (examples/MNISTFromScratch.java:103-125).  Under a trace a
layer records one FFI_CALL equation -- the reference's primitive for a
registered function with its own VJP (api/FFI.java:17-51) -- so grad, pmap,
jit, scan and checkpoint compose with it as with any other equation.
"""
from __future__ import annotations

import functools
import math
from typing import List, Optional

import torch

from . import _lib
from ._lib import call
from .core import (ConcreteNDArray, DType, IllegalArgumentException, NDArray, Shape, UnsupportedOperationException,
                   _make_splits, _split_of, stream_of)
from .tracing import FfiMeta

# J4C_ACT_* (include/jax4j_cuda.h)
ACTIVATIONS = {"none": 0, "relu": 1, "tanh": 2, "sigmoid": 3, "silu": 4, "gelu": 5}


def activation_code(name: Optional[str]) -> int:
    code = ACTIVATIONS.get("none" if name is None else name)
    if code is None:
        raise IllegalArgumentException(f"unknown activation {name!r}: one of {', '.join(ACTIVATIONS)}")
    return code


def _device_of(inputs: List[ConcreteNDArray]):
    """The result's device, by the rules of elementwise operations
    (core/ConcreteNDArray.java:261-267)."""
    dev = inputs[0]._device
    for x in inputs:
        if x._device is not dev:
            first = ConcreteNDArray._wrap(inputs[0]._t, inputs[0]._shape, inputs[0]._dtype, dev)
            dev = first._check_devices(x)
    return dev


def _floating(what: str, first: NDArray, others) -> None:
    dt = first.dtype()
    if not dt.is_floating():
        raise IllegalArgumentException(f"{what} requires FLOAT32 or FLOAT64 operands, got {dt}")
    for x in others:
        if x is not None and x.dtype() is not dt:
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
    whole = int(groups)
    if whole != groups or whole < 1 or C < 1 or C % whole:
        raise IllegalArgumentException(f"groupNorm: {C} channels do not divide into {groups} groups")
    groups = whole
    for name, p in (("gamma", gamma), ("beta", beta)):
        if p is not None and p.shape().dimensions() != (C,):
            raise IllegalArgumentException(f"groupNorm: {name} is {p.shape()}, the channels are [{C}]")
    if not eps >= 0.0:
        raise IllegalArgumentException(f"groupNorm: eps is not negative, got {eps}")
    inputs = [x] + [p for p in (gamma, beta) if p is not None]
    return _GroupNorm(groups, gamma is not None, beta is not None, float(eps), act).apply(inputs)


class _GroupNorm(FfiMeta):
    name = "group_norm"

    def __init__(self, groups: int, has_gamma: bool, has_beta: bool, eps: float, act: int, sample_axes: int = 1):
        self.groups, self.has_gamma, self.has_beta, self.eps, self.act = groups, has_gamma, has_beta, eps, act
        self.sample_axes = sample_axes  # leading axes that count samples: 1 and those that vmap adds

    def outShape(self, inputs):
        return inputs[0].shape()

    def _params(self, inputs):
        gamma = inputs[1] if self.has_gamma else None
        beta = inputs[-1] if self.has_beta else None
        return gamma, beta

    def _extents(self, shape: Shape):
        d, lead = shape.dimensions(), self.sample_axes
        return math.prod(d[:lead]), math.prod(d[lead:-1]), d[-1]

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
        return _GroupNorm(self.groups, self.has_gamma, self.has_beta, self.eps, self.act,
                          self.sample_axes + 1).run(inputs, False)[0]


# ---------------------------------------------------------------------------
# dense layer
# ---------------------------------------------------------------------------
# FLOAT64 products, and FLOAT32 ones of at most this many multiply-adds, run
# straight from their arrays (j4c_dot_act); the FLOAT32 product on the tcgen05
# tensor cores first splits both operands (three launches more forward), which
# larger ones win back: forward of [1024,1024]x[1024,512] 48 against 60 us, with
# gradients 153 against 167; of [1024,1024]x[1024,1024] 89 against 60 and 270
# against 169.
SMALL_PRODUCT = 1 << 29

# The CUDA cores' tiles have 64 columns whether they hold outputs or not, so these
# count: [8192,4096]x[4096,10] takes 162 us there and 107 on the tensor cores, with
# gradients 474 and 333.  Not where a sum is longer than this, which the tensor
# cores cut into four parts at most: [512,65536]x[65536,10] 200 against 365 us
# ([16384,2048]x[2048,10] 165 against 114, [1024,32768]x[32768,10] 201 against 241
# and with gradients 552 against 425).
TILE_COLUMNS = 64
LONG_SUM = 1 << 15

# As many rows or fewer run there whatever the weight's size: they are bound by
# reading it once, which the splits read, write and read again.
FEW_ROWS = 16


def _small(M: int, K: int, N: int) -> bool:
    if M * K * (-(-N // TILE_COLUMNS) * TILE_COLUMNS) <= SMALL_PRODUCT:
        return True
    return not (M and N and K) or M * K * N <= SMALL_PRODUCT and max(M, K, N) > LONG_SUM


def dense(x: NDArray, w: NDArray, bias: Optional[NDArray], activation: Optional[str],
          residual: Optional[NDArray]) -> NDArray:
    xd, wd, dt = x.shape()._d, w.shape()._d, x.dtype()
    act = ACTIVATIONS.get(activation)
    if act is None:
        act = activation_code(activation)
    if len(xd) < 1 or len(wd) != 2:
        raise IllegalArgumentException(f"dense takes [..., K] and a weight [K, N], got {x.shape()} and {w.shape()}")
    if xd[-1] != wd[0]:
        raise IllegalArgumentException(f"dense: inner dimensions differ ({x.shape()} . {w.shape()})")
    if (not dt._floating or w.dtype() is not dt or bias is not None and bias.dtype() is not dt
            or residual is not None and residual.dtype() is not dt):
        _floating("dense", x, (w, bias, residual))
    inputs = [x, w]
    if bias is not None:
        if bias.shape()._d != wd[1:]:
            raise IllegalArgumentException(f"dense: bias is {bias.shape()}, the outputs are [{wd[1]}]")
        inputs.append(bias)
    if residual is not None:
        if residual.shape()._d != xd[:-1] + wd[1:]:
            raise IllegalArgumentException(f"dense: residual is {residual.shape()}, the output {Shape(xd[:-1] + wd[1:])}")
        inputs.append(residual)
    return _dense_meta(bias is not None, residual is not None, act).apply(inputs)


def _split_product(a, a_kind: str, b, b_kind: str, M: int, K: int, N: int, bias, act: int, residual, z, out: torch.Tensor,
                   stream) -> None:
    """out [M, N] = act(A . B^T + bias) + residual on the tensor cores, with A
    [M, K] and B [N, K] the splits of a and b by rows of these kinds."""
    (ah, al), (bh, bl) = _split_of(a, a_kind), _split_of(b, b_kind)
    call("j4c_dot_split_act", ah.data_ptr(), al.data_ptr(), bh.data_ptr(), bl.data_ptr(), M, K, N, bias, act, residual, z,
         out.data_ptr(), stream)


@functools.lru_cache(maxsize=4096)
def _grad_workspace(gpu: int, dtype: int, M: int, N: int) -> int:
    """j4c_dense_grad_workspace on this GPU (the current one)."""
    return int(_lib.lib().j4c_dense_grad_workspace(dtype, M, N))


class _Dense(FfiMeta):
    name = "dense"

    def __init__(self, has_bias: bool, has_residual: bool, act: int):
        self.has_bias, self.has_residual, self.act = has_bias, has_residual, act

    def outShape(self, inputs):
        return Shape(inputs[0].shape()._d[:-1] + inputs[1].shape()._d[1:])

    def _params(self, inputs):
        return inputs[2] if self.has_bias else None, inputs[-1] if self.has_residual else None

    @staticmethod
    def _extents(inputs):
        K, N = inputs[1]._shape._d
        return math.prod(inputs[0]._shape._d[:-1]), K, N

    # The output tells the slope (and is kept anyway) unless a residual was
    # added to it or the activation is not monotone.
    def _from_output(self) -> bool:
        return not self.has_residual and self.act <= ACTIVATIONS["sigmoid"]

    def forward(self, inputs, keep):
        x, w = inputs[0], inputs[1]
        bias, residual = self._params(inputs)
        dev = _device_of(inputs)
        M, K, N = self._extents(inputs)
        dt, t = x._dtype, x._t
        stream = x._stream()
        x2 = x if len(x._shape._d) == 2 else x.reshape(Shape(M, K))
        out_shape = Shape(x._shape._d[:-1] + (N,))
        keep_z = keep and self.act and not self._from_output()
        y = t.new_empty(M * N)
        z = t.new_empty(M * N) if keep_z else None
        bp = bias._t.data_ptr() if bias is not None else None
        rp = residual._t.data_ptr() if residual is not None else None
        zp = z.data_ptr() if z is not None else None
        if dt is not DType.FLOAT32 or M <= FEW_ROWS or _small(M, K, N):
            call("j4c_dot_act", dt.ordinal, t.data_ptr(), w._t.data_ptr(), M, K, N, 0, 0, bp, self.act, rp, zp, y.data_ptr(),
                 stream)
        else:
            if keep:  # with those that the gradient's products take, each operand's in one pass
                _make_splits(x2, ["r", "t"])
                _make_splits(w, ["t", "r"])
            _split_product(x2, "r", w, "t", M, K, N, bp, self.act, rp, zp, y, stream)
        return ConcreteNDArray._wrap(y, out_shape, dt, dev), ((x2, z) if keep else None)

    def vjp(self, inputs, out, saved, g, wanted):
        x, w = inputs[0], inputs[1]
        x2, z = saved
        (M, K), N = x2._shape._d, w._shape._d[1]
        dt, t, dev = x._dtype, g._t, g._device
        gpu = t.get_device()
        stream = stream_of(gpu)
        want_bias = self.has_bias and wanted[2]
        products = wanted[0] or wanted[1]
        small = dt is not DType.FLOAT32 or _small(M, K, N)
        dz, dbias, lines = t, None, None
        grads: List[Optional[ConcreteNDArray]] = [None, None]
        if want_bias or products:
            # the pass over g, and without splits all of the gradient
            need = _grad_workspace(gpu, dt.ordinal, M, N) if want_bias else 0
            ws = torch.empty(need, dtype=torch.uint8, device=t.device) if need else None
            wp = ws.data_ptr() if need else None
            if self.act:
                dz = torch.empty_like(t)
            if want_bias:
                dbias = torch.empty_like(inputs[2]._t)
            up = (z if z is not None else out._t).data_ptr() if self.act else None
            zp, bp = dz.data_ptr() if self.act else None, dbias.data_ptr() if want_bias else None
            if small and products:
                dx = torch.empty_like(x2._t) if wanted[0] else None
                dw = torch.empty_like(w._t) if wanted[1] else None
                call("j4c_dense_backward", dt.ordinal, x2._t.data_ptr(), w._t.data_ptr(), M, K, N, t.data_ptr(), up, self.act,
                     int(z is None), zp, dx.data_ptr() if wanted[0] else None, dw.data_ptr() if wanted[1] else None, bp,
                     wp, need, stream)
                grads = [ConcreteNDArray._wrap(dx, x._shape, dt, dev) if wanted[0] else None,
                         ConcreteNDArray._wrap(dw, w._shape, dt, dev) if wanted[1] else None]
            else:
                if products:
                    lines = torch.empty(M + N + 1, dtype=torch.int32, device=t.device)
                call("j4c_dense_grad", dt.ordinal, M, N, t.data_ptr(), up, self.act, int(z is None), zp, bp,
                     lines.data_ptr() if lines is not None else None, wp, need, stream)
        if products and not small:
            d = ConcreteNDArray._wrap(dz, Shape(M, N), dt, dev)
            d._lines = lines
            _make_splits(d, (["r"] if wanted[0] else []) + (["t"] if wanted[1] else []))
            # dx = dz . w^T and dw = x^T . dz, every operand read along its rows
            if wanted[0]:
                dx = torch.empty_like(x2._t)
                _split_product(d, "r", w, "r", M, N, K, None, 0, None, None, dx, stream)
                grads[0] = ConcreteNDArray._wrap(dx, x._shape, dt, dev)
            if wanted[1]:
                dw = torch.empty_like(w._t)
                _split_product(x2, "t", d, "t", K, M, N, None, 0, None, None, dw, stream)
                grads[1] = ConcreteNDArray._wrap(dw, w._shape, dt, dev)
        if self.has_bias:
            grads.append(ConcreteNDArray._wrap(dbias, inputs[2]._shape, dt, dev) if want_bias else None)
        if self.has_residual:
            grads.append(g)
        return grads

    def batch(self, inputs, batched, batch):
        # x alone, or x and the residual: examples are rows side by side
        if not batched[0] or batched[1] or (self.has_bias and batched[2]) or (self.has_residual and not batched[-1]):
            raise UnsupportedOperationException("vmap of dense batches x, together with the residual")
        return self.run(inputs, False)[0]


@functools.lru_cache(maxsize=None)
def _dense_meta(has_bias: bool, has_residual: bool, act: int) -> _Dense:
    return _Dense(has_bias, has_residual, act)  # 24 of them, which hold nothing else
