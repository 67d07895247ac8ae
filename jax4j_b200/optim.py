"""Optimisers with state: the AdamW step of a whole parameter tree.

The reference updates parameters with elementwise arithmetic on each leaf
(examples/MNISTFromScratch.java:103-136); an optimiser with moments has no
counterpart there.  A step is one launch for every leaf of the tree
(j4c_adamw_step) and, like every operation on arrays, functional: it returns
new parameters and a new state and leaves its arguments as they were.

    state = Optim.adamWInit(params)                  # or stateBits=8
    params, state = Optim.adamW(params, grads, state, lr=1e-3)

The count of steps lives on the GPU with the moments, so a step recorded in a
CUDA graph counts on when it is replayed: `state.arrays()` are the arrays to
carry (graphs.CapturedStep's `donate`), `state.withArrays` puts them back.
"""
from __future__ import annotations

import ctypes as C
from typing import List, Sequence, Tuple, Union

import torch

from ._lib import call
from .core import (ConcreteNDArray, Device, DType, IllegalArgumentException, IllegalStateException, NDArray, Shape,
                   UnsupportedOperationException, stream_of)
from .pytree import PyTree, PyTrees
from .tracing import Tracer


class _Leaf:
    """What a state remembers of a parameter: no reference to its values."""

    __slots__ = ("shape", "dtype", "size")

    def __init__(self, a: NDArray):
        self.shape, self.dtype, self.size = a.shape(), a.dtype(), a.shape().size()


def _q8_words(n: int) -> int:
    """j4c_adamw_q8_words: per 128 elements 2 x 32 words of codes and 2 steps."""
    return (n + 127) // 128 * 66


class AdamWState:
    """The moments of a parameter tree and the count of steps taken.

    stateBits 32 holds, per leaf, m and v in the leaf's dtype (FLOAT32 or
    FLOAT64); stateBits 8 (FLOAT32 leaves) holds them in 8 bits as one INT32
    array of packed words per leaf, whose layout include/jax4j_cuda.h gives:
    2.06 bytes per parameter instead of 8, each first moment within 2^-4 and
    each second moment's root within 2^-5 of its value, block steps aside.

    `step` is a FLOAT64 array of three: the steps taken and the betas to that
    power (what the bias corrections need).  `arrays` are, leaf by leaf in
    PyTrees.flatten order, m and v (32) or the packed words (8)."""

    __slots__ = ("_tree", "_leaves", "_bits", "_step", "_arrays")

    def __init__(self, params: PyTree, stateBits: int, step: ConcreteNDArray, arrays: Sequence[ConcreteNDArray]):
        leaves = [_Leaf(a) for a in PyTrees.flatten(params)]
        if stateBits not in (8, 32):
            raise IllegalArgumentException(f"AdamW: moments are held in 8 or 32 bits, got {stateBits}")
        for l in leaves:
            if not l.dtype.is_floating():
                raise IllegalArgumentException(f"AdamW requires FLOAT32 or FLOAT64 parameters, got {l.dtype}")
            if stateBits == 8 and l.dtype != DType.FLOAT32:
                raise IllegalArgumentException(f"AdamW: 8-bit moments are for FLOAT32 parameters, got {l.dtype}")
        if step.dtype() != DType.FLOAT64 or step.shape().size() != 3:
            raise IllegalArgumentException(f"AdamW: the step is three FLOAT64 values, got {step.shape()} {step.dtype()}")
        arrays = list(arrays)
        per = 1 if stateBits == 8 else 2
        if len(arrays) != per * len(leaves):
            raise IllegalArgumentException(f"AdamW: {len(leaves)} parameters take {per * len(leaves)} arrays of "
                                           f"{stateBits}-bit moments, got {len(arrays)}")
        for i, a in enumerate(arrays):
            l = leaves[i // per]
            dt, n = (DType.INT32, _q8_words(l.size)) if stateBits == 8 else (l.dtype, l.size)
            if a.dtype() is not dt or a.shape().size() != n:
                raise IllegalArgumentException(f"AdamW: array {i} of the state is {a.shape()} {a.dtype()}, "
                                               f"parameter {i // per} {l.shape} takes {n} x {dt}")
        self._set(PyTrees.unflatten(params, leaves), leaves, stateBits, step, arrays)

    def _set(self, tree, leaves, bits, step, arrays) -> "AdamWState":
        self._tree, self._leaves, self._bits, self._step, self._arrays = tree, leaves, bits, step, arrays
        return self

    def stateBits(self) -> int:
        return self._bits

    def step(self) -> ConcreteNDArray:
        return self._step

    def arrays(self) -> List[ConcreteNDArray]:
        """The step, then the moments' arrays: everything a step updates."""
        return [self._step] + list(self._arrays)

    def withArrays(self, arrays: Sequence[ConcreteNDArray]) -> "AdamWState":
        """This state with other values: `arrays` as arrays() lists them."""
        mine = self.arrays()
        arrays = list(arrays)
        if len(arrays) != len(mine) or any(a.dtype() != b.dtype() or a.shape().size() != b.shape().size()
                                           for a, b in zip(arrays, mine)):
            raise IllegalArgumentException("AdamW: the arrays do not match those of the state")
        return AdamWState.__new__(AdamWState)._set(self._tree, self._leaves, self._bits, arrays[0], arrays[1:])

    def to(self, device: Device) -> "AdamWState":
        """This state on `device` (ConcreteNDArray.to for every array: copied
        only if the device is another GPU)."""
        return self.withArrays([a.to(device) for a in self.arrays()])

    def moments(self) -> Tuple[PyTree, PyTree]:
        """(m, v) as trees of the parameters' shapes; for 8-bit moments the
        FLOAT32 values that the codes stand for, one launch for all leaves."""
        ls = self._leaves
        if self._bits == 32:
            return (PyTrees.unflatten(self._tree, self._arrays[0::2]), PyTrees.unflatten(self._tree, self._arrays[1::2]))
        if not ls:
            return self._tree, self._tree
        _one_gpu(self._arrays)
        dev = self._arrays[0].tensor().device
        stream = stream_of(dev.index)
        out = _carve([l.size for l in ls] * 2, torch.float32, dev)
        n = len(ls)
        call("j4c_adamw_moments", n, (C.c_int64 * n)(*[l.size for l in ls]), _pointers(self._arrays),
             (C.c_void_p * n)(*[t.data_ptr() for t in out[:n]]), (C.c_void_p * n)(*[t.data_ptr() for t in out[n:]]),
             stream)
        trees = [PyTrees.unflatten(self._tree, [ConcreteNDArray._wrap(t, l.shape, DType.FLOAT32, a._device)
                                                for t, l, a in zip(part, ls, self._arrays)])
                 for part in (out[:n], out[n:])]
        return trees[0], trees[1]


def _pointers(arrays) -> C.Array:
    return (C.c_void_p * len(arrays))(*[a._t.data_ptr() for a in arrays])


def _carve(sizes: List[int], dtype: torch.dtype, device) -> List[torch.Tensor]:
    """Uninitialised flat tensors of these sizes from one allocation, each on
    a 256-byte boundary (one allocator call and one view call for a tree)."""
    unit = 256 // dtype.itemsize
    cuts = []
    for n in sizes:
        cuts += (n, -n % unit)
    return torch.split_with_sizes(torch.empty(sum(cuts), dtype=dtype, device=device), cuts)[0::2]


def _one_gpu(arrays) -> None:
    first = arrays[0]._t.get_device()
    for a in arrays:
        if a._t.get_device() != first:
            raise IllegalStateException(f"AdamW: the tree's arrays lie on different GPUs ({arrays[0]._t.device} and "
                                        f"{a._t.device})")


class Optim:
    @staticmethod
    def adamWInit(params: PyTree, stateBits: int = 32) -> AdamWState:
        """The state before the first step: moments of zero, next to their
        parameters.  See AdamWState for stateBits."""
        leaves = PyTrees.flatten(params)
        arrays = []
        for a in leaves:
            if not isinstance(a, ConcreteNDArray):
                raise UnsupportedOperationException("AdamW takes concrete arrays, not traced ones")
            n, dt = a.shape().size(), a.dtype()
            if stateBits == 8:
                w = _q8_words(n)
                arrays.append(ConcreteNDArray.full(Shape(w), 0, DType.INT32, a.device()))
            else:
                arrays += [ConcreteNDArray.full(a.shape(), 0.0, dt, a.device()) for _ in range(2)]
        dev = leaves[0].device() if leaves else Device.defaultDevice()
        step = ConcreteNDArray.of([0.0, 1.0, 1.0], dtype=DType.FLOAT64, device=dev)
        return AdamWState(params, stateBits, step, arrays)

    @staticmethod
    def adamW(params: PyTree, grads: PyTree, state: AdamWState, lr: Union[float, ConcreteNDArray], beta1: float = 0.9,
              beta2: float = 0.999, eps: float = 1e-8, weightDecay: Union[float, Sequence[float]] = 0.01,
              scale: float = 1.0) -> Tuple[PyTree, AdamWState]:
        """One AdamW step: (new parameters, new state).  For every element,
        with g' = g * scale and t this step's number,

            m' = beta1 m + (1 - beta1) g'        v' = beta2 v + (1 - beta2) g'^2
            w' = w - lr weightDecay w - lr (m' / (1 - beta1^t)) / (sqrt(v' / (1 - beta2^t)) + eps)

        in the leaf's dtype, each product and sum rounded on its own.  lr is a
        number or a FLOAT32 array of one element on the GPU (a schedule that a
        recorded step can follow); weightDecay a number or one per leaf, in
        PyTrees.flatten order; scale e.g. 1/D for summed gradients.

        The new parameters of a dtype are views of one allocation, and so are
        the new moments: a leaf that is kept alone keeps the memory of all."""
        if Tracer.current() is not None:
            raise UnsupportedOperationException("Optim.adamW is a step between traces, not part of one")
        pl, gl = PyTrees.flatten(params), PyTrees.flatten(grads)
        ls = state._leaves
        n = len(pl)
        if len(gl) != n or len(ls) != n:
            raise IllegalArgumentException(f"adamW: {n} parameters, {len(gl)} gradients, a state of {len(ls)} parameters")
        for w, g, l in zip(pl, gl, ls):
            if not (isinstance(w, ConcreteNDArray) and isinstance(g, ConcreteNDArray)):
                raise UnsupportedOperationException("AdamW takes concrete arrays, not traced ones")
            d, dt = w._shape._d, w._dtype
            if g._shape._d != d or l.shape._d != d or g._dtype is not dt or l.dtype is not dt:
                raise IllegalArgumentException(f"adamW: parameter {w._shape} {w._dtype}, gradient {g._shape} {g._dtype} "
                                               f"and state {l.shape} {l.dtype} do not match")
        if not (0.0 <= beta1 < 1.0 and 0.0 <= beta2 < 1.0):
            raise IllegalArgumentException(f"adamW: betas lie in [0, 1), got {beta1} and {beta2}")
        if not eps >= 0.0:
            raise IllegalArgumentException(f"adamW: eps is not negative, got {eps}")
        if state._bits == 8 and eps and not 2.0 ** -126 <= eps <= 2.0 ** 125:
            raise IllegalArgumentException(f"adamW: with 8-bit moments eps is 0 or from 2^-126 to 2^125, got {eps}")
        wd = [float(x) for x in weightDecay] if isinstance(weightDecay, (list, tuple)) else [float(weightDecay)] * n
        if len(wd) != n:
            raise IllegalArgumentException(f"adamW: {len(wd)} weight decays for {n} parameters")
        lr_dev = None
        if isinstance(lr, NDArray):
            if not isinstance(lr, ConcreteNDArray) or lr.dtype() != DType.FLOAT32 or lr.shape().size() != 1:
                raise IllegalArgumentException("adamW: lr is a number or one FLOAT32 value")
            lr_dev, lr = lr, 0.0
        _one_gpu([state._step, *pl, *gl, *state._arrays] + ([lr_dev] if lr_dev is not None else []))
        dev = state._step._t.device
        stream = stream_of(dev.index)
        step = torch.empty(3, dtype=torch.float64, device=dev)
        new_w: List = [None] * n
        per = 1 if state._bits == 8 else 2
        new_s: List = [None] * (per * n)
        # one launch per dtype (a tree of one dtype: one launch); the first advances the step
        kinds = [(dt, [i for i in range(n) if pl[i]._dtype is dt]) for dt in (DType.FLOAT32, DType.FLOAT64)]
        kinds = [k for k in kinds if k[1]] or [(DType.FLOAT32, [])]
        steps_out = step.data_ptr()
        wrap = ConcreteNDArray._wrap
        for dt, idx in kinds:
            k, all_of = len(idx), len(idx) == n
            sizes = [ls[i].size for i in idx]
            ws = _carve(sizes, dt.torch, dev)
            ss = (_carve([_q8_words(s) for s in sizes], torch.int32, dev) if per == 1 else
                  _carve([s for s in sizes for _ in range(2)], dt.torch, dev))
            pk, gk = (pl, gl) if all_of else ([pl[i] for i in idx], [gl[i] for i in idx])
            old = state._arrays if all_of else [state._arrays[per * i + j] for i in idx for j in range(per)]
            call("j4c_adamw_step", dt.ordinal, state._bits, k, (C.c_int64 * k)(*sizes), _pointers(pk), _pointers(gk),
                 _pointers(old), (C.c_void_p * k)(*[t.data_ptr() for t in ws]),
                 (C.c_void_p * (per * k))(*[t.data_ptr() for t in ss]), (C.c_double * k)(*[wd[i] for i in idx]),
                 state._step._t.data_ptr(), steps_out, lr_dev._t.data_ptr() if lr_dev is not None else None, float(lr),
                 float(scale), float(beta1), float(beta2), float(eps), stream)
            steps_out = None
            for i, w, t in zip(idx, pk, ws):
                new_w[i] = wrap(t, w._shape, dt, w._device)
            for j, (a, t) in enumerate(zip(old, ss)):
                new_s[per * idx[j // per] + j % per] = wrap(t, a._shape, a._dtype, a._device)
        new_step = ConcreteNDArray._wrap(step, state._step._shape, DType.FLOAT64, state._step._device)
        return (PyTrees.unflatten(params, new_w),
                AdamWState.__new__(AdamWState)._set(state._tree, ls, state._bits, new_step, new_s))
