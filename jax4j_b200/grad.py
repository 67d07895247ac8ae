"""Reverse-mode AD interpreter (api/Grad.java of the reference).

The interpreter itself stays host-side, as in the reference: it walks a
traced Jaxpr forward (fillForwardValues, Grad.java:192-211) and backward
(doBackward, Grad.java:154-189) applying the VJP rules of
Grad.computeVJPs (Grad.java:341-472).  What changes is where the work
runs: every rule is a sequence of libjax4j_cuda kernels on resident
buffers, and the host helpers the reference runs through toFloatArray()
(broadcastLike :539-582, reluGrad :585-598, axisBroadcastLike :608-641,
transpose :643-664, maxMinGrad :500-530) are device ops.

Two evaluation shortcuts keep the results identical to the reference's
rules while doing less work:
  * a cotangent is computed only for equation inputs that depend on a
    differentiated input (the reference computes and then discards the
    rest, e.g. the DOT VJP w.r.t. a constant data batch);
  * TANH/SIGMOID/EXP VJPs reuse the forward output instead of recomputing
    the same deterministic kernel on the same input.
With fusion on, the elementwise parts of the rules are deferred inside the
backward walk and evaluated as generated kernels (lazy.py).
"""
from __future__ import annotations

import os
import threading
from typing import Callable, Dict, List

import torch

from . import lazy
from .lazy import Deferred, materialize

from ._lib import call, dims as _dims
from .core import (ConcreteNDArray, DType, IllegalArgumentException, NDArray, Primitive, Shape,
                   UnsupportedOperationException, _dot_raw)
from .tracing import (AxisMeta, CheckpointMeta, CondMeta, Jaxpr, PmapMeta, ScanMeta, Tracer, TracedNDArray, Var,
                      WhileMeta)


# ---------------------------------------------------------------------------
# constants (Grad.java:841-903)
# ---------------------------------------------------------------------------
def _float_or_default(dtype: DType) -> DType:
    return dtype if dtype._floating else DType.FLOAT32


_CONSTS: Dict[tuple, ConcreteNDArray] = {}


def _scalar_like(v: float, like: NDArray, dtype: DType = None) -> ConcreteNDArray:
    """A [1] constant next to `like`.  Constants are immutable, so each
    (value, dtype, device) is made once -- outside a stream capture, where
    making it waits for its fill -- and reused."""
    dtype = dtype or like.dtype()
    dev = like.device()
    key = (float(v), dtype, dev.ordinal() if dev is not None else None)
    c = _CONSTS.get(key)
    if c is not None:
        return c
    c = ConcreteNDArray.scalar(v, dtype, dev)
    if not torch.cuda.is_current_stream_capturing():
        torch.cuda.current_stream(c.tensor().device).synchronize()
        _CONSTS[key] = c
    return c


# Deferred (fused) cotangents are built only inside the backward walk, per thread.
_lazy_scope = threading.local()


def _lazy_on() -> bool:
    return FUSION and lazy.ENABLED and getattr(_lazy_scope, "depth", 0) > 0


def ones(shape: Shape, dtype: DType, device=None) -> ConcreteNDArray:
    return ConcreteNDArray.full(shape, 1.0, _float_or_default(dtype), device)


def zeros(shape: Shape, dtype: DType, device=None) -> ConcreteNDArray:
    return ConcreteNDArray.full(shape, 0.0, _float_or_default(dtype), device)


def zeros_like(x: NDArray) -> ConcreteNDArray:
    return zeros(x.shape(), x.dtype(), x.device())


def _zeros_for(var: Var, like: ConcreteNDArray) -> ConcreteNDArray:
    """Zero cotangent of a Var (Grad.zerosLike, Grad.java:884-887) next to `like`."""
    return zeros(var.shape, var.dtype, like.device())


# ---------------------------------------------------------------------------
# device versions of the Grad.java host helpers
# ---------------------------------------------------------------------------
def broadcast_like(g: NDArray, target_shape: Shape) -> NDArray:
    """Grad.broadcastLike (Grad.java:539-582): copy/reshape, expand, or sum down."""
    gs = g.shape()
    if gs == target_shape:
        return g
    if _lazy_on() and gs.size() != target_shape.size():
        d = (lazy.expand(g, target_shape) if target_shape.size() > gs.size()
             else lazy.row_sum(g, target_shape))
        if d is not None:
            return d
    g = materialize(g)
    if gs.size() == target_shape.size():
        return g.reshape(target_shape)
    out = torch.empty(target_shape.size(), dtype=g.dtype().torch, device=g.tensor().device)
    call("j4c_broadcast_like", g.dtype().ordinal, g.data_ptr(), _dims(gs), gs.rank(), out.data_ptr(),
         _dims(target_shape), target_shape.rank(), g._stream())
    return ConcreteNDArray._wrap(out, target_shape, g.dtype(), g.device())


def axis_broadcast_like(g: ConcreteNDArray, original: Shape, axis: int) -> ConcreteNDArray:
    """Grad.axisBroadcastLike (Grad.java:608-641): g (with or without the
    reduced dim) viewed as [outer, 1, inner], broadcast to [outer, axis, inner]."""
    outer, n, inner = original.axis_split(axis)
    if _lazy_on() and inner == 1:
        # the last axis: g as [..., 1] broadcasts over it as a column
        col = Shape(original.dimensions()[:-1] + (1,))
        gv = g if g.shape() == col else materialize(g).reshape(col)
        d = lazy.expand(gv, original)
        if d is not None:
            return d
    g = materialize(g)
    src = Shape(outer, 1, inner)
    dst = Shape(outer, n, inner)
    out = torch.empty(dst.size(), dtype=g.dtype().torch, device=g.tensor().device)
    call("j4c_broadcast_like", g.dtype().ordinal, g.data_ptr(), _dims(src), 3, out.data_ptr(),
         _dims(dst), 3, g._stream())
    return ConcreteNDArray._wrap(out, original, g.dtype(), g.device())


def relu_grad(g: ConcreteNDArray, x: ConcreteNDArray) -> ConcreteNDArray:
    """Grad.reluGrad (Grad.java:585-598)."""
    g = materialize(g)
    out = torch.empty_like(x.tensor())
    call("j4c_relu_grad", x.dtype().ordinal, g.data_ptr(), x.data_ptr(), x.shape().size(),
         out.data_ptr(), x._stream())
    return ConcreteNDArray._wrap(out, x.shape(), x.dtype(), x.device())


def maxmin_grad(g: ConcreteNDArray, a: ConcreteNDArray, b: ConcreteNDArray, is_max: bool):
    """Grad.maxMinGrad (Grad.java:500-530): ties go to a."""
    g = materialize(g)
    gs = g.shape()
    ga = torch.empty_like(g.tensor())
    gb = torch.empty_like(g.tensor())
    call("j4c_maxmin_grad", int(is_max), g.dtype().ordinal, g.data_ptr(), _dims(gs), gs.rank(),
         a.data_ptr(), _dims(a.shape()), a.shape().rank(), b.data_ptr(), _dims(b.shape()),
         b.shape().rank(), ga.data_ptr(), gb.data_ptr(), g._stream())
    GA = ConcreteNDArray._wrap(ga, gs, g.dtype(), g.device())
    GB = ConcreteNDArray._wrap(gb, gs, g.dtype(), g.device())
    return [broadcast_like(GA, a.shape()), broadcast_like(GB, b.shape())]


def _neg(x: ConcreteNDArray) -> ConcreteNDArray:
    """x.mul(minusOne(x.shape())) with the -1 broadcast instead of materialised."""
    return _bin(x, _scalar_like(-1.0, x), Primitive.MUL)


def _bin(a: ConcreteNDArray, b: ConcreteNDArray, prim: Primitive) -> ConcreteNDArray:
    """A binary kernel without the public method's device-tag rules (the
    interpreter's helper constants are created next to their operands);
    deferred inside the backward walk when it fits a generated kernel."""
    if _lazy_on():
        d = lazy.binary(a, b, prim)
        if d is not None:
            return d
    a, b = materialize(a), materialize(b)
    out_shape = Shape.broadcast(a.shape(), b.shape())
    out = torch.empty(out_shape.size(), dtype=a.dtype().torch, device=a.tensor().device)
    call("j4c_binary", int(prim), a.dtype().ordinal, a.data_ptr(), _dims(a.shape()), a.shape().rank(),
         b.data_ptr(), _dims(b.shape()), b.shape().rank(), out.data_ptr(), a._stream())
    return ConcreteNDArray._wrap(out, out_shape, a.dtype(), a.device())


# ---------------------------------------------------------------------------
# forward / backward interpretation
# ---------------------------------------------------------------------------
def _needs_grad(jaxpr: Jaxpr) -> set:
    """Var ids that depend on some inVar (only their cotangents are read)."""
    cached = getattr(jaxpr, "_needs_grad", None)
    if cached is not None:
        return cached
    need = {v.id for v in jaxpr.inVars}
    for eq in jaxpr.equations:
        if any(v.id in need for v in eq.inputs):
            for o in eq.outputs:
                need.add(o.id)
    jaxpr._needs_grad = need
    return need


# Elementwise chains of an interpreted Jaxpr run as fused generated kernels
# (jax4j_b200/fusion.py); J4C_FUSION=0 runs every equation on its own.
FUSION = os.environ.get("J4C_FUSION", "1") != "0"


def _dot_split_kinds(jaxpr: Jaxpr, eq) -> tuple:
    """The operand splits a DOT equation's forward and, for the cotangents the
    backward will compute, its VJP read (Grad.java:385-390), as split kinds of
    core._split_of: the forward reads A with row lines and B transposed;
    dA = g . B^T reads B with row lines; dB = A^T . g reads A with column
    lines, or transposed when A is the smaller operand."""
    need = _needs_grad(jaxpr)
    a, b = eq.inputs
    ka, kb = ["r"], ["t"]
    if b.id in need:
        ka.append("t" if a.shape.size() < eq.outputs[0].shape.size() else "c")
    if a.id in need:
        kb.append("r")
    return ka, kb


def _presplit_dot(jaxpr: Jaxpr, eq, values) -> None:
    """Makes every split a DOT's operands will take, each operand's in one
    pass over it, before the forward product (the backward then finds them)."""
    from .core import _make_splits
    a, b = values.get(eq.inputs[0].id), values.get(eq.inputs[1].id)
    if not (isinstance(a, ConcreteNDArray) and isinstance(b, ConcreteNDArray)):
        return
    if a.dtype() != DType.FLOAT32 or b.dtype() != DType.FLOAT32 or a.shape().rank() != 2 or b.shape().rank() != 2:
        return
    if not (a.shape().size() and b.shape().size()):
        return
    ka, kb = _dot_split_kinds(jaxpr, eq)
    _make_splits(a, ka)
    _make_splits(b, kb)


def _evaluate(jaxpr: Jaxpr, args: List[NDArray], keep_for_vjp: bool) -> Dict[int, NDArray]:
    values: Dict[int, NDArray] = dict(jaxpr.consts)
    if len(args) != len(jaxpr.inVars):
        raise IllegalArgumentException(f"expected {len(jaxpr.inVars)} arguments, got {len(args)}")
    for v, a in zip(jaxpr.inVars, args):
        values[v.id] = a
    if len(jaxpr.equations) == 1 and jaxpr.equations[0].primitive is Primitive.FFI_CALL:
        _run_equation(jaxpr.equations[0], values, keep_for_vjp)  # one layer: nothing to plan
        return values
    if FUSION and all(isinstance(a, ConcreteNDArray) for a in values.values()):
        from . import fusion
        for kind, item in fusion.plan_for(jaxpr, keep_for_vjp).steps:
            if kind == "eq":
                if keep_for_vjp and item.primitive == Primitive.DOT:
                    _presplit_dot(jaxpr, item, values)
                _run_equation(item, values, keep_for_vjp)
            elif kind == "dot_ep":
                if keep_for_vjp:
                    _presplit_dot(jaxpr, item.dot, values)
                fusion.run_dot_epilogue(item, values)
            else:
                fusion.run_group(item, values)
        return values
    for eq in jaxpr.equations:
        if keep_for_vjp and eq.primitive == Primitive.DOT:
            _presplit_dot(jaxpr, eq, values)
        _run_equation(eq, values, keep_for_vjp)
    return values


def _run_equation(eq, values: Dict[int, NDArray], keep_for_vjp: bool = False) -> None:
    inputs = [values[v.id] for v in eq.inputs]
    if eq.primitive is Primitive.FFI_CALL:
        out = eq.outputs[0].id
        values[out], saved = eq.metadata.run(inputs, keep_for_vjp)
        if saved is not None:
            values[~out] = saved  # for its VJP, under an id no Var has
        return
    if eq.primitive == Primitive.SCAN:  # the one two-output primitive
        carry, ys = scan_forward(eq, inputs)
        values[eq.outputs[0].id] = carry
        values[eq.outputs[1].id] = ys
    else:
        values[eq.outputs[0].id] = execute_primitive(eq.primitive, eq, inputs)


# ---- Numpy.take (GATHER) ------------------------------------------------------------------
def take_eager(table: ConcreteNDArray, indices: ConcreteNDArray) -> ConcreteNDArray:
    """Numpy.takeEager (Numpy.java:68-76): rows of a [rows, dim] table at
    integer indices -> [*indices.shape, dim]."""
    td = table.shape().dimensions()
    if len(td) != 2:
        raise IllegalArgumentException(f"take: table must be [rows, dim], got {table.shape()}")
    if indices.dtype() not in (DType.INT32, DType.INT64):
        raise IllegalArgumentException(f"take: indices must be INT32 or INT64, got {indices.dtype()}")
    rows, dim = td
    n = indices.shape().size()
    if n:
        host = indices.numpy()
        lo, hi = int(host.min()), int(host.max())
        if lo < 0 or hi >= rows:
            raise IllegalArgumentException(f"take: index {lo if lo < 0 else hi} out of range for {rows} rows")
    import torch
    out = torch.empty(n * dim, dtype=table.dtype().torch, device=table.tensor().device)
    call("j4c_gather_rows", table.dtype().ordinal, table.data_ptr(), rows, dim, indices.dtype().ordinal,
         indices.data_ptr(), n, out.data_ptr(), table._stream())
    return ConcreteNDArray._wrap(out, Shape(indices.shape().dimensions() + (dim,)), table.dtype(), table.device())


def gather_backward(g: ConcreteNDArray, table_shape: Shape, indices: ConcreteNDArray) -> ConcreteNDArray:
    """Grad.gatherBackward (Grad.java:474-493): scatter-add of g's rows."""
    rows, dim = table_shape.dimensions()
    out = zeros(table_shape, g.dtype(), g.device())
    call("j4c_scatter_add_rows", g.dtype().ordinal, g.data_ptr(), rows, dim, indices.dtype().ordinal,
         indices.data_ptr(), indices.shape().size(), out.data_ptr(), g._stream())
    return out


# ---- forward mode (Grad.forwardAd, Grad.java:668-835) -----------------------------------
def forward_ad(jaxpr: Jaxpr, args: List[NDArray], tangents_in: List[NDArray]):
    """Grad.forwardAd: primals and tangents pushed forward together; returns
    (output primals, output tangents)."""
    primals: Dict[int, NDArray] = dict(jaxpr.consts)
    tangents: Dict[int, NDArray] = {k: zeros_like(v) for k, v in jaxpr.consts.items()}
    for v, a, t in zip(jaxpr.inVars, args, tangents_in):
        primals[v.id] = a
        tangents[v.id] = t
    for eq in jaxpr.equations:
        if eq.primitive == Primitive.FFI_CALL:
            raise UnsupportedOperationException(f"{eq.metadata.name} is not forward-mode differentiable")
        ins = [primals[v.id] for v in eq.inputs]
        tins = [tangents[v.id] for v in eq.inputs]
        if eq.primitive == Primitive.SCAN:
            c, ys, ct, yst = _scan_jvp(eq, ins, tins)
            primals[eq.outputs[0].id], primals[eq.outputs[1].id] = c, ys
            tangents[eq.outputs[0].id], tangents[eq.outputs[1].id] = ct, yst
            continue
        out = execute_primitive(eq.primitive, eq, ins)
        primals[eq.outputs[0].id] = out
        tangents[eq.outputs[0].id] = compute_jvp(eq.primitive, eq, out, ins, tins)
    return [primals[v.id] for v in jaxpr.outVars], [tangents[v.id] for v in jaxpr.outVars]


def _scan_jvp(eq, primals: List[NDArray], tangents: List[NDArray]):
    """Grad.scanJVP (Grad.java:707-731)."""
    m: ScanMeta = eq.metadata
    carry, xs = primals
    carry_t, xs_t = tangents
    ys, ys_t = [], []
    for t in range(xs.shape().dimensions()[0]):
        (carry, y), (carry_t, y_t) = forward_ad(m.stepFn, [carry, slice_leading(xs, t)],
                                                [carry_t, slice_leading(xs_t, t)])
        ys.append(y)
        ys_t.append(y_t)
    return carry, stack_leading(ys), carry_t, stack_leading(ys_t)


def compute_jvp(p: Primitive, eq, out: ConcreteNDArray, x: List[NDArray], t: List[NDArray]) -> NDArray:
    """Grad.computeJVP (Grad.java:733-835), op for op."""
    from . import pmap as _pm
    dtype, shape, dev = out.dtype(), out.shape(), out.device()

    def full(v):
        return ConcreteNDArray.full(shape, v, dtype, dev)

    if p == Primitive.ADD: return t[0].add(t[1])
    if p == Primitive.SUB: return t[0].sub(t[1])
    if p == Primitive.MUL: return t[0].mul(x[1]).add(x[0].mul(t[1]))
    if p == Primitive.DIV:
        b = x[1]
        return t[0].mul(b).sub(x[0].mul(t[1])).div(b.mul(b))
    if p == Primitive.MEAN: return t[0].mean()
    if p == Primitive.SUM: return t[0].sum()
    if p in (Primitive.SUM_AXIS, Primitive.MEAN_AXIS):
        m: AxisMeta = eq.metadata
        return t[0].sum(m.axis, m.keepDims) if p == Primitive.SUM_AXIS else t[0].mean(m.axis, m.keepDims)
    if p == Primitive.EXP: return t[0].mul(out)
    if p == Primitive.LOG: return t[0].div(x[0])
    if p == Primitive.SIN: return t[0].mul(x[0].cos())
    if p == Primitive.COS: return t[0].mul(x[0].sin()).mul(full(-1.0))
    if p == Primitive.TANH: return t[0].mul(full(1.0).sub(out.mul(out)))
    if p == Primitive.RELU:
        zero = ConcreteNDArray.full(x[0].shape(), 0.0, x[0].dtype(), x[0].device())
        return t[0].mul(x[0].gt(zero).astype(x[0].dtype()))
    if p == Primitive.SIGMOID: return t[0].mul(out.mul(full(1.0).sub(out)))
    if p == Primitive.DOT: return t[0].dot(x[1]).add(x[0].dot(t[1]))
    if p == Primitive.COND:
        m: CondMeta = eq.metadata
        branch = m.trueBranch if is_true(x[0]) else m.falseBranch
        return forward_ad(branch, [x[1]], [t[1]])[1][0]
    if p == Primitive.WHILE:
        raise UnsupportedOperationException("Lax.whileLoop is not forward-mode differentiable")
    if p == Primitive.CAST: return t[0].astype(eq.metadata)
    if p == Primitive.GATHER: return take_eager(t[0], x[1])
    if p in (Primitive.GT, Primitive.GE, Primitive.LT, Primitive.LE, Primitive.EQ, Primitive.NE,
             Primitive.ARGMAX, Primitive.ARGMIN):
        return zeros(shape, dtype, dev)
    if p == Primitive.CHECKPOINT:
        m: CheckpointMeta = eq.metadata
        return forward_ad(m.subJaxpr, [x[0]], [t[0]])[1][0]
    if p == Primitive.PMAP:
        # each shard's body pushed forward in turn, as the reference does (its
        # collectives see no pmap context there, so they act as identities)
        m: PmapMeta = eq.metadata
        ps, ts = _pm.split(x[0], m.numDevices()), _pm.split(t[0], m.numDevices())
        return _pm.stack([forward_ad(m.bodyJaxpr, [ps[i]], [ts[i]])[1][0] for i in range(m.numDevices())])
    if p == Primitive.PSUM: return _pm.psum_value(t[0])
    if p == Primitive.ALL_GATHER: return _pm.all_gather_value(t[0])
    raise UnsupportedOperationException(f"No JVP rule defined for primitive: {p.name}")


# ---- control flow (api/Lax.java:69-217, Grad.java:213-265) ----------------------------
def is_true(pred: NDArray) -> bool:
    """Lax.isTrue (Lax.java:60-62): the first element, nonzero."""
    return float(pred.numpy().reshape(-1)[0]) != 0.0


def slice_leading(a: ConcreteNDArray, t: int) -> ConcreteNDArray:
    """ScanUtil.sliceLeading: step t of a [T, *step] array (a view)."""
    step = Shape(a.shape().dimensions()[1:])
    n = step.size()
    return ConcreteNDArray._wrap(a.tensor()[t * n:(t + 1) * n], step, a.dtype(), a.device())


def stack_leading(items: List[ConcreteNDArray]) -> ConcreteNDArray:
    """ScanUtil.stackLeading: [T, *step]."""
    from . import pmap as _pm
    return _pm.stack(items)


def scan_forward(eq, inputs: List[NDArray]):
    """Grad.scanForward (Grad.java:213-230): the step once per leading slice."""
    m: ScanMeta = eq.metadata
    carry, xs = inputs
    ys = []
    for t in range(xs.shape().dimensions()[0]):
        carry, y = forward_interpret(m.stepFn, [carry, slice_leading(xs, t)])
        ys.append(y)
    return carry, stack_leading(ys)


def scan_backward(eq, inputs: List[NDArray], g_carry_final, g_ys):
    """Grad.scanBackward (Grad.java:232-265): re-runs the forward to record
    every step's (carry, x), then backward-interprets the step in reverse."""
    m: ScanMeta = eq.metadata
    init, xs = inputs
    steps = xs.shape().dimensions()[0]
    y_shape = m.stepFn.outVars[1].shape
    carry_in, x_in = [], []
    carry = init
    for t in range(steps):
        carry_in.append(carry)
        x_in.append(slice_leading(xs, t))
        carry = forward_interpret(m.stepFn, [carry, x_in[t]])[0]
    dev = init.device()
    g_carry = g_carry_final if g_carry_final is not None else zeros(init.shape(), init.dtype(), dev)
    g_xs = [None] * steps
    for t in range(steps - 1, -1, -1):
        g_y = slice_leading(g_ys, t) if g_ys is not None else zeros(y_shape, m.stepFn.outVars[1].dtype, dev)
        g_carry, g_xs[t] = backward_interpret(m.stepFn, [carry_in[t], x_in[t]], [g_carry, g_y])
    return g_carry, stack_leading(g_xs)


def fill_forward_values(jaxpr: Jaxpr, args: List[NDArray]) -> Dict[int, NDArray]:
    """Grad.fillForwardValues (Grad.java:192-211): every value a VJP rule
    reads is kept; values only used inside a fused chain are not written."""
    return _evaluate(jaxpr, args, True)


def forward_interpret(jaxpr: Jaxpr, args: List[NDArray]) -> List[NDArray]:
    """Grad.forwardInterpret (Grad.java:135-138)."""
    values = _evaluate(jaxpr, args, False)
    return [values[v.id] for v in jaxpr.outVars]


def backward_interpret(jaxpr: Jaxpr, args: List[NDArray], seeds: List[NDArray]) -> List[NDArray]:
    """Grad.backwardInterpret (Grad.java:150-152)."""
    return do_backward(jaxpr, fill_forward_values(jaxpr, args), seeds)


def _merge(grads: Dict[int, NDArray], vid: int, g: NDArray) -> None:
    prev = grads.get(vid)
    if prev is None:
        grads[vid] = g
    elif isinstance(prev, Deferred) or isinstance(g, Deferred):
        grads[vid] = _bin(prev, g, Primitive.ADD)
    else:
        grads[vid] = prev.add(g)


def _split_g_both(g, a, want_a: bool, want_b: bool) -> None:
    """A DOT VJP reads its output gradient g with row lines (g . B^T) and,
    for A^T . g, transposed when A is at least as large as g (the smaller
    operand goes in transposed) or else with column lines: both splits of g
    are made in one pass."""
    from .core import _make_splits
    if (want_a and want_b and isinstance(g, ConcreteNDArray) and isinstance(a, ConcreteNDArray)
            and g.dtype() == DType.FLOAT32 and g.shape().rank() == 2 and g.shape().size()):
        _make_splits(g, ["r", "t" if a.shape().size() >= g.shape().size() else "c"])


def _relu_fed_dots(jaxpr: Jaxpr, need) -> Dict[int, object]:
    """DOT equations whose first input h = relu(z) feeds nothing else: the
    input gradient g . W^T is masked by h > 0 (the same elements as z > 0:
    relu keeps a positive z and maps every other z, NaN included, to 0 or
    NaN) in the GEMM's store and credited to z, so relu's own VJP
    (relu_grad, Grad.java:585-598) has nothing left to do.  Keyed by
    id(dot equation) -> (z, h)."""
    uses: Dict[int, int] = {}
    producer = {}
    for eq in jaxpr.equations:
        for v in eq.inputs:
            uses[v.id] = uses.get(v.id, 0) + 1
        for o in eq.outputs:
            producer[o.id] = eq
    outs = {v.id for v in jaxpr.outVars}
    found = {}
    for eq in jaxpr.equations:
        if eq.primitive != Primitive.DOT:
            continue
        h = eq.inputs[0]
        r = producer.get(h.id)
        if (r is None or r.primitive != Primitive.RELU or uses.get(h.id) != 1 or h.id in outs
                or h.dtype != DType.FLOAT32 or r.inputs[0].id not in need):
            continue
        found[id(eq)] = (r.inputs[0], h)
    return found


_current_pmap = None  # PmapContext.current, imported at its first use (pmap imports this module)


def _pmap_context():
    global _current_pmap
    if _current_pmap is None:
        from .pmap import PmapContext
        _current_pmap = PmapContext.current
    return _current_pmap()


def do_backward(jaxpr: Jaxpr, values: Dict[int, NDArray], seeds: List[NDArray]) -> List[NDArray]:
    """Grad.doBackward (Grad.java:154-189)."""
    eqs = jaxpr.equations
    if (len(eqs) == 1 and eqs[0].primitive is Primitive.FFI_CALL and len(seeds) == 1
            and jaxpr.outVars[0].id == eqs[0].outputs[0].id and _pmap_context() is None):
        return _layer_backward(jaxpr, values, seeds[0])  # one layer: nothing to walk
    _lazy_scope.depth = getattr(_lazy_scope, "depth", 0) + 1
    try:
        return _do_backward(jaxpr, values, seeds)
    finally:
        _lazy_scope.depth -= 1


def _layer_backward(jaxpr: Jaxpr, values: Dict[int, NDArray], seed: NDArray) -> List[NDArray]:
    """do_backward of a Jaxpr that is one FFI_CALL and its output."""
    eq = jaxpr.equations[0]
    ids, eq_ids, out = [v.id for v in jaxpr.inVars], [v.id for v in eq.inputs], eq.outputs[0].id
    g_ins = eq.metadata.pull([values[i] for i in eq_ids], values[out], values.get(~out), materialize(seed),
                             [i in ids for i in eq_ids])
    grads: Dict[int, NDArray] = {}
    for v, g in zip(eq.inputs, g_ins):
        if g is not None:
            _merge(grads, v.id, g)
    return [materialize(grads[v.id]) if v.id in grads else zeros(v.shape, v.dtype, _device_of(values.get(v.id)))
            for v in jaxpr.inVars]


def _do_backward(jaxpr: Jaxpr, values: Dict[int, NDArray], seeds: List[NDArray]) -> List[NDArray]:
    need = _needs_grad(jaxpr)
    fused_relu = _relu_fed_dots(jaxpr, need) if FUSION else {}
    grads: Dict[int, NDArray] = {}
    for v, s in zip(jaxpr.outVars, seeds):
        _merge(grads, v.id, s)
    # The equation after which each input's cotangent is complete (its first
    # consumer): inside a pmap there a CUDA event is recorded on the gradient,
    # so a collective over it (Lax.psumTree) can start while the rest of the
    # backward pass still runs.
    overlap = _pmap_context() is not None
    in_ids = {v.id for v in jaxpr.inVars}
    last_use = {}
    for i, e in enumerate(jaxpr.equations):
        for v in e.inputs:
            if v.id in in_ids and v.id not in last_use:
                last_use[v.id] = i
    done_at: Dict[int, list] = {}
    for vid, i in last_use.items():
        done_at.setdefault(i, []).append(vid)
    for i_eq, eq in reversed(list(enumerate(jaxpr.equations))):
        _process_backward_eq(eq, values, grads, need, fused_relu)
        for vid in done_at.get(i_eq, ()):
            g = grads.get(vid)
            if isinstance(g, Deferred):
                g = grads[vid] = materialize(g)
            if overlap and isinstance(g, ConcreteNDArray) and g.tensor().is_cuda:
                ev = torch.cuda.Event()
                ev.record(torch.cuda.current_stream(g.tensor().device))
                g._ready = ev
    result = []
    for v in jaxpr.inVars:
        g = materialize(grads.get(v.id))
        result.append(g if g is not None else zeros(v.shape, v.dtype, _device_of(values.get(v.id))))
    return result


def _process_backward_eq(eq, values, grads, need, fused_relu) -> None:
    """One equation of Grad.doBackward's reverse walk (Grad.java:162-185)."""
    if eq.primitive == Primitive.SCAN:
        g_c, g_y = materialize(grads.get(eq.outputs[0].id)), materialize(grads.get(eq.outputs[1].id))
        if (g_c is None and g_y is None) or not any(v.id in need for v in eq.inputs):
            return
        gi = scan_backward(eq, [values.get(v.id) for v in eq.inputs], g_c, g_y)
        for v, g in zip(eq.inputs, gi):
            if v.id in need:
                _merge(grads, v.id, g)
        return
    g_out = grads.get(eq.outputs[0].id)
    if g_out is None:
        return
    wanted = [v.id in need for v in eq.inputs]
    if not any(wanted):
        return
    zh = fused_relu.get(id(eq))
    if zh is not None and wanted[0]:
        z, h = zh
        g_out = materialize(g_out)
        a, b = values.get(eq.inputs[0].id), values.get(eq.inputs[1].id)
        zv = values.get(h.id)  # the mask: h > 0 where z > 0
        if (isinstance(g_out, ConcreteNDArray) and isinstance(b, ConcreteNDArray) and
                isinstance(zv, ConcreteNDArray) and g_out.dtype() == b.dtype() == zv.dtype() == DType.FLOAT32):
            # dz = (g . W^T) masked by z > 0 in one GEMM; dW as usual
            _split_g_both(g_out, a, True, wanted[1])
            _merge(grads, z.id, _dot_raw(g_out, b, False, True, g_out.device(), mask=zv))
            if wanted[1]:
                _merge(grads, eq.inputs[1].id, _dot_raw(a, g_out, True, False, g_out.device()))
            return
    inputs = [values.get(v.id) for v in eq.inputs]
    out_value = values.get(eq.outputs[0].id)
    if eq.primitive == Primitive.FFI_CALL:
        g_ins = eq.metadata.pull(inputs, out_value, values.get(~eq.outputs[0].id), materialize(g_out), wanted)
    else:
        g_ins = compute_vjps(eq.primitive, eq, g_out, inputs, out_value, wanted)
    for v, w, g in zip(eq.inputs, wanted, g_ins):
        if w and g is not None:
            _merge(grads, v.id, g)


def _device_of(x):
    return x.device() if isinstance(x, ConcreteNDArray) else None


def execute_primitive(p: Primitive, eq, inputs: List[NDArray]) -> NDArray:
    """Grad.executePrimitive (Grad.java:268-339)."""
    from . import pmap as _pm
    if p == Primitive.ADD: return inputs[0].add(inputs[1])
    if p == Primitive.SUB: return inputs[0].sub(inputs[1])
    if p == Primitive.MUL: return inputs[0].mul(inputs[1])
    if p == Primitive.DIV: return inputs[0].div(inputs[1])
    if p == Primitive.DOT: return inputs[0].dot(inputs[1])
    if p == Primitive.MEAN: return inputs[0].mean()
    if p == Primitive.SUM: return inputs[0].sum()
    if p in (Primitive.SUM_AXIS, Primitive.MEAN_AXIS):
        m: AxisMeta = eq.metadata
        return (inputs[0].sum(m.axis, m.keepDims) if p == Primitive.SUM_AXIS
                else inputs[0].mean(m.axis, m.keepDims))
    if p == Primitive.EXP: return inputs[0].exp()
    if p == Primitive.LOG: return inputs[0].log()
    if p == Primitive.SIN: return inputs[0].sin()
    if p == Primitive.COS: return inputs[0].cos()
    if p == Primitive.TANH: return inputs[0].tanh()
    if p == Primitive.RELU: return inputs[0].relu()
    if p == Primitive.SIGMOID: return inputs[0].sigmoid()
    if p == Primitive.GT: return inputs[0].gt(inputs[1])
    if p == Primitive.GE: return inputs[0].ge(inputs[1])
    if p == Primitive.LT: return inputs[0].lt(inputs[1])
    if p == Primitive.LE: return inputs[0].le(inputs[1])
    if p == Primitive.EQ: return inputs[0].eq(inputs[1])
    if p == Primitive.NE: return inputs[0].ne(inputs[1])
    if p == Primitive.MAX: return inputs[0].max(inputs[1])
    if p == Primitive.MIN: return inputs[0].min(inputs[1])
    if p in (Primitive.ARGMAX, Primitive.ARGMIN):
        m = eq.metadata
        return inputs[0].argmax(m.axis) if p == Primitive.ARGMAX else inputs[0].argmin(m.axis)
    if p == Primitive.CAST: return inputs[0].astype(eq.metadata)
    if p == Primitive.GATHER:
        return take_eager(inputs[0], inputs[1])
    if p == Primitive.COND:
        m: CondMeta = eq.metadata
        return forward_interpret(m.trueBranch if is_true(inputs[0]) else m.falseBranch, [inputs[1]])[0]
    if p == Primitive.WHILE:
        m: WhileMeta = eq.metadata
        state = inputs[0]
        while is_true(forward_interpret(m.condFn, [state])[0]):
            state = forward_interpret(m.bodyFn, [state])[0]
        return state
    if p == Primitive.PMAP:
        m: PmapMeta = eq.metadata
        shards = [_pm.shards_of(x, m.numDevices()) for x in inputs]
        return _pm.run_forward_jaxpr(m.bodyJaxpr, m.devices, shards)
    if p == Primitive.PSUM:
        return _pm.psum_value(inputs[0])
    if p == Primitive.ALL_GATHER:
        return _pm.all_gather_value(inputs[0])
    if p == Primitive.CHECKPOINT:
        m: CheckpointMeta = eq.metadata
        return forward_interpret(m.subJaxpr, [inputs[0]])[0]
    if p == Primitive.FFI_CALL:
        return eq.metadata.run(inputs, False)[0]
    raise UnsupportedOperationException(str(p))


# rules built only from _bin / broadcasts, whose cotangent may stay deferred
_DEFERRABLE_RULES = {Primitive.ADD, Primitive.SUB, Primitive.MUL, Primitive.DIV, Primitive.MEAN, Primitive.SUM,
                     Primitive.SUM_AXIS, Primitive.MEAN_AXIS, Primitive.EXP, Primitive.LOG, Primitive.SIN,
                     Primitive.COS, Primitive.TANH, Primitive.SIGMOID, Primitive.CAST,
                     # zero cotangents: g is not read
                     Primitive.GT, Primitive.GE, Primitive.LT, Primitive.LE, Primitive.EQ, Primitive.NE,
                     Primitive.ARGMAX, Primitive.ARGMIN}


def compute_vjps(p: Primitive, eq, g: ConcreteNDArray, inputs: List[NDArray], out_value,
                 wanted: List[bool]) -> List:
    """Grad.computeVJPs (Grad.java:341-472).  Entries of inputs whose cotangent is
    not wanted may come back as None."""
    from . import pmap as _pm
    if p not in _DEFERRABLE_RULES:
        g = materialize(g)
    want_a = wanted[0]
    want_b = len(wanted) > 1 and wanted[1]
    shapes = [v.shape for v in eq.inputs]  # rules that need only shapes read them from the Vars
    if p == Primitive.ADD:
        return [broadcast_like(g, shapes[0]) if want_a else None,
                broadcast_like(g, shapes[1]) if want_b else None]
    if p == Primitive.SUB:
        return [broadcast_like(g, shapes[0]) if want_a else None,
                broadcast_like(_neg(g), shapes[1]) if want_b else None]
    if p == Primitive.MUL:
        return [broadcast_like(_bin(g, inputs[1], Primitive.MUL), shapes[0]) if want_a else None,
                broadcast_like(_bin(g, inputs[0], Primitive.MUL), shapes[1]) if want_b else None]
    if p == Primitive.DIV:
        a, b = inputs
        ga = broadcast_like(_bin(g, b, Primitive.DIV), shapes[0]) if want_a else None
        gb = None
        if want_b:
            t = _bin(_bin(_bin(g, a, Primitive.MUL), b, Primitive.DIV), b, Primitive.DIV)
            gb = broadcast_like(_neg(t), shapes[1])
        return [ga, gb]
    if p == Primitive.MEAN:
        n = float(shapes[0].size())
        return [broadcast_like(_bin(g, _scalar_like(n, g), Primitive.DIV), shapes[0])]
    if p == Primitive.SUM:
        return [broadcast_like(g, shapes[0])]
    if p == Primitive.SUM_AXIS:
        return [axis_broadcast_like(g, shapes[0], eq.metadata.axis)]
    if p == Primitive.MEAN_AXIS:
        m = eq.metadata
        n = float(shapes[0][m.axis])
        return [axis_broadcast_like(_bin(g, _scalar_like(n, g), Primitive.DIV), shapes[0], m.axis)]
    if p == Primitive.EXP:
        e = out_value if out_value is not None else inputs[0].exp()
        return [_bin(g, e, Primitive.MUL)]
    if p == Primitive.LOG:
        return [_bin(g, inputs[0], Primitive.DIV)]
    if p == Primitive.SIN:
        return [_bin(g, inputs[0].cos(), Primitive.MUL)]
    if p == Primitive.COS:
        return [_neg(_bin(g, inputs[0].sin(), Primitive.MUL))]
    if p == Primitive.TANH:
        t = out_value if out_value is not None else inputs[0].tanh()
        one_m = _bin(_scalar_like(1.0, t), _bin(t, t, Primitive.MUL), Primitive.SUB)
        return [_bin(g, one_m, Primitive.MUL)]
    if p == Primitive.RELU:
        # h = relu(z) > 0 exactly where z > 0, so the output serves as the mask
        return [relu_grad(g, out_value if out_value is not None else inputs[0])]
    if p == Primitive.SIGMOID:
        s = out_value if out_value is not None else inputs[0].sigmoid()
        one_m = _bin(_scalar_like(1.0, s), s, Primitive.SUB)
        return [_bin(g, _bin(s, one_m, Primitive.MUL), Primitive.MUL)]
    if p == Primitive.DOT:
        a, b = inputs
        _split_g_both(g, a, want_a, want_b)
        # dA = gOut . B^T, dB = A^T . gOut (Grad.java:385-390), transposes as layout flags
        ga = _dot_raw(g, b, False, True, g.device()) if want_a else None
        gb = _dot_raw(a, g, True, False, g.device()) if want_b else None
        return [ga, gb]
    if p in (Primitive.GT, Primitive.GE, Primitive.LT, Primitive.LE, Primitive.EQ, Primitive.NE):
        return [_zeros_for(eq.inputs[0], g) if want_a else None,
                _zeros_for(eq.inputs[1], g) if want_b else None]
    if p == Primitive.MAX:
        return maxmin_grad(g, inputs[0], inputs[1], True)
    if p == Primitive.MIN:
        return maxmin_grad(g, inputs[0], inputs[1], False)
    if p in (Primitive.ARGMAX, Primitive.ARGMIN):
        return [_zeros_for(eq.inputs[0], g)]
    if p == Primitive.GATHER:
        # embedding backward: scatter-add into a table-shaped zero gradient
        return [gather_backward(g, shapes[0], inputs[1]) if want_a else None,
                _zeros_for(eq.inputs[1], g) if want_b else None]
    if p == Primitive.COND:
        # pred is not differentiable (Grad.java:391-397)
        m: CondMeta = eq.metadata
        branch = m.trueBranch if is_true(inputs[0]) else m.falseBranch
        g_operand = backward_interpret(branch, [inputs[1]], [g])[0] if want_b else None
        return [_zeros_for(eq.inputs[0], g) if want_a else None, g_operand]
    if p == Primitive.WHILE:
        raise UnsupportedOperationException(
            "Lax.whileLoop is not reverse-mode differentiable (mirrors jax.lax.while_loop, whose iteration "
            "count is itself data-dependent); use Lax.scan or Lax.foriLoop for a differentiable loop.")
    if p == Primitive.PMAP:
        m: PmapMeta = eq.metadata
        D = m.numDevices()
        in_shards = [_pm.shards_of(x, D) for x in inputs]
        g_shards = _pm.shards_of(g, D)
        g_in = _pm.run_backward_jaxpr(m.bodyJaxpr, m.devices, in_shards, g_shards)
        return [_pm.stack([gi[k] for gi in g_in]) for k in range(len(inputs))]
    if p == Primitive.PSUM:
        # psum is linear and its transpose is another psum (Grad.java:425-434)
        return [_pm.psum_value(g)]
    if p == Primitive.ALL_GATHER:
        return [_pm.all_gather_vjp(g)]
    if p == Primitive.CAST:
        target = eq.metadata
        identity = eq.inputs[0].dtype == target and target.is_floating()
        return [broadcast_like(g, shapes[0]) if identity else _zeros_for(eq.inputs[0], g)]
    if p == Primitive.CHECKPOINT:
        return [backward_interpret(eq.metadata.subJaxpr, [inputs[0]], [g])[0]]
    if p == Primitive.WHILE:
        raise UnsupportedOperationException(
            "Lax.whileLoop is not reverse-mode differentiable (mirrors jax.lax.while_loop)")
    raise UnsupportedOperationException(str(p))


# ---------------------------------------------------------------------------
# public transforms (Grad.java:37-119)
# ---------------------------------------------------------------------------
def make_jaxpr(fn: Callable, *args: NDArray) -> Jaxpr:
    """JAX.make_jaxpr (JAX.java:30-55), any number of arguments; a function
    returning a tuple or list of arrays gives a Jaxpr with that many outputs."""
    Tracer.start()
    try:
        t = Tracer.current()
        in_vars = [t.nextVar(a.shape(), a.dtype()) for a in args]
        result = fn(*[TracedNDArray(v) for v in in_vars])
        results = list(result) if isinstance(result, (tuple, list)) else [result]
        out_vars = []
        for r in results:
            if not isinstance(r, TracedNDArray):
                r = TracedNDArray(t.nextConstant(r))
            out_vars.append(r.getVar())
        jaxpr = Tracer.stop(in_vars, out_vars)
        jaxpr.__dict__["_tuple_out"] = isinstance(result, (tuple, list))
        return jaxpr
    except BaseException:
        Tracer.abort()
        raise


def _seed_for(var: Var, like=None) -> ConcreteNDArray:
    return ones(var.shape, _float_or_default(var.dtype), _device_of(like))


def _backward(jaxpr: Jaxpr, args: List[NDArray]) -> List[NDArray]:
    """Grad.backward (Grad.java:121-125): seed = ones of the output."""
    values = fill_forward_values(jaxpr, args)
    out = values[jaxpr.outVars[0].id]
    return do_backward(jaxpr, values, [_seed_for(jaxpr.outVars[0], out)])


def grad(fn: Callable, argnum: int = None) -> Callable:
    """Grad.grad (Grad.java:37-57); with argnum, the two-argument form."""
    if argnum is None:
        def g1(arg):
            return _backward(make_jaxpr(fn, arg), [arg])[0]
        return g1
    if argnum not in (0, 1):
        raise IllegalArgumentException(f"argnum must be 0 or 1, got {argnum}")

    def g2(a0, a1):
        return _backward(make_jaxpr(fn, a0, a1), [a0, a1])[argnum]
    return g2


def grad_both(fn: Callable) -> Callable:
    """Grad.gradBoth (Grad.java:63-69)."""
    def g(a0, a1):
        return _backward(make_jaxpr(fn, a0, a1), [a0, a1])
    return g


def vjp(fn: Callable, *args: NDArray):
    """JAX.vjp: (fn(*args), pullback)."""
    if Tracer.current() is not None:
        raise UnsupportedOperationException("JAX.vjp inside a trace")
    jaxpr = make_jaxpr(fn, *args)
    eqs, tuple_out = jaxpr.equations, jaxpr.__dict__.get("_tuple_out")
    if (len(eqs) == 1 and eqs[0].primitive is Primitive.FFI_CALL and not tuple_out and not jaxpr.consts
            and [v.id for v in eqs[0].inputs] == [v.id for v in jaxpr.inVars] and jaxpr.outVars[0] is eqs[0].outputs[0]):
        return _layer_vjp(jaxpr, list(args))
    values = fill_forward_values(jaxpr, list(args))
    outs = [values[v.id] for v in jaxpr.outVars]

    def pullback(*seeds: NDArray) -> List[NDArray]:
        _check_seeds(jaxpr, seeds)
        return do_backward(jaxpr, values, list(seeds))

    return (tuple(outs) if tuple_out else outs[0]), pullback


def _check_seeds(jaxpr: Jaxpr, seeds) -> None:
    if len(seeds) != len(jaxpr.outVars):
        raise IllegalArgumentException(f"pullback: {len(jaxpr.outVars)} outputs take as many cotangents, got {len(seeds)}")
    for s, v in zip(seeds, jaxpr.outVars):
        if s.shape()._d != v.shape._d or s.dtype() is not _float_or_default(v.dtype):
            raise IllegalArgumentException(f"pullback: cotangent {s.shape()} {s.dtype()} of an output {v.shape} {v.dtype}")


def _layer_vjp(jaxpr: Jaxpr, args: List[NDArray]):
    """vjp of a Jaxpr that is one FFI_CALL of its arguments, each once and in
    order: the layer's own forward and VJP, with no maps of values."""
    eq = jaxpr.equations[0]
    out, saved = eq.metadata.forward(args, True)
    wanted = [True] * len(args)

    def pullback(*seeds: NDArray) -> List[NDArray]:
        _check_seeds(jaxpr, seeds)
        if _pmap_context() is not None:  # there the walk notes when each gradient is complete
            values = dict(zip([v.id for v in eq.inputs], args))
            values[eq.outputs[0].id], values[~eq.outputs[0].id] = out, saved
            return do_backward(jaxpr, values, list(seeds))
        return eq.metadata.pull(args, out, saved, materialize(seeds[0]), wanted)

    return out, pullback


def _trace_tree(fn: Callable, tree, leaves: List[NDArray]) -> Jaxpr:
    from .pytree import PyTrees
    Tracer.start()
    try:
        t = Tracer.current()
        in_vars = [t.nextVar(l.shape(), l.dtype()) for l in leaves]
        traced_tree = PyTrees.unflatten(tree, [TracedNDArray(v) for v in in_vars])
        result = fn(traced_tree)
        if not isinstance(result, TracedNDArray):
            result = TracedNDArray(t.nextConstant(result))
        return Tracer.stop(in_vars, [result.getVar()])
    except BaseException:
        Tracer.abort()
        raise


def grad_tree(fn: Callable) -> Callable:
    """Grad.gradTree (Grad.java:77-103)."""
    from .pytree import PyTrees

    def g(tree):
        leaves = PyTrees.flatten(tree)
        jaxpr = _trace_tree(fn, tree, leaves)
        return PyTrees.unflatten(tree, _backward(jaxpr, leaves))
    return g


def value_and_grad(fn: Callable) -> Callable:
    """Grad.value_and_grad (Grad.java:110-119): one forward + backward pass."""
    def vg(arg):
        jaxpr = make_jaxpr(fn, arg)
        values = fill_forward_values(jaxpr, [arg])
        value = values[jaxpr.outVars[0].id]
        grads = do_backward(jaxpr, values, [_seed_for(jaxpr.outVars[0], value)])
        return [value, grads[0]]
    return vg


def value_and_grad_tree(fn: Callable) -> Callable:
    """value_and_grad over a PyTree of parameters: returns [value, grads tree]
    from one forward and one backward pass (the pytree analogue of
    Grad.value_and_grad, Grad.java:110-119)."""
    from .pytree import PyTrees

    def vg(tree):
        leaves = PyTrees.flatten(tree)
        jaxpr = _trace_tree(fn, tree, leaves)
        values = fill_forward_values(jaxpr, leaves)
        value = values[jaxpr.outVars[0].id]
        grads = do_backward(jaxpr, values, [_seed_for(jaxpr.outVars[0], value)])
        return [value, PyTrees.unflatten(tree, grads)]
    return vg
