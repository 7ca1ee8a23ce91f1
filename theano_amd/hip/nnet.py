"""Device versions of the row operators of ``theano_amd.tensor.nnet_lm``.

Each subclasses its host counterpart, as the other device ops do (``ops.py``), and runs one call of the library:
the kernels are compiled into it, so nothing is built at run time.  An operand whose rows do not lie at one stride (a
transposed view, say) is copied to a C-contiguous array first; every other layout is read where it lies.
"""
import ctypes

import numpy as np

from .. import scalar as scal
from ..gof import Apply, Op
from ..tensor import basic as T
from ..tensor import nnet_lm as L
from ..tensor.elemwise import DimShuffle, Elemwise
from ..tensor.type import TensorType
from .ops import HipArrayType, as_hip_variable
from .runtime import HipArray, _Buffer, call_flags, check, lib, mark_reused, thx_array

_UNSUPPORTED = 6


class _RowOp(object):
    """``make_node`` and the calling sequence shared by the operators."""

    def make_node(self, *inputs):
        ins = [as_hip_variable(i) for i in inputs]
        host = self.host_op.make_node(self, *[TensorType(i.type.dtype, i.type.broadcastable)() for i in ins])
        if [i.type.dtype for i in host.inputs] != [i.type.dtype for i in ins]:
            raise TypeError("%s: operands of types %s" % (self, [str(i.type) for i in ins]))
        return Apply(self, ins, [HipArrayType(o.type.dtype, o.type.broadcastable)() for o in host.outputs])

    def perform(self, node, inputs, output_storage):
        slots = node.tag.get("thx")
        if slots is None:
            slots = node.tag["thx"] = ((thx_array * len(inputs))(), (thx_array * len(node.outputs))(),
                                       [np.dtype(o.type.dtype) for o in node.outputs])
        ins, outs, dtypes = slots
        shapes = self.infer_shape(node, [i.shape for i in inputs])
        results = []
        for k, v in enumerate(inputs):
            v.as_thx(ins[k])
        for k, dt in enumerate(dtypes):
            arr = HipArray._new_contiguous(tuple(shapes[k]), dt)
            arr.as_thx(outs[k])
            results.append(arr)
        mark_reused(node, ins, outs)
        flags = call_flags(node)
        rc = self.call(node, ins, outs, flags)
        if rc == _UNSUPPORTED:          # rows at more than one stride, or columns apart
            copies = [v if v.c_contiguous else v.copy() for v in inputs]
            if all(c is v for c, v in zip(copies, inputs)):
                check(rc)
            for k, v in enumerate(copies):
                v.as_thx(ins[k])
            rc = self.call(node, ins, outs, flags)
        if rc:
            check(rc)
        for k, arr in enumerate(results):
            output_storage[k][0] = arr

    def workspace(self, node, ins, query, *args):
        """A buffer for the partial results of a call on ``ins``, kept for the length of the call alone (or by the
        recording the call is made in): (address, size)."""
        key = (tuple(ins[0].shape[:ins[0].nd]),) + tuple(ins[0].strides_bytes[:ins[0].nd])
        known = node.tag.get("workspace")
        if known is None or known[0] != key:
            n = ctypes.c_size_t()
            rc = query(ctypes.byref(ins[0]), *(args + (ctypes.byref(n),)))
            if rc:
                return rc, None, 0
            known = node.tag["workspace"] = (key, n.value)
        return 0, (_Buffer(known[1]) if known[1] else None), known[1]


def _at(arrays, k):
    return ctypes.byref(arrays[k]) if k is not None else None


class HipLayerNormalization(_RowOp, L.LayerNormalization):
    host_op = L.LayerNormalization

    def call(self, node, ins, outs, flags):
        n = len(node.inputs)
        return lib.thx_layernorm_call(_at(ins, 0), _at(ins, 1 if n > 1 else None), _at(ins, 2 if n > 2 else None),
                                      self.epsilon, _at(outs, 0), _at(outs, 1), _at(outs, 2), flags)


class HipLayerNormalizationGrad(_RowOp, L.LayerNormalizationGrad):
    host_op = L.LayerNormalizationGrad

    def call(self, node, ins, outs, flags):
        n = self.n_params
        rc, ws, size = self.workspace(node, ins, lib.thx_layernorm_grad_workspace, _at(outs, 1 if n else None))
        return rc or lib.thx_layernorm_grad_call(
            _at(ins, 0), _at(ins, 1), _at(ins, 4 if n else None), _at(ins, 2), _at(ins, 3), _at(outs, 0),
            _at(outs, 1 if n else None), _at(outs, 2 if n > 1 else None), ws.ptr if ws else None, size, flags)


class HipTokenLogProbs(_RowOp, L.TokenLogProbs):
    host_op = L.TokenLogProbs

    def call(self, node, ins, outs, flags):
        rc, ws, size = self.workspace(node, ins, lib.thx_token_logprob_workspace, self.n_top)
        k = self.n_top
        return rc or lib.thx_token_logprob_call(
            _at(ins, 0), _at(ins, 1), self.temperature, k, _at(outs, 0), _at(outs, 1), _at(outs, 2 if k else None),
            _at(outs, 3 if k else None), _at(outs, 4 if k else 2), ws.ptr if ws else None, size, flags)


class HipTokenLogProbsGrad(_RowOp, L.TokenLogProbsGrad):
    host_op = L.TokenLogProbsGrad

    def call(self, node, ins, outs, flags):
        at = iter(range(4, len(node.inputs)))
        top = next(at) if self.given[2] else None
        g, u, gt = [next(at) if there else None for there in self.given]
        return lib.thx_token_logprob_grad_call(_at(ins, 0), _at(ins, 1), _at(ins, 2), _at(ins, 3), _at(ins, top), _at(ins, g),
                                               _at(ins, u), _at(ins, gt), self.temperature, _at(outs, 0), flags)


class HipTopKDistillation(_RowOp, L.TopKDistillation):
    host_op = L.TopKDistillation

    def call(self, node, ins, outs, flags):
        rc, ws, size = self.workspace(node, ins, lib.thx_topk_distill_workspace)
        return rc or lib.thx_topk_distill_call(_at(ins, 0), _at(ins, 1), _at(ins, 2), self.temperature, _at(outs, 0),
                                               _at(outs, 1), ws.ptr if ws else None, size, flags)


class HipTopKDistillationGrad(_RowOp, L.TopKDistillationGrad):
    host_op = L.TopKDistillationGrad

    def call(self, node, ins, outs, flags):
        return lib.thx_topk_distill_grad_call(_at(ins, 0), _at(ins, 1), _at(ins, 2), _at(ins, 3), _at(ins, 4),
                                              self.temperature, _at(outs, 0), flags)


class _TrainOp(_RowOp):
    """A forward operator and its gradient in one launch, for gradients of the result that do not depend on the result:
    what ``fuse_known_gradients`` makes of the two nodes.  There is no host counterpart."""

    def make_node(self, *inputs):
        ins = [as_hip_variable(i) for i in inputs]
        n = self.n_forward
        outs = self.forward.make_node(*ins[:n]).outputs
        acc = outs[0].type.dtype
        for g in ins[n:]:
            if g.type.dtype != acc or g.type.ndim != ins[0].type.ndim - 1:
                raise TypeError("%s: a gradient of type %s" % (self, g.type))
        return Apply(self, ins, [o.type() for o in outs] + [ins[0].type()])

    def infer_shape(self, node, shapes):
        return self.forward.infer_shape(node, shapes[:self.n_forward]) + [shapes[0]]


class HipTokenLogProbsTrain(_TrainOp, Op):
    """``HipTokenLogProbs`` without alternatives and ``HipTokenLogProbsGrad``; ``given`` says which of the gradients of
    ``log_prob`` and ``entropy`` follow the logits and the tokens."""

    __props__ = ("temperature", "given")
    n_forward = 2

    def __init__(self, temperature, given):
        self.temperature, self.given = float(temperature), tuple(bool(g) for g in given)
        self.forward = HipTokenLogProbs(0, temperature)

    def call(self, node, ins, outs, flags):
        rc, ws, size = self.workspace(node, ins, lib.thx_token_logprob_workspace, 0)
        at = iter(range(2, len(node.inputs)))
        g, u = [next(at) if there else None for there in self.given]
        return rc or lib.thx_token_logprob_train_call(_at(ins, 0), _at(ins, 1), _at(ins, g), _at(ins, u), self.temperature,
                                                      _at(outs, 0), _at(outs, 1), _at(outs, 2), _at(outs, 3),
                                                      ws.ptr if ws else None, size, flags)


class HipTopKDistillationTrain(_TrainOp, Op):
    """``HipTopKDistillation`` and ``HipTopKDistillationGrad``; the gradient of the loss follows the teacher's tokens."""

    __props__ = ("temperature",)
    n_forward = 3

    def __init__(self, temperature):
        self.temperature = float(temperature)
        self.forward = HipTopKDistillation(temperature)

    def call(self, node, ins, outs, flags):
        rc, ws, size = self.workspace(node, ins, lib.thx_topk_distill_workspace)
        return rc or lib.thx_topk_distill_train_call(_at(ins, 0), _at(ins, 1), _at(ins, 2), _at(ins, 3), self.temperature,
                                                     _at(outs, 0), _at(outs, 1), _at(outs, 2), ws.ptr if ws else None,
                                                     size, flags)


class _Apart(object):
    """Rewrites expressions so that they no longer depend on the results of one node, where all they take from them is
    their shape: the fills that sums and means leave in gradients."""

    def __init__(self, node, rows):
        self.node, self.rows = node, rows     # ``rows``: makes a variable with the shape of the node's results per row
        self.known, self.model = {}, None

    def depends(self, v):
        if v not in self.known:
            n = v.owner
            self.known[v] = n is not None and (n is self.node or any(self.depends(i) for i in n.inputs))
        return self.known[v]

    def row_shaped(self, v):
        """Elementwise over a result of the node, and nowhere broadcast against anything larger."""
        first = self.node.outputs[0].type
        n = v.owner
        if n is None or v.type.broadcastable != first.broadcastable:
            return False
        return n is self.node or (isinstance(n.op, Elemwise) and any(self.row_shaped(i) for i in n.inputs))

    def shape_of_rows(self):
        if self.model is None:
            self.model = self.rows()
        return self.model

    def __call__(self, v):
        """``v`` without the dependence, or None."""
        if not self.depends(v):
            return v
        n = v.owner
        if n is self.node:
            return None
        if isinstance(n.op, T.ShapeFloat) and self.row_shaped(n.inputs[0]):
            return n.op(self.shape_of_rows())
        if isinstance(n.op, Elemwise) and isinstance(n.op.scalar_op, scal.Second):
            value = self(n.inputs[1])
            if value is None:
                return None
            if not self.depends(n.inputs[0]):
                model = n.inputs[0]
            elif self.row_shaped(n.inputs[0]):
                model = self.shape_of_rows()
            else:
                return None
            return n.op.make_node(model, value).outputs[0]
        if isinstance(n.op, (Elemwise, DimShuffle)) and not getattr(n.op, "inplace_pattern", None):
            ins = [self(i) for i in n.inputs]
            if any(i is None for i in ins):
                return None
            return n.op.make_node(*ins).outputs[v.index]
        return None


def _one_value(g):
    """The single value that a fill repeats over the rows, if it can be had without a launch or a transfer: such an
    operand is read with a stride of 0."""
    n = g.owner
    if n is None or not isinstance(n.op, Elemwise) or not isinstance(n.op.scalar_op, scal.Second):
        return g
    v = n.inputs[1]
    if v.type.ndim != g.type.ndim or not all(v.type.broadcastable) or v.type.dtype != g.type.dtype:
        return g
    return v if isinstance(v.type, HipArrayType) else g


def fuse_known_gradients(fgraph):
    """A forward node over the vocabulary and its gradient node become one where the gradients of the results do not
    depend on the results: a weighted sum or mean of the losses, not a function such as a ratio of probabilities."""
    count = 0
    for node in fgraph.toposort():
        if node not in fgraph.apply_nodes:
            continue
        if isinstance(node.op, HipTokenLogProbsGrad):
            if node.op.given[2]:
                continue
            fwd, first = node.inputs[2].owner, 4
            if fwd is None or not isinstance(fwd.op, HipTokenLogProbs) or fwd.op.n_top or node.inputs[3] is not fwd.outputs[1]:
                continue
            new_op = HipTokenLogProbsTrain(node.op.temperature, node.op.given[:2])
            rows = lambda: fwd.inputs[1]                                                  # noqa: E731
        elif isinstance(node.op, HipTopKDistillationGrad):
            fwd, first = node.inputs[3].owner, 4
            if fwd is None or not isinstance(fwd.op, HipTopKDistillation):
                continue
            new_op = HipTopKDistillationTrain(node.op.temperature)

            def rows():     # the first entry of every row
                from .views import HipSubtensor
                ids = fwd.inputs[2]
                return HipSubtensor((slice(None),) * (ids.type.ndim - 1) + (0,)).make_node(ids).outputs[0]
        else:
            continue
        n = new_op.n_forward
        if fwd.op.temperature != node.op.temperature or list(fwd.inputs) != list(node.inputs[:n]):
            continue
        apart = _Apart(fwd, rows)
        gs = [apart(g) for g in node.inputs[first:]]
        if any(g is None for g in gs):
            continue
        new = new_op.make_node(*(list(fwd.inputs) + [_one_value(g) for g in gs]))
        if new.outputs[-1].type != node.outputs[0].type:
            continue
        dx = node.outputs[0]
        fgraph.replace(dx, new.outputs[-1])
        for o, no in zip(fwd.outputs, new.outputs):
            fgraph.replace(o, no)
        count += 1
    return count


LIFT = {L.LayerNormalization: lambda op: HipLayerNormalization(op.epsilon),
        L.LayerNormalizationGrad: lambda op: HipLayerNormalizationGrad(op.n_params),
        L.TokenLogProbs: lambda op: HipTokenLogProbs(op.n_top, op.temperature),
        L.TokenLogProbsGrad: lambda op: HipTokenLogProbsGrad(op.temperature, op.given),
        L.TopKDistillation: lambda op: HipTopKDistillation(op.temperature),
        L.TopKDistillationGrad: lambda op: HipTopKDistillationGrad(op.temperature)}

DEVICE_OPS = (_RowOp,)
