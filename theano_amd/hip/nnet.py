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
from .runtime import HipArray, _Buffer, _CODE_OF, _c_strides, call_flags, check, lib, mark_reused, thx_array

_UNSUPPORTED = 6


class _RowOp(object):
    """``make_node`` and the calling sequence shared by the operators; ``call(node, ins, outs)`` gives the library
    function, its arguments up to the workspace, and the query for the workspace's size with its arguments (None where
    the function takes no workspace)."""

    def make_node(self, *inputs):
        ins = [as_hip_variable(i) for i in inputs]
        host = self.host_op.make_node(self, *[TensorType(i.type.dtype, i.type.broadcastable)() for i in ins])
        if [i.type.dtype for i in host.inputs] != [i.type.dtype for i in ins]:
            raise TypeError("%s: operands of types %s" % (self, [str(i.type) for i in ins]))
        return Apply(self, ins, [HipArrayType(o.type.dtype, o.type.broadcastable)() for o in host.outputs])

    def perform(self, node, inputs, output_storage):
        state = node.tag.get("thx")
        if state is None:
            state = node.tag["thx"] = _State(self, node)
        results = state.run(inputs, call_flags(node))
        for k, arr in enumerate(results):
            output_storage[k][0] = arr


class _State(object):
    """What a node keeps from one call to the next: the descriptors of its operands and results, the library call's
    arguments (addresses of those descriptors), and for the layout of the last call the results' shapes, the offsets of
    the small ones in a buffer they share, and the size of the workspace.  No values and no addresses of data."""

    _SHARED = 1 << 16      # results of up to so many bytes lie in one buffer with others of the same call

    def __init__(self, op, node):
        self.op, self.node = op, node
        self.ins = (thx_array * len(node.inputs))()
        self.outs = (thx_array * len(node.outputs))()
        self.in_slots, self.out_slots = list(self.ins), list(self.outs)
        self.dtypes = [np.dtype(o.type.dtype) for o in node.outputs]
        fn, args, self.query = op.call(node, self.ins, self.outs)
        # the call without the declared types, whose check of every argument costs more than the library's: all that is
        # passed is made here or below, as what the declaration says (an int is a C int)
        self.fn = lib[fn.__name__]
        self.args = tuple(ctypes.c_double(a) if isinstance(a, float) else a for a in args)
        self.layout = None

    def plan(self, inputs, layout):
        """Everything of a call that depends on the operands' layout alone."""
        self.layout = None
        for v, slot in zip(inputs, self.in_slots):
            v.as_thx(slot)
        shapes = [tuple(s) for s in self.op.infer_shape(self.node, [v.shape for v in inputs])]
        self.results, at = [], 0
        for shape, dtype in zip(shapes, self.dtypes):
            nbytes = dtype.itemsize
            for s in shape:
                nbytes *= s
            if nbytes <= self._SHARED:
                offset, at = at, at + (nbytes + 63) // 64 * 64
            else:
                offset = None
            self.results.append((shape, _c_strides(shape, dtype.itemsize), dtype, _CODE_OF[dtype], nbytes, offset))
        self.shared_bytes = max(at, 1) if any(r[5] is not None for r in self.results) else 0
        for (shape, strides, dtype, code, nbytes, offset), slot in zip(self.results, self.out_slots):
            slot.offset_bytes, slot.nd, slot.dtype = offset or 0, len(shape), code
            slot.shape[:len(shape)] = shape
            slot.strides_bytes[:len(shape)] = strides
        mark_reused(self.node, self.ins, self.outs)
        self.workspace = ctypes.c_size_t()
        if self.query is not None:
            rc = self.query[0](*(self.query[1:] + (ctypes.byref(self.workspace),)))
            if rc:
                return rc
        self.layout = layout
        return 0

    def run(self, inputs, flags):
        layout = [(v.shape, v.strides) for v in inputs]
        rc = 0
        if layout != self.layout:
            rc = self.plan(inputs, layout)
        else:
            for v, slot in zip(inputs, self.in_slots):
                slot.base = v.buffer.ptr
                slot.offset_bytes = v.offset
        if not rc:
            shared = _Buffer(self.shared_bytes) if self.shared_bytes else None
            results = []
            for (shape, strides, dtype, code, nbytes, offset), slot in zip(self.results, self.out_slots):
                buffer = _Buffer(nbytes) if offset is None else shared
                slot.base = buffer.ptr
                results.append(HipArray._raw(buffer, offset or 0, shape, strides, dtype, code))
            if self.query is None:
                rc = self.fn(*self.args, flags)
            else:
                # kept for the length of the call alone, or by the recording the call is made in
                ws = _Buffer(self.workspace.value) if self.workspace.value else None
                rc = self.fn(*self.args, ctypes.c_void_p(ws.ptr) if ws else None, self.workspace, flags)
            if not rc:
                return results
        if rc == _UNSUPPORTED:          # rows at more than one stride, or columns apart
            copies = [v if v.c_contiguous else v.copy() for v in inputs]
            if any(c is not v for c, v in zip(copies, inputs)):
                return self.run(copies, flags)
        check(rc)


def _at(arrays, k):
    return ctypes.byref(arrays[k]) if k is not None else None


class HipLayerNormalization(_RowOp, L.LayerNormalization):
    host_op = L.LayerNormalization

    def call(self, node, ins, outs):
        n = len(node.inputs)
        return lib.thx_layernorm_call, (_at(ins, 0), _at(ins, 1 if n > 1 else None), _at(ins, 2 if n > 2 else None),
                                        self.epsilon, _at(outs, 0), _at(outs, 1), _at(outs, 2)), None


class HipLayerNormalizationGrad(_RowOp, L.LayerNormalizationGrad):
    host_op = L.LayerNormalizationGrad

    def call(self, node, ins, outs):
        n = self.n_params
        dgamma = _at(outs, 1 if n else None)
        return lib.thx_layernorm_grad_call, (
            _at(ins, 0), _at(ins, 1), _at(ins, 4 if n else None), _at(ins, 2), _at(ins, 3), _at(outs, 0), dgamma,
            _at(outs, 2 if n > 1 else None)), (lib.thx_layernorm_grad_workspace, _at(ins, 0), dgamma)


class HipTokenLogProbs(_RowOp, L.TokenLogProbs):
    host_op = L.TokenLogProbs

    def call(self, node, ins, outs):
        k = self.n_top
        return lib.thx_token_logprob_call, (
            _at(ins, 0), _at(ins, 1), self.temperature, k, _at(outs, 0), _at(outs, 1), _at(outs, 2 if k else None),
            _at(outs, 3 if k else None), _at(outs, 4 if k else 2)), (lib.thx_token_logprob_workspace, _at(ins, 0), k)


class HipTokenLogProbsGrad(_RowOp, L.TokenLogProbsGrad):
    host_op = L.TokenLogProbsGrad

    def call(self, node, ins, outs):
        at = iter(range(4, len(node.inputs)))
        top = next(at) if self.given[2] else None
        g, u, gt = [next(at) if there else None for there in self.given]
        return lib.thx_token_logprob_grad_call, (_at(ins, 0), _at(ins, 1), _at(ins, 2), _at(ins, 3), _at(ins, top),
                                                 _at(ins, g), _at(ins, u), _at(ins, gt), self.temperature,
                                                 _at(outs, 0)), None


class HipTopKDistillation(_RowOp, L.TopKDistillation):
    host_op = L.TopKDistillation

    def call(self, node, ins, outs):
        return lib.thx_topk_distill_call, (_at(ins, 0), _at(ins, 1), _at(ins, 2), self.temperature, _at(outs, 0),
                                           _at(outs, 1)), (lib.thx_topk_distill_workspace, _at(ins, 0))


class HipTopKDistillationGrad(_RowOp, L.TopKDistillationGrad):
    host_op = L.TopKDistillationGrad

    def call(self, node, ins, outs):
        return lib.thx_topk_distill_grad_call, (_at(ins, 0), _at(ins, 1), _at(ins, 2), _at(ins, 3), _at(ins, 4),
                                                self.temperature, _at(outs, 0)), None


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


class HipLayerNormalizationTrain(_RowOp, Op):
    """``HipLayerNormalization`` and ``HipLayerNormalizationGrad`` for a ``dy`` that does not depend on the result (the
    first step back of a part of a model whose forward pass is run again): ``x, dy[, gamma[, beta]]``, then the results
    of both."""

    __props__ = ("epsilon", "n_params")

    def __init__(self, epsilon, n_params):
        self.epsilon, self.n_params = float(epsilon), int(n_params)

    def make_node(self, x, dy, *params):
        x, dy = as_hip_variable(x), as_hip_variable(dy)
        params = [as_hip_variable(p) for p in params]
        outs = HipLayerNormalization(self.epsilon).make_node(x, *params).outputs
        grads = HipLayerNormalizationGrad(self.n_params).make_node(x, dy, outs[1], outs[2], *params[:1]).outputs
        return Apply(self, [x, dy] + params, [o.type() for o in outs + grads])

    def infer_shape(self, node, shapes):
        return [shapes[0], shapes[0][:-1], shapes[0][:-1], shapes[0]] + [shapes[2] for _ in range(self.n_params)]

    def call(self, node, ins, outs):
        n = self.n_params
        dgamma = _at(outs, 4 if n else None)
        return lib.thx_layernorm_train_call, (
            _at(ins, 0), _at(ins, 1), _at(ins, 2 if n else None), _at(ins, 3 if n > 1 else None), self.epsilon, _at(outs, 0),
            _at(outs, 1), _at(outs, 2), _at(outs, 3), dgamma, _at(outs, 5 if n > 1 else None)), (
            lib.thx_layernorm_grad_workspace, _at(ins, 0), dgamma)


class HipTokenLogProbsTrain(_TrainOp, Op):
    """``HipTokenLogProbs`` without alternatives and ``HipTokenLogProbsGrad``; ``given`` says which of the gradients of
    ``log_prob`` and ``entropy`` follow the logits and the tokens."""

    __props__ = ("temperature", "given")
    n_forward = 2

    def __init__(self, temperature, given):
        self.temperature, self.given = float(temperature), tuple(bool(g) for g in given)
        self.forward = HipTokenLogProbs(0, temperature)

    def call(self, node, ins, outs):
        at = iter(range(2, len(node.inputs)))
        g, u = [next(at) if there else None for there in self.given]
        return lib.thx_token_logprob_train_call, (
            _at(ins, 0), _at(ins, 1), _at(ins, g), _at(ins, u), self.temperature, _at(outs, 0), _at(outs, 1), _at(outs, 2),
            _at(outs, 3)), (lib.thx_token_logprob_workspace, _at(ins, 0), 0)


class HipTopKDistillationTrain(_TrainOp, Op):
    """``HipTopKDistillation`` and ``HipTopKDistillationGrad``; the gradient of the loss follows the teacher's tokens."""

    __props__ = ("temperature",)
    n_forward = 3

    def __init__(self, temperature):
        self.temperature = float(temperature)
        self.forward = HipTopKDistillation(temperature)

    def call(self, node, ins, outs):
        return lib.thx_topk_distill_train_call, (
            _at(ins, 0), _at(ins, 1), _at(ins, 2), _at(ins, 3), self.temperature, _at(outs, 0), _at(outs, 1),
            _at(outs, 2)), (lib.thx_topk_distill_workspace, _at(ins, 0))


class _Apart(object):
    """Rewrites expressions so that they no longer depend on the results of one node, where all they take from them is
    their shape: the fills that sums and means leave in gradients."""

    _DEEP = 64      # such fills are a few nodes; what is deeper stays as it is

    def __init__(self, node, rows, order):
        self.node, self.rows = node, rows     # ``rows``: makes a variable with the shape of the node's results per row
        self.order = order                    # place of every node of the graph; none ahead of ``node`` depends on it
        self.free, self.shaped, self.done, self.model = set(), {}, {}, None

    def depends(self, v):
        """Graphs are deep and their nodes shared: every variable is visited once, without recursion."""
        place = self.order.get(self.node, -1)
        seen, todo = set(), [v]
        while todo:
            w = todo.pop()
            n = w.owner
            if n is self.node:
                return True
            if n is None or w in seen or w in self.free or self.order.get(n, place) < place:
                continue
            seen.add(w)
            todo.extend(n.inputs)
        self.free |= seen
        return False

    def row_shaped(self, v, depth=0):
        """Elementwise over a result of the node, and nowhere broadcast against anything larger."""
        n = v.owner
        if n is None or depth > self._DEEP or v.type.broadcastable != self.node.outputs[0].type.broadcastable:
            return False
        if v not in self.shaped:
            self.shaped[v] = n is self.node or (isinstance(n.op, Elemwise) and
                                                any(self.row_shaped(i, depth + 1) for i in n.inputs))
        return self.shaped[v]

    def shape_of_rows(self):
        if self.model is None:
            self.model = self.rows()
        return self.model

    def __call__(self, v, depth=0):
        """``v`` without the dependence, or None."""
        if v not in self.done:
            self.done[v] = self.rewritten(v, depth) if depth <= self._DEEP else None
        return self.done[v]

    def rewritten(self, v, depth):
        if not self.depends(v):
            return v
        n = v.owner
        if n is self.node:
            return None
        if isinstance(n.op, T.ShapeFloat) and self.row_shaped(n.inputs[0]):
            return n.op(self.shape_of_rows())
        if isinstance(n.op, Elemwise) and isinstance(n.op.scalar_op, scal.Second):
            value = self(n.inputs[1], depth + 1)
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
            ins = []
            for i in n.inputs:
                ins.append(self(i, depth + 1))
                if ins[-1] is None:
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


def _places(fgraph):
    return dict((n, k) for k, n in enumerate(fgraph.toposort()))


def _fuse_layer_normalization(fgraph, node, order):
    x, dy, mean, invstd = node.inputs[:4]
    fwd = mean.owner
    if fwd is None or not isinstance(fwd.op, HipLayerNormalization) or [mean, invstd] != list(fwd.outputs[1:]):
        return 0
    if fwd.inputs[0] is not x or list(fwd.inputs[1:2]) != list(node.inputs[4:5]) or len(fwd.inputs) - 1 != node.op.n_params:
        return 0
    dy = _Apart(fwd, lambda: x, order)(dy)
    if dy is None:
        return 0
    new = HipLayerNormalizationTrain(fwd.op.epsilon, node.op.n_params).make_node(x, dy, *fwd.inputs[1:])
    old = list(fwd.outputs) + list(node.outputs)
    if [o.type for o in old] != [o.type for o in new.outputs]:
        return 0
    for o, no in reversed(list(zip(old, new.outputs))):
        fgraph.replace(o, no)
    return 1


def fuse_known_gradients(fgraph):
    """A forward node and its gradient node become one where the gradients of the results do not depend on the results:
    a weighted sum or mean of losses, not a function such as a ratio of probabilities; of layer normalisation a gradient
    that is an argument."""
    count = 0
    order = _places(fgraph)
    for node in list(order):
        if node not in fgraph.apply_nodes:
            continue
        if isinstance(node.op, HipLayerNormalizationGrad):
            if _fuse_layer_normalization(fgraph, node, order):
                order = _places(fgraph)      # what read the result may now stand behind more than it did
                count += 1
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
        apart = _Apart(fwd, rows, order)
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
        order = _places(fgraph)
        count += 1
    return count


LIFT = {L.LayerNormalization: lambda op: HipLayerNormalization(op.epsilon),
        L.LayerNormalizationGrad: lambda op: HipLayerNormalizationGrad(op.n_params),
        L.TokenLogProbs: lambda op: HipTokenLogProbs(op.n_top, op.temperature),
        L.TokenLogProbsGrad: lambda op: HipTokenLogProbsGrad(op.temperature, op.given),
        L.TopKDistillation: lambda op: HipTopKDistillation(op.temperature),
        L.TopKDistillationGrad: lambda op: HipTopKDistillationGrad(op.temperature)}

DEVICE_OPS = (_RowOp,)
