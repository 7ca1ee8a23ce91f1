"""Device versions of the row operators of ``theano_amd.tensor.nnet_lm``.

Each subclasses its host counterpart, as the other device ops do (``ops.py``), and runs one call of the library:
the kernels are compiled into it, so nothing is built at run time.  An operand whose rows do not lie at one stride (a
transposed view, say) is copied to a C-contiguous array first; every other layout is read where it lies.
"""
import ctypes

import numpy as np

from ..gof import Apply
from ..tensor import nnet_lm as L
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


LIFT = {L.LayerNormalization: lambda op: HipLayerNormalization(op.epsilon),
        L.LayerNormalizationGrad: lambda op: HipLayerNormalizationGrad(op.n_params),
        L.TokenLogProbs: lambda op: HipTokenLogProbs(op.n_top, op.temperature),
        L.TokenLogProbsGrad: lambda op: HipTokenLogProbsGrad(op.temperature, op.given),
        L.TopKDistillation: lambda op: HipTopKDistillation(op.temperature),
        L.TopKDistillationGrad: lambda op: HipTopKDistillationGrad(op.temperature)}

DEVICE_OPS = (_RowOp,)
