"""The row operators at the head of a language model, reached through ``theano_amd.tensor.nnet``: layer
normalisation, log probabilities of given tokens, and distillation from a teacher's best logits.

The reference's ``nnet`` has none of them; they stand beside its batch normalisation
(``theano/tensor/nnet/bn.py:79-263``) and its row softmax and cross-entropies
(``theano/tensor/nnet/nnet.py:411-646, 2053-2102``) and keep their manner: an ``Op`` with ``make_node`` checks and
``L_op``, and a function that builds the node.  Each Op has a device counterpart in ``theano_amd.hip.nnet`` that runs
one hand-written kernel per pass over the data; nothing runs on the host.

Statistics, sums and probabilities are computed in float32 for float16 and float32 data and in float64 for float64
data; every result is rounded once, to its own type.
"""
import math

from .. import scalar as scal
from ..gof import Apply, MethodNotDefined, Op, clone_get_equiv
from . import basic as T
from .elemwise import DimShuffle, Elemwise
from .type import TensorType, as_tensor_variable

_FLOATS = ("float16", "float32", "float64")
_TOKENS = ("int32", "int64")

# most alternatives token_log_probs lists per row: one per lane of a wave while they are selected
MAX_TOP = 64
# most teacher entries per row: the list is held on chip while entries that name the same token are added up
MAX_TEACHER = 1024


def _no_host(op):
    raise NotImplementedError("%s has no host implementation: it is lifted onto its device operator before the graph "
                              "runs" % op)


def compute_dtype(dtype):
    """The type of statistics, sums and probabilities of ``dtype`` data."""
    return "float64" if dtype == "float64" else "float32"


def _is_zero(g):
    """Is ``g`` the gradient of a result that nothing uses: absent, or the zeros ``grad`` puts in its place?"""
    if g is None or isinstance(g.type, scal.DisconnectedType):
        return True
    if g.owner is None or not isinstance(g.owner.op, Elemwise) or not isinstance(g.owner.op.scalar_op, scal.Second):
        return False
    v = g.owner.inputs[1]
    if v.owner is not None and isinstance(v.owner.op, DimShuffle):
        v = v.owner.inputs[0]
    data = getattr(v, "data", None)
    return data is not None and getattr(data, "size", 0) == 1 and float(data.reshape(())) == 0.0


def _disconnected():
    return scal.DisconnectedType()()


# ---- layer normalisation -----------------------------------------------------------------------------------

class LayerNormalization(Op):
    """``(x - mean) * invstd * gamma + beta`` with the mean and the inverse standard deviation
    ``1 / sqrt(var + epsilon)`` of each row (the last axis) of ``x``.  Inputs ``x[, gamma[, beta]]``, outputs ``out,
    mean, invstd``: ``out`` in the type of ``x``, the statistics per row in float32 (float64 for float64)."""

    __props__ = ("epsilon",)

    def __init__(self, epsilon=1e-5):
        self.epsilon = float(epsilon)
        if not (self.epsilon >= 0.0 and math.isfinite(self.epsilon)):
            raise ValueError("epsilon must be a finite number of at least 0, got %s" % epsilon)

    def make_node(self, x, *params):
        x = as_tensor_variable(x)
        params = [as_tensor_variable(p) for p in params]
        if x.type.ndim < 1 or x.type.dtype not in _FLOATS:
            raise TypeError("layer normalization takes a tensor of floats with at least one axis, got %s" % x.type)
        if len(params) > 2:
            raise TypeError("layer normalization takes a scale and a bias")
        for p, n in zip(params, ("gamma", "beta")):
            if p.type.ndim != 1 or p.type.dtype != params[0].type.dtype:
                raise TypeError("%s must be a vector of the type of gamma, got %s" % (n, p.type))
            if p.type.dtype != x.type.dtype and not (x.type.dtype == "float16" and p.type.dtype == "float32"):
                raise TypeError("%s must have the type of the inputs (or float32 beside float16), got %s beside %s"
                                % (n, p.type.dtype, x.type.dtype))
            if p.type.broadcastable[0] and not x.type.broadcastable[-1]:
                raise TypeError("%s must have one element per column of the inputs" % n)
        stat = TensorType(compute_dtype(x.type.dtype), x.type.broadcastable[:-1])
        return Apply(self, [x] + params, [x.type(), stat(), stat()])

    def perform(self, node, inputs, output_storage):
        _no_host(self)

    def infer_shape(self, node, shapes):
        return [shapes[0], shapes[0][:-1], shapes[0][:-1]]

    def L_op(self, inputs, outputs, grads):
        x, params = inputs[0], inputs[1:]
        _, mean, invstd = outputs
        dy, dmean, dinvstd = grads
        acc = mean.type.dtype
        if _is_zero(dy):
            res = [None] * len(inputs)
        else:
            args = [x, dy] + params[:1]
            if x.type.dtype != acc and not (_is_zero(dmean) and _is_zero(dinvstd)):
                args = [T.cast(v, acc) for v in args]       # dx is added to below, and rounded behind that
            res = list(LayerNormalizationGrad(len(params))(*(args[:2] + [mean, invstd] + args[2:]), return_list=True))
            res[1:] = [r if r.type.dtype == p.type.dtype else T.cast(r, p.type.dtype) for r, p in zip(res[1:], params)]
        # what arrives through the statistics: d mean / dx = 1 / n, d invstd / dx = -invstd^3 (x - mean) / n
        nd = x.type.ndim
        col = list(range(nd - 1)) + ["x"]
        n = T.ShapeFloat(nd - 1, acc)(x)
        extra = None
        if not _is_zero(dmean):
            extra = T.second(x, (dmean / n).dimshuffle(*col))
        if not _is_zero(dinvstd):
            term = (-dinvstd * invstd ** 3 / n).dimshuffle(*col) * (x - mean.dimshuffle(*col))
            extra = term if extra is None else extra + term
        if extra is not None:
            res[0] = T.cast(extra if res[0] is None else res[0] + extra, x.type.dtype)
        return [_disconnected() if r is None else r for r in res]

    def connection_pattern(self, node):
        return [[True, True, True]] + [[True, False, False] for _ in node.inputs[1:]]


class LayerNormalizationGrad(Op):
    """The gradients of layer normalisation with respect to ``x`` and its ``n_params`` parameters, from the gradient
    ``dy`` of the result and the saved statistics.  With ``a = dy * gamma`` and ``xhat = (x - mean) * invstd``:
    ``dx = invstd * (a - mean(a) - xhat * mean(a * xhat))``, ``dgamma = sum(dy * xhat)`` and ``dbeta = sum(dy)`` over
    the rows."""

    __props__ = ("n_params",)

    def __init__(self, n_params):
        self.n_params = int(n_params)

    def make_node(self, x, dy, mean, invstd, *gamma):
        x, dy, mean, invstd = [as_tensor_variable(v) for v in (x, dy, mean, invstd)]
        gamma = [as_tensor_variable(v) for v in gamma]
        if x.type.dtype not in _FLOATS or dy.type.dtype != x.type.dtype or dy.type.ndim != x.type.ndim:
            raise TypeError("dy must have the type of x, got %s beside %s" % (dy.type, x.type))
        for v in (mean, invstd):
            if v.type.ndim != x.type.ndim - 1 or v.type.dtype != compute_dtype(x.type.dtype):
                raise TypeError("mean and invstd must hold one %s value per row, got %s" % (compute_dtype(x.type.dtype), v.type))
        if len(gamma) != (1 if self.n_params else 0) or any(g.type.ndim != 1 for g in gamma):
            raise TypeError("gamma must be given as a vector when there are parameters, and only then")
        outs = [x.type()] + [gamma[0].type() for _ in range(self.n_params)]
        return Apply(self, [x, dy, mean, invstd] + gamma, outs)

    def perform(self, node, inputs, output_storage):
        _no_host(self)

    def infer_shape(self, node, shapes):
        return [shapes[0]] + [shapes[4] for _ in range(self.n_params)]

    def graph(self, x, dy, mean, invstd, *gamma):
        """The same gradients as a graph of elementary operations: what second derivatives go through."""
        nd = x.type.ndim
        acc = mean.type.dtype
        col, rows = list(range(nd - 1)) + ["x"], list(range(nd - 1))
        row = ["x"] * (nd - 1) + [0]
        xf, g = T.cast(x, acc), T.cast(dy, acc)
        xhat = (xf - mean.dimshuffle(*col)) * invstd.dimshuffle(*col)
        a = g * T.cast(gamma[0], acc).dimshuffle(*row) if gamma else g
        keep = dict(axis=nd - 1, keepdims=True)
        dx = invstd.dimshuffle(*col) * (a - T.mean(a, **keep) - xhat * T.mean(a * xhat, **keep))
        outs = [T.cast(dx, x.type.dtype)]
        for v in [g * xhat, g][:self.n_params]:
            outs.append(T.cast(T.sum(v, axis=rows) if rows else v, gamma[0].type.dtype))
        return outs

    def L_op(self, inputs, outputs, grads):
        from ..gradient import grad
        # on variables of its own: the statistics are functions of x in the caller's graph, here they are operands
        own = [i.type() for i in inputs]
        known, actual = {}, dict(zip(own, inputs))
        for o, g in zip(self.graph(*own), grads):
            if not _is_zero(g):
                known[o] = g.type()
                actual[known[o]] = g
        if not known:
            return [_disconnected() for _ in inputs]
        res = grad(None, own, known_grads=known, disconnected_inputs="ignore", return_disconnected="None")
        there = [r for r in res if r is not None]
        memo = clone_get_equiv(list(actual), there, copy_inputs=False, memo=actual)
        return [_disconnected() if r is None else memo[r] for r in res]

    def connection_pattern(self, node):
        # dbeta is the sum of dy alone; dgamma does not read gamma
        pat = [[True, True, False], [True, True, True], [True, True, False], [True, True, False], [True, False, False]]
        return [p[:1 + self.n_params] for p in pat[:len(node.inputs)]]


def _row_param(p, x, name):
    """A parameter per column, given as a vector or with the inputs' rank and broadcastable on every axis but the last."""
    p = as_tensor_variable(p)
    if p.type.ndim == 1:
        return p
    if p.type.ndim != x.type.ndim or not all(p.type.broadcastable[:-1]):
        raise ValueError("%s must be a vector with one element per column, or have the rank of the inputs and be "
                         "broadcastable along every axis but the last; got %s" % (name, p.type))
    return p.dimshuffle(p.type.ndim - 1)


def layer_normalization(inputs, gamma=None, beta=None, epsilon=1e-5):
    """Layer normalisation over the last axis: ``(x - mean) / sqrt(var + epsilon) * gamma + beta`` with the mean and
    the (biased) variance of each row.  Returns ``(out, mean, invstd)`` as ``batch_normalization_train`` does; the
    statistics have the shape of the inputs without the last axis.

    ``gamma`` and ``beta`` hold one value per column, as vectors or in the inputs' rank; either both, ``gamma`` alone or
    neither.  ``inputs`` are float16, float32 or float64; parameters have the inputs' type, or float32 beside float16
    inputs (parameters narrower than that are converted).  The result has the inputs' type, the statistics are float32
    (float64 for float64 inputs)."""
    x = as_tensor_variable(inputs)
    if beta is not None and gamma is None:
        raise ValueError("layer_normalization takes beta only together with gamma")
    params = [_row_param(p, x, n) for p, n in ((gamma, "gamma"), (beta, "beta")) if p is not None]
    if params and x.type.dtype in _FLOATS:
        for p, n in zip(params, ("gamma", "beta")):
            if p.type.dtype not in _FLOATS and p.type.dtype not in scal.discrete_dtypes:
                raise TypeError("%s must hold real numbers, got %s" % (n, p.type))
        dt = scal.upcast(*[p.type.dtype for p in params])
        if dt not in _FLOATS or (dt == "float16" and x.type.dtype != "float16") or (dt == "float32" and x.type.dtype == "float64"):
            dt = x.type.dtype
        params = [T.cast(p, dt) if p.type.dtype != dt else p for p in params]
    return tuple(LayerNormalization(epsilon)(x, *params, return_list=True))


# ---- operators over the vocabulary -------------------------------------------------------------------------

def _temperature(t):
    t = float(t)
    if not (1e-6 <= t <= 1e6):
        raise ValueError("temperature must lie between 1e-6 and 1e6, got %s" % t)
    return t


def _check_logits(x, who):
    if x.type.ndim < 2 or x.type.dtype not in _FLOATS:
        raise TypeError("%s takes logits of floats with at least two axes, the last one the vocabulary, got %s" % (who, x.type))


def _lead_type(x, dtype):
    return TensorType(dtype, x.type.broadcastable[:-1])


class TokenLogProbs(Op):
    """Log probability of one given token per row of ``logits / temperature``, the row's entropy and its ``n_top`` most
    probable tokens.  Inputs ``logits, tokens``; outputs ``log_prob, entropy[, top_log_probs, top_tokens], stats``:
    ``stats`` holds each row's largest logit and the binary logarithm of ``sum(exp((logits - largest) /
    temperature))``, which the gradient reads."""

    __props__ = ("n_top", "temperature")

    def __init__(self, n_top=0, temperature=1.0):
        self.n_top = int(n_top)
        self.temperature = _temperature(temperature)
        if not 0 <= self.n_top <= MAX_TOP:
            raise ValueError("n_top must lie between 0 and %d, got %s" % (MAX_TOP, n_top))

    def make_node(self, logits, tokens):
        x, tokens = as_tensor_variable(logits), as_tensor_variable(tokens)
        _check_logits(x, "token_log_probs")
        if tokens.type.dtype not in _TOKENS or tokens.type.ndim != x.type.ndim - 1:
            raise TypeError("tokens must hold one int32 or int64 index per row of the logits, got %s" % tokens.type)
        acc = compute_dtype(x.type.dtype)
        row = _lead_type(x, acc)
        lead = x.type.broadcastable[:-1]
        outs = [row(), row()]
        if self.n_top:
            outs += [TensorType(dt, lead + (self.n_top == 1,))() for dt in (acc, "int64")]
        return Apply(self, [x, tokens], outs + [TensorType(acc, lead + (False,))()])

    def perform(self, node, inputs, output_storage):
        _no_host(self)

    def infer_shape(self, node, shapes):
        lead = tuple(shapes[0][:-1])
        return [lead, lead] + ([lead + (self.n_top,)] * 2 if self.n_top else []) + [lead + (2,)]

    def L_op(self, inputs, outputs, grads):
        x, tokens = inputs
        g = [None if _is_zero(v) else v for v in (grads[0], grads[1], grads[2] if self.n_top else None)]
        if g == [None, None, None]:
            return [_disconnected(), _disconnected()]
        given = tuple(v is not None for v in g)
        args = [x, tokens, outputs[-1], outputs[1]] + ([outputs[3]] if given[2] else []) + [v for v in g if v is not None]
        return [TokenLogProbsGrad(self.temperature, given)(*args), _disconnected()]

    def connection_pattern(self, node):
        n = len(node.outputs)
        top = [True, False] if self.n_top else []
        return [[True, True] + top + [False], [False] * n]


class TokenLogProbsGrad(Op):
    """The gradient of the logits for given gradients of ``log_prob``, ``entropy`` and ``top_log_probs`` (``given`` says
    which of them there are).  With ``p`` the probabilities, ``w`` the gradient of the token's log probability, ``c_k``
    those of the alternatives' and ``u`` that of the entropy ``H``:
    ``dx_j = ([j = token] w + sum_k [j = top_k] c_k - p_j (w + sum_k c_k + u (log p_j + H))) / temperature``."""

    __props__ = ("temperature", "given")

    def __init__(self, temperature, given):
        self.temperature = float(temperature)
        self.given = tuple(bool(g) for g in given)

    def make_node(self, logits, tokens, stats, entropy, *rest):
        ins = [as_tensor_variable(v) for v in (logits, tokens, stats, entropy) + rest]
        if len(rest) != sum(self.given) + self.given[2]:
            raise TypeError("TokenLogProbsGrad: %d operands for the gradients %s" % (len(rest), self.given))
        x = ins[0]
        acc = compute_dtype(x.type.dtype)
        for v in ins[2:4] + ins[4 + self.given[2]:]:
            if v.type.dtype != acc:
                raise TypeError("TokenLogProbsGrad takes %s statistics and gradients beside %s logits, got %s"
                                % (acc, x.type.dtype, v.type))
        return Apply(self, ins, [x.type()])

    def perform(self, node, inputs, output_storage):
        _no_host(self)

    def infer_shape(self, node, shapes):
        return [shapes[0]]

    def L_op(self, inputs, outputs, grads):
        raise MethodNotDefined("L_op", "second derivatives of token_log_probs")


def _tokens(v, name):
    v = as_tensor_variable(v)
    if v.type.dtype not in scal.discrete_dtypes or v.type.dtype == "bool":
        raise TypeError("%s must be integers, got %s" % (name, v.type))
    return v if v.type.dtype in _TOKENS else T.cast(v, "int64")


def token_log_probs(logits, tokens, n_top=0, temperature=1.0):
    """Log probabilities of given tokens: with ``z = logits / temperature`` and ``p = softmax(z)`` along the last axis,
    returns ``(log_prob, entropy)``, or ``(log_prob, entropy, top_log_probs, top_tokens)`` when ``n_top`` (at most 64,
    and no more than there are columns) is not 0:

    ``log_prob``       ``log p`` at each row's token, ``tokens`` having the shape of the logits without the last axis
    ``entropy``        ``-sum(p * log p)`` of each row
    ``top_log_probs``  the ``n_top`` largest ``log p`` of each row in falling order, along a new last axis
    ``top_tokens``     where they are (int64); of equal logits the lowest index comes first, NaN counts as largest

    Results are float32 (float64 for float64 logits).  All three floating-point results carry a gradient to the logits.

    A logit of -infinity is a token that cannot occur: probability 0, log probability -infinity, and a gradient of 0 unless
    it is the row's given token (or among its alternatives), whose own weight it gets.  A row of nothing else has log probabilities of -infinity, an entropy of 0 and no gradient.  A negative token stands for none
    (padding): ``log_prob`` 0, no gradient through it.  A token beyond the last column makes its row's ``log_prob`` NaN,
    and the row's gradient where the one of ``log_prob`` is asked for.  NaN or +infinity among a row's logits make its
    floating-point results and its gradient NaN."""
    outs = TokenLogProbs(n_top, temperature)(as_tensor_variable(logits), _tokens(tokens, "tokens"), return_list=True)
    return tuple(outs[:-1])


class TopKDistillation(Op):
    """Loss of each row of ``logits`` against a teacher's best logits (see ``topk_distillation_loss``).  Inputs
    ``logits, teacher_logits, teacher_tokens``; outputs ``loss, stats``: ``stats`` holds the row's largest logit and the
    binary logarithm of its sum of exponentials, and the same of the teacher's."""

    __props__ = ("temperature",)

    def __init__(self, temperature=1.0):
        self.temperature = _temperature(temperature)

    def make_node(self, logits, teacher_logits, teacher_tokens):
        x, t, ids = [as_tensor_variable(v) for v in (logits, teacher_logits, teacher_tokens)]
        _check_logits(x, "topk_distillation_loss")
        if t.type.dtype not in _FLOATS or t.type.ndim != x.type.ndim:
            raise TypeError("teacher_logits must be floats of the logits' rank, got %s" % t.type)
        if ids.type.dtype not in _TOKENS or ids.type.ndim != x.type.ndim:
            raise TypeError("teacher_tokens must be int32 or int64 of the logits' rank, got %s" % ids.type)
        acc = compute_dtype(x.type.dtype)
        return Apply(self, [x, t, ids], [_lead_type(x, acc)(), TensorType(acc, x.type.broadcastable[:-1] + (False,))()])

    def perform(self, node, inputs, output_storage):
        _no_host(self)

    def infer_shape(self, node, shapes):
        lead = tuple(shapes[0][:-1])
        return [lead, lead + (4,)]

    def L_op(self, inputs, outputs, grads):
        if _is_zero(grads[0]):
            return [_disconnected()] * 3
        dx = TopKDistillationGrad(self.temperature)(inputs[0], inputs[1], inputs[2], outputs[1], grads[0])
        return [dx, _disconnected(), _disconnected()]

    def connection_pattern(self, node):
        return [[True, False], [False, False], [False, False]]


class TopKDistillationGrad(Op):
    """``dx_j = g * temperature * (p_j * sum(q) - sum_k q_k [j = token_k])`` with ``g`` the gradient of the row's loss,
    ``p`` the student's and ``q`` the teacher's probabilities."""

    __props__ = ("temperature",)

    def __init__(self, temperature):
        self.temperature = float(temperature)

    def make_node(self, logits, teacher_logits, teacher_tokens, stats, g_loss):
        ins = [as_tensor_variable(v) for v in (logits, teacher_logits, teacher_tokens, stats, g_loss)]
        acc = compute_dtype(ins[0].type.dtype)
        if any(v.type.dtype != acc for v in ins[3:]):
            raise TypeError("TopKDistillationGrad takes %s statistics and gradients beside %s logits" % (acc, ins[0].type.dtype))
        return Apply(self, ins, [ins[0].type()])

    def perform(self, node, inputs, output_storage):
        _no_host(self)

    def infer_shape(self, node, shapes):
        return [shapes[0]]

    def L_op(self, inputs, outputs, grads):
        raise MethodNotDefined("L_op", "second derivatives of topk_distillation_loss")


def topk_distillation_loss(logits, teacher_logits, teacher_tokens, temperature=1.0):
    """Distillation from a teacher of which each row's best logits are known: ``teacher_logits`` and ``teacher_tokens``
    (integers) have the shape of the logits but for the last axis, which holds 1 to 1024 entries.  With ``q`` the
    softmax of a row's ``teacher_logits / temperature`` over its entries and ``p`` that of ``logits / temperature`` over
    the vocabulary, the loss of a row is ``temperature**2 * sum(q * (log q - log p[teacher_tokens]))``; returned with the
    shape of the logits without the last axis, in float32 (float64 for float64 logits).

    The teacher is a constant: the gradient goes to the logits alone.  An entry with a negative token stands for none
    (rows with fewer entries), one with a teacher's logit of -infinity has ``q = 0`` and counts for nothing; a row
    without entries has loss and gradient 0.  A token named twice gets both shares.  A logit of -infinity under an entry
    with ``q > 0`` makes the loss infinite and leaves the gradient finite; a row of nothing but -infinity has no gradient.
    A token beyond the last column makes its row's loss and gradient NaN, as do NaN or +infinity among its logits."""
    op = TopKDistillation(temperature)
    return op(as_tensor_variable(logits), as_tensor_variable(teacher_logits), _tokens(teacher_tokens, "teacher_tokens"),
              return_list=True)[0]
