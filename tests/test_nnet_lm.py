"""Layer normalisation, token log probabilities and distillation without a device: node construction, gradient graphs,
what is refused, and the library's checks of its operands in dry-run mode."""
import ctypes

import numpy as np
import pytest

import theano_amd as th
from theano_amd import hip, tensor as T
from theano_amd.gradient import DisconnectedInputError
from theano_amd.hip import runtime
from theano_amd.hip.runtime import HipArray, lib, thx_array
from theano_amd.tensor import nnet


def tensor(dtype, nd):
    return T.TensorType(dtype, (False,) * nd)()


def device_nodes(f):
    return [type(n.op).__name__ for n in f.toposort() if type(n.op).__name__ not in ("HostToHip", "HipToHost")]


def test_types_of_the_results():
    for dt, p, acc in [("float16", "float16", "float32"), ("float16", "float32", "float32"), ("float32", "float32", "float32"),
                       ("float64", "float64", "float64")]:
        x, g = tensor(dt, 3), tensor(p, 1)
        y, m, i = nnet.layer_normalization(x, g, g)
        assert (y.type.dtype, m.type.dtype, i.type.dtype) == (dt, acc, acc)
        assert (y.type.ndim, m.type.ndim, i.type.ndim) == (3, 2, 2)
        assert [v.type.dtype for v in th.grad(None, [x, g], known_grads={y: x})] == [dt, p]
        lp, h, tv, ti = nnet.token_log_probs(x, T.imatrix(), n_top=5)
        assert (lp.type.dtype, h.type.dtype, tv.type.dtype, ti.type.dtype) == (acc, acc, acc, "int64")
        assert (lp.type.ndim, h.type.ndim, tv.type.ndim, ti.type.ndim) == (2, 2, 3, 3)
        loss = nnet.topk_distillation_loss(x, tensor("float16", 3), T.itensor3())
        assert loss.type.dtype == acc and loss.type.ndim == 2
        assert th.grad(T.sum(loss), x).type == x.type
    assert len(nnet.token_log_probs(T.fmatrix(), T.lvector())) == 2


def test_parameters_in_either_form_and_type():
    x = T.ftensor3()
    row = T.TensorType("float32", (True, True, False))
    y = nnet.layer_normalization(x, row(), row())[0]
    assert y.type == x.type
    assert nnet.layer_normalization(T.dmatrix(), T.fvector())[0].type.dtype == "float64"
    assert nnet.layer_normalization(T.fmatrix(), T.hvector(), T.fvector())[0].type.dtype == "float32"
    assert nnet.layer_normalization(T.hmatrix(), T.hvector(), T.fvector())[0].type.dtype == "float16"
    with pytest.raises(TypeError, match="type of the inputs"):
        nnet.layer_normalization(T.fmatrix(), T.dvector())
    with pytest.raises(TypeError, match="type of the inputs"):
        nnet.layer_normalization(T.hmatrix(), T.dvector())
    with pytest.raises(ValueError, match="gamma must be a vector"):
        nnet.layer_normalization(x, T.fmatrix())
    with pytest.raises(ValueError, match="only together"):
        nnet.layer_normalization(x, None, T.fvector())
    with pytest.raises(TypeError, match="one element per column"):
        nnet.layer_normalization(x, T.TensorType("float32", (True,))())
    for bad in (T.imatrix(), T.fscalar(), T.cmatrix()):
        with pytest.raises(TypeError):
            nnet.layer_normalization(bad)
    with pytest.raises(TypeError):
        nnet.layer_normalization(x, T.cvector())
    for eps in (-1e-5, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="epsilon"):
            nnet.layer_normalization(x, epsilon=eps)


def test_what_the_vocabulary_operators_refuse():
    x = T.fmatrix()
    for bad in (T.fvector(), T.imatrix()):
        with pytest.raises(TypeError):
            nnet.token_log_probs(bad, T.lvector())
        with pytest.raises(TypeError):
            nnet.topk_distillation_loss(bad, T.fmatrix(), T.lmatrix())
    for tokens in (T.fvector(), T.lmatrix(), T.lscalar(), T.TensorType("bool", (False,))()):
        with pytest.raises(TypeError, match="tokens"):
            nnet.token_log_probs(x, tokens)
    for n in (-1, 65):
        with pytest.raises(ValueError, match="n_top"):
            nnet.token_log_probs(x, T.lvector(), n_top=n)
    for t in (0.0, -1.0, float("nan"), float("inf"), 1e-9):
        with pytest.raises(ValueError, match="temperature"):
            nnet.token_log_probs(x, T.lvector(), temperature=t)
        with pytest.raises(ValueError, match="temperature"):
            nnet.topk_distillation_loss(x, x, T.lmatrix(), temperature=t)
    with pytest.raises(TypeError, match="teacher_logits"):
        nnet.topk_distillation_loss(x, T.imatrix(), T.lmatrix())
    with pytest.raises(TypeError, match="teacher_tokens"):
        nnet.topk_distillation_loss(x, x, T.lvector())
    with pytest.raises(TypeError, match="teacher_tokens"):
        nnet.topk_distillation_loss(x, x, x)


def test_layer_normalization_with_a_known_gradient_is_one_node(dry_run):
    x, g, b, dy = T.fmatrix(), T.fvector(), T.fvector(), T.fmatrix()
    y, mean, invstd = nnet.layer_normalization(x, g, b)
    norms = lambda f: [n for n in device_nodes(f) if n.startswith("HipLayer")]       # noqa: E731
    one, two = ["HipLayerNormalizationTrain"], ["HipLayerNormalization", "HipLayerNormalizationGrad"]
    known = th.grad(None, [x, g, b], known_grads={y: dy})
    assert norms(th.function([x, g, b, dy], [y, mean] + known)) == one
    assert norms(th.function([x, g, b, dy], known)) == one
    assert norms(th.function([x, g, b, dy], known, fuse=False)) == two
    assert norms(th.function([x, g, b], th.grad(T.sum(y), [x, g, b]))) == one
    # a gradient that hangs on the result, or on the statistics
    assert norms(th.function([x, g, b], th.grad(T.sum(T.sqr(y)), x))) == two
    assert norms(th.function([x, g, b, dy], th.grad(None, x, known_grads={y: dy * mean.dimshuffle(0, "x")}))) == two
    # of two layers the second alone
    z = nnet.layer_normalization(y, g)[0]
    f = th.function([x, g, b, dy], th.grad(None, [x, g, b], known_grads={z: dy}))
    assert sorted(norms(f)) == sorted(one + two)
    # statistics of another call on the same rows are not its own
    other = nnet.layer_normalization(x, g, b, epsilon=1e-3)
    f = th.function([x, g, b, dy], known + [other[0]])
    assert sorted(norms(f)) == sorted(one + two[:1])


def test_known_gradients_are_looked_for_in_deep_and_shared_graphs(dry_run):
    """Far more nodes between a result and its gradient than the interpreter nests calls, and far more paths than nodes."""
    from theano_amd.hip.nnet import _Apart
    x, g = T.fmatrix(), T.fvector()
    y = nnet.layer_normalization(x, g)[0]
    deep, shared = y, y
    for _ in range(3000):
        deep = T.tanh(deep)
    for _ in range(200):
        shared = shared * shared
    order = {}
    for v in (deep, shared):
        apart = _Apart(y.owner, lambda: x, order)
        assert apart.depends(v) and not apart.depends(x * 2) and apart(v) is None
        assert apart(T.second(v, x)) is None                 # the shape of something that far is not looked into
        assert apart(x * 2).owner.inputs[0] is x
    z = y
    for _ in range(60):
        z = nnet.layer_normalization(z * z + 1, g)[0]
    f = th.function([x, g], th.grad(T.sum(z), x))
    assert device_nodes(f).count("HipLayerNormalizationTrain") == 1


def test_known_gradients_make_no_cycle(dry_run):
    """Two results that are each other's gradients: when the one pair has become one node, the other's gradient hangs on it."""
    a, b = T.fmatrix(), T.fmatrix()
    ya, yb = nnet.layer_normalization(a)[0], nnet.layer_normalization(b)[0]
    f = th.function([a, b], [th.grad(None, a, known_grads={ya: yb * 2}), th.grad(None, b, known_grads={yb: ya * 3})])
    names = [n for n in device_nodes(f) if n.startswith("HipLayer")]
    assert sorted(names) == ["HipLayerNormalization", "HipLayerNormalizationGrad", "HipLayerNormalizationTrain"]


def test_narrow_token_types_are_converted():
    for dt in ("int8", "uint8", "int16", "uint16", "uint32", "uint64"):
        assert nnet.token_log_probs(T.fmatrix(), tensor(dt, 1))[0].type.dtype == "float32"


def test_gradient_graphs(dry_run):
    """One node per pass: results that nothing uses cost nothing, and their missing gradients are not made up."""
    x, g, b = T.fmatrix(), T.fvector(), T.fvector()
    y = nnet.layer_normalization(x, g, b)[0]
    f = th.function([x, g, b], th.grad(T.sum(y), [x, g, b]), fuse=False)
    names = device_nodes(f)
    assert names.count("HipLayerNormalization") == 1 and names.count("HipLayerNormalizationGrad") == 1
    t, w = T.lvector(), T.fvector()
    lp, h, tv, ti = nnet.token_log_probs(x, t, n_top=3)
    f = th.function([x, t, w], th.grad(None, x, known_grads={lp: w}), fuse=False)
    assert device_nodes(f) == ["HipTokenLogProbs", "HipTokenLogProbsGrad"]
    assert f.toposort()[-2].op.given == (True, False, False)
    f = th.function([x, t, w], th.grad(None, x, known_grads={h: w}), fuse=False)
    assert f.toposort()[-2].op.given == (False, True, False)
    ids, teacher = T.imatrix(), T.fmatrix()
    loss = nnet.topk_distillation_loss(x, teacher, ids)
    with pytest.raises(DisconnectedInputError):
        th.grad(T.sum(loss), teacher)
    with pytest.raises(DisconnectedInputError):
        th.grad(T.sum(lp), t)
    with pytest.raises(NotImplementedError, match="second derivatives|gradient"):
        th.grad(T.sum(T.sqr(th.grad(T.sum(lp), x))), x)
    with pytest.raises(NotImplementedError):
        th.Rop(lp, x, T.fmatrix())
    # equal calls on the same variables are one node
    f = th.function([x, t], [nnet.token_log_probs(x, t)[0], nnet.token_log_probs(x, t)[1]])
    assert device_nodes(f) == ["HipTokenLogProbs"]


def test_one_launch_for_a_loss_and_its_gradient(dry_run):
    """Gradients of the results that do not depend on the results are known before the launch."""
    x, t, w = T.fmatrix(), T.lvector(), T.fvector()
    ids, teacher = T.imatrix(), T.fmatrix()
    lp, h = nnet.token_log_probs(x, t)
    kd = nnet.topk_distillation_loss(x, teacher, ids)

    def names(cost, **kw):
        ins = [x, t, w, ids, teacher]
        f = th.function(ins, [cost, th.grad(cost, x)], on_unused_input="ignore", **kw)
        return [n for n in device_nodes(f) if "Token" in n or "TopK" in n]

    for cost in (T.sum(-w * lp), T.mean(-lp), -T.sum(w * lp) / T.sum(w), T.sum(w * lp + np.float32(0.1) * h), T.mean(h),
                 T.sum(w * lp) + T.mean(T.exp(w) * h)):
        assert names(cost) == ["HipTokenLogProbsTrain"], cost
        assert names(cost, fuse=False) == ["HipTokenLogProbs", "HipTokenLogProbsGrad"]
    for cost in (T.sum(w * kd), T.mean(kd), T.sum(kd)):
        assert names(cost) == ["HipTopKDistillationTrain"], cost
    # the mean's weight is read as one value for all rows
    f = th.function([x, teacher, ids], th.grad(T.mean(kd), x))
    node = [n for n in f.toposort() if type(n.op).__name__ == "HipTopKDistillationTrain"][0]
    assert node.inputs[3].type.broadcastable == (True,)
    f(np.zeros((3, 5), "float32"), np.zeros((3, 2), "float32"), np.zeros((3, 2), "int32"))
    # functions of the results themselves are not
    for cost in (T.sum(T.exp(lp - w)), T.sum(lp * h), T.sum(T.sqr(h))):
        assert names(cost) == ["HipTokenLogProbs", "HipTokenLogProbsGrad"], cost
    assert names(T.sum(T.sqr(kd))) == ["HipTopKDistillation", "HipTopKDistillationGrad"]
    assert names(T.sum(w * lp) + T.sum(T.sqr(kd))) == ["HipTokenLogProbsTrain", "HipTopKDistillation", "HipTopKDistillationGrad"]
    # both losses of one batch of logits
    assert sorted(names(T.sum(w * lp) + T.mean(kd))) == ["HipTokenLogProbsTrain", "HipTopKDistillationTrain"]


def test_shapes_that_do_not_fit(dry_run):
    def z(*shape, **kw):
        return np.zeros(shape, kw.get("dt", "float32"))

    x, g, b, dy = T.fmatrix(), T.fvector(), T.fvector(), T.fmatrix()
    y = nnet.layer_normalization(x, g, b)[0]
    f = th.function([x, g, b], y)
    f(z(3, 5), z(5), z(5))
    for bad in ((z(3, 5), z(4), z(5)), (z(3, 5), z(5), z(6)), (z(3, 5), z(1), z(5))):
        with pytest.raises(ValueError, match="mis-match"):
            f(*bad)
    f = th.function([x, g, b, dy], th.grad(None, x, known_grads={y: dy}))
    with pytest.raises(ValueError, match="mis-match"):
        f(z(3, 5), z(5), z(5), z(2, 5))
    t = T.lvector()
    f = th.function([x, t], list(nnet.token_log_probs(x, t, n_top=4)))
    f(z(3, 5), z(3, dt="int64"))
    for bad, word in (((z(3, 5), z(2, dt="int64")), "mis-match"), ((z(3, 3), z(3, dt="int64")), "alternatives"),
                      ((z(3, 0), z(3, dt="int64")), "columns")):
        with pytest.raises(ValueError, match=word):
            f(*bad)
    ids = T.imatrix()
    f = th.function([x, dy, ids], nnet.topk_distillation_loss(x, dy, ids))
    f(z(3, 5), z(3, 9), z(3, 9, dt="int32"))
    for bad, word in (((z(3, 5), z(3, 9), z(3, 8, dt="int32")), "mis-match"), ((z(3, 5), z(2, 9), z(2, 9, dt="int32")), "mis-match"),
                      ((z(3, 5), z(3, 0), z(3, 0, dt="int32")), "entries"),
                      ((z(3, 5), z(3, 1025), z(3, 1025, dt="int32")), "entries")):
        with pytest.raises(ValueError, match=word):
            f(*bad)


def descriptors(*arrays):
    out = []
    for a in arrays:
        d = thx_array()
        if a is not None:
            a.as_thx(d)
        out.append(d)
    return out


def test_the_library_checks_its_operands():
    """Straight calls of the C interface with operands that do not fit: a code and a message, nothing is launched.  No
    device is needed: each is refused before one is looked for."""
    fake = 1 << 40

    def arr(shape, dtype, base=fake, strides=None, code=None):
        a = thx_array()
        a.base, a.offset_bytes, a.nd = base, 0, len(shape)
        a.dtype = runtime._CODE_OF[np.dtype(dtype)] if code is None else code
        size = np.dtype(dtype).itemsize
        for d, s in enumerate(shape):
            a.shape[d] = s
            a.strides_bytes[d] = strides[d] if strides else int(np.prod(shape[d + 1:], dtype="int64")) * size
        return a

    step = [0]

    def at(shape, dtype, **kw):
        step[0] += 1
        return arr(shape, dtype, base=fake + (step[0] << 24), **kw)

    def refused(rc, code, word):
        assert rc == code, (rc, lib.thx_last_error())
        assert word in lib.thx_last_error().decode(), lib.thx_last_error()

    def ln(x=None, g=None, b=None, y=None, m=None, i=None, eps=1e-5, flags=0):
        parts = [at((4, 8), "float32") if x is None else x, g, b, at((4, 8), "float32") if y is None else y,
                 at((4,), "float32") if m is None else m, at((4,), "float32") if i is None else i]
        refs = [None if p is None or p == "null" else ctypes.byref(p) for p in parts]
        return lib.thx_layernorm_call(refs[0], refs[1], refs[2], eps, refs[3], refs[4], refs[5], flags)

    refused(ln(x="null"), 7, "missing")
    refused(ln(y="null"), 7, "missing")
    refused(ln(x=at((4, 8), "int32")), 3, "dtype")
    refused(ln(x=at((4, 8), "float32", code=runtime._CODE_OF[np.dtype("float32")] | runtime.THX_HOST_SCALAR)), 3, "device array")
    refused(ln(x=arr((4, 8), "float32", base=None)), 7, "no base")
    refused(ln(x=arr((4, 8), "float32", base=fake + 2)), 3, "aligned")
    refused(ln(x=at((4, 8), "float32", strides=(34, 4))), 3, "multiple")
    refused(ln(x=at((4, 8), "float32", strides=(4, 16))), 6, "side by side")
    refused(ln(x=at((2, 2, 8), "float32", strides=(32, 64, 4)), y=at((2, 2, 8), "float32"), m=at((2, 2), "float32"),
               i=at((2, 2), "float32")), 6, "one stride")
    refused(ln(b=at((8,), "float32")), 7, "beta without gamma")
    refused(ln(g=at((8,), "float64")), 3, "parameters")
    refused(ln(g=at((7,), "float32")), 2, "mis-match")
    refused(ln(y=at((4, 7), "float32")), 2, "mis-match")
    refused(ln(y=at((4, 8), "float16")), 3, "dtype")
    refused(ln(y=at((4, 8), "float32", strides=(64, 4))), 3, "C-contiguous")
    refused(ln(m=at((4,), "float64")), 3, "dtype")
    refused(ln(eps=-1.0), 7, "epsilon")
    refused(ln(eps=float("nan")), 7, "epsilon")
    x = at((4, 8), "float32")
    refused(ln(x=x, y=x), 7, "overlaps")
    m = at((4,), "float32")
    refused(ln(m=m, i=m), 7, "overlap")
    ext = at((4, 8), "float32")
    ext.shape[0] = -4
    refused(ln(x=ext), 7, "negative")
    big = at((4, 8), "float32")
    big.nd = 9
    refused(ln(x=big), 3, "rank")

    def lng(ws=fake, size=1 << 20, dg="yes", g="yes", db=None):
        a = [at((4, 8), "float32"), at((4, 8), "float32"), at((8,), "float32") if g else None, at((4,), "float32"),
             at((4,), "float32"), at((4, 8), "float32"), at((8,), "float32") if dg else None, db]
        return lib.thx_layernorm_grad_call(*([None if p is None else ctypes.byref(p) for p in a] + [ws, size, 0]))

    refused(lng(size=0), 7, "workspace of")
    refused(lng(ws=None), 7, "no address")
    refused(lng(ws=fake + 8), 7, "16 bytes")
    refused(lng(g=None), 7, "without gamma")
    refused(lng(dg=None, db=at((8,), "float32")), 7, "without dgamma")

    def lnt(**kw):
        a = dict(x=at((4, 8), "float32"), dy=at((4, 8), "float32"), g=at((8,), "float32"), b=at((8,), "float32"),
                 y=at((4, 8), "float32"), m=at((4,), "float32"), i=at((4,), "float32"), dx=at((4, 8), "float32"),
                 dg=at((8,), "float32"), db=at((8,), "float32"), ws=fake, size=1 << 20, eps=1e-5)
        a.update((k, a[v] if isinstance(v, str) else v) for k, v in kw.items())
        r = [None if a[k] is None else ctypes.byref(a[k]) for k in ("x", "dy", "g", "b", "y", "m", "i", "dx", "dg", "db")]
        return lib.thx_layernorm_train_call(*(r[:4] + [a["eps"]] + r[4:] + [a["ws"], a["size"], 0]))

    refused(lnt(x=None), 7, "missing")
    refused(lnt(dy=None), 7, "missing")
    refused(lnt(dy=at((4, 7), "float32")), 2, "mis-match")
    refused(lnt(dy=at((4, 8), "float16")), 3, "dtype")
    refused(lnt(dy=arr((4, 8), "float32", base=None)), 7, "no base")
    refused(lnt(eps=-1.0), 7, "epsilon")
    refused(lnt(g=None), 7, "without gamma")
    refused(lnt(dg=None), 7, "without dgamma")
    refused(lnt(y="dy"), 7, "overlaps")
    refused(lnt(dx="dy"), 7, "overlaps")
    refused(lnt(dx="y"), 7, "overlap")
    refused(lnt(dg="b"), 7, "overlaps")
    refused(lnt(size=0), 7, "workspace of")
    refused(lnt(ws=None), 7, "no address")
    refused(lnt(ws=fake + 8), 7, "16 bytes")

    def lp(V=8, t="int64", k=0, temp=1.0, top="yes", rows=4, x=None):
        a = [at((rows, V), "float32") if x is None else x, at((rows,), t)]
        o = [at((rows,), "float32"), at((rows,), "float32"), at((rows, k), "float32") if k > 0 and top else None,
             at((rows, k), "int64") if k > 0 else None, at((rows, 2), "float32")]
        r = [None if p is None else ctypes.byref(p) for p in a + o]
        return lib.thx_token_logprob_call(r[0], r[1], temp, k, r[2], r[3], r[4], r[5], r[6], fake, 1 << 20, 0)

    refused(lp(t="float32"), 3, "int32 or int64")
    refused(lp(k=9), 7, "alternatives")
    refused(lp(k=-1), 7, "alternatives")
    refused(lp(k=65, V=100), 7, "alternatives")
    refused(lp(k=3, top=None), 7, "missing")
    refused(lp(temp=0.0), 7, "temperature")
    refused(lp(V=0), 7, "columns")
    wide = at((1, 8), "float32")
    wide.shape[1] = 1 << 31
    refused(lp(x=wide, rows=1), 6, "columns")

    def kd(n=3, tdt="float32", idt="int32", m=None):
        a = [at((4, 8), "float32"), at((4, n), tdt), at((4, n if m is None else m), idt)]
        o = [at((4,), "float32"), at((4, 4), "float32")]
        r = [ctypes.byref(p) for p in a + o]
        return lib.thx_topk_distill_call(r[0], r[1], r[2], 1.0, r[3], r[4], fake, 1 << 20, 0)

    refused(kd(tdt="int32"), 3, "teacher")
    refused(kd(idt="int16"), 3, "int32 or int64")
    refused(kd(n=0), 7, "entries")
    refused(kd(n=1025), 7, "entries")
    refused(kd(m=4), 2, "mis-match")
    for call, n in ((lib.thx_layernorm_grad_workspace, 2), (lib.thx_topk_distill_workspace, 1)):
        refused(call(*([None] * (n + 1))), 7, "null")
    refused(lib.thx_token_logprob_workspace(None, 0, None), 7, "null")


def test_operands_that_are_not_rows_are_copied(dry_run):
    """Rows at more than one stride, or columns apart: the operator copies them, whatever the operand."""
    x, t = T.ftensor3(), T.lmatrix()
    f = th.function([x, t], [th.Out(o, device=True) for o in nnet.token_log_probs(x, t)])
    a = HipArray.empty((3, 4, 5), "float32")
    i = HipArray.empty((4, 3), "int64")
    got = f(a.view((4, 3, 5), (20, 80, 4)), i)
    assert got[0].shape == (4, 3)
    f(HipArray.empty((5, 4, 3), "float32").transpose(), HipArray.empty((3, 4), "int64"))
    f(HipArray.empty((4, 3, 5), "float32"), HipArray.empty((3, 4), "int64").transpose())


def test_views_of_other_libraries_arrays(dry_run):
    class Other(object):
        def __init__(self, **kw):
            self.__cuda_array_interface__ = dict({"typestr": "<f4", "shape": (3, 4), "data": (1 << 20, False), "version": 3}, **kw)

    a = HipArray.from_cuda_array_interface(Other())
    assert a.shape == (3, 4) and a.strides == (16, 4) and a.ptr == 1 << 20 and a.buffer.owner is not None
    a = HipArray.from_cuda_array_interface(Other(strides=(4, 12)))
    assert a.strides == (4, 12)
    for bad in (dict(typestr="<U4"), dict(typestr=">f4"), dict(mask=1), dict(shape=(1,) * 9)):
        with pytest.raises(TypeError):
            HipArray.from_cuda_array_interface(Other(**bad))
    assert HipArray.from_cuda_array_interface(Other(shape=(0, 4), data=(0, False))).shape == (0, 4)
    assert not hasattr(HipArray.empty((3,), "float32"), "__cuda_array_interface__")     # no memory behind it here


def test_other_libraries_arrays_that_cannot_be_taken(dry_run):
    class Other(object):
        def __init__(self, **kw):
            self.__cuda_array_interface__ = dict({"typestr": "<f4", "shape": (3,), "data": (1 << 20, False), "version": 3}, **kw)

    for stream in (None, 1, 2, 1 << 30):
        assert HipArray.from_cuda_array_interface(Other(stream=stream)).shape == (3,)
    with pytest.raises(ValueError, match="ambiguous"):
        HipArray.from_cuda_array_interface(Other(stream=0))
    from theano_amd.tensor import inplace
    x, y = T.fvector(), T.fvector()
    f = th.function([x, y], inplace.add_inplace(x, y), accept_inplace=True)
    plain, fixed = [HipArray.from_cuda_array_interface(Other(data=(1 << 20, ro))) for ro in (False, True)]
    f(plain, fixed)
    with pytest.raises(ValueError, match="read-only"):
        f(fixed, plain)
