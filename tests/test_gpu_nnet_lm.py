"""Layer normalisation, token log probabilities and distillation on the device, against plain NumPy in float64.

Tolerances are counted in roundings.  A result may be off by half a step of its own type (``eps / 2`` of the value, and
half the smallest subnormal) for the one rounding at the end, plus ``n`` roundings of the type it is computed in,
``eps(acc) / 2`` each, of the ``scale`` of what is added up on the way (the sum of the moduli of the terms).  ``n`` is
the longest chain of roundings: a row of C columns is summed by 64 lanes or more, so at most C / 64 additions in one lane
and 6 + 4 between lanes and waves; 16 more cover the conversions, products, exponential, logarithm and square root of one
element (each within a unit of the last place)."""
import numpy as np
import pytest

import theano_amd as th
from theano_amd import hip, tensor as T
from theano_amd.compile import Out
from theano_amd.hip.runtime import HipArray
from theano_amd.hip.views import copy_into

pytestmark = pytest.mark.gpu

INF = float("inf")


def acc_of(dtype):
    return "float64" if dtype == "float64" else "float32"


def chain(cols, rows=0):
    return 26 + cols / 64 + rows


def close(got, ref, scale, n, what, acc, flush=0.0):
    """``acc``: the type the result was computed in; ``flush``: what a result may lack where an exponential on the way to
    it lies below the smallest normal number of that type."""
    got = np.asarray(got)
    fin = np.isfinite(ref)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    g = got.astype("float64")
    with np.errstate(over="ignore"):
        out = ref.astype(got.dtype).astype("float64")
    over = fin & ~np.isfinite(out)          # beyond the type's range: infinity, or the largest finite value
    np.testing.assert_array_equal(g[~fin], ref[~fin], err_msg=what)
    info = np.finfo(got.dtype)
    assert (np.abs(g[over]) >= float(info.max)).all(), what
    fin &= ~over
    tol = (float(info.eps) / 2 * np.abs(ref) + float(info.smallest_subnormal) / 2 +
           n * float(np.finfo(acc).eps) / 2 * np.broadcast_to(scale, ref.shape) + flush)
    with np.errstate(invalid="ignore"):
        bad = fin & ~(np.abs(g - ref) <= tol)
    assert not bad.any(), "%s: %d of %d values, first at %s: got %r, expected %r within %r" % (
        what, bad.sum(), bad.size, tuple(np.argwhere(bad)[0]), g[bad][0], ref[bad][0], tol[bad][0])


# ---- plain forms in float64 --------------------------------------------------------------------------------

def ln_ref(x, gamma, beta, eps, dy=None):
    """(name -> (value, scale)) of layer normalisation over the last axis."""
    with np.errstate(all="ignore"):
        x = x.astype("float64")
        mean = x.mean(-1, keepdims=True)
        xc = x - mean
        inv = 1 / np.sqrt((xc * xc).mean(-1, keepdims=True) + eps)
        xhat = xc * inv
        big = np.abs(x).max(-1, keepdims=True) if x.shape[-1] else np.zeros(x.shape[:-1] + (1,))
        mag = np.abs(xhat) + big * inv          # of x * invstd and mean * invstd, whose difference xhat is
        g = np.ones(x.shape[-1]) if gamma is None else gamma.astype("float64")
        b = np.zeros(x.shape[-1]) if beta is None else beta.astype("float64")
        # an error of the variance is one of invstd: relative to the squares that were added
        rel = 1 + (mag * mag).mean(-1, keepdims=True) if x.shape[-1] else 1
        out = {"y": (xhat * g + b, mag * rel * np.abs(g) + np.abs(b)), "mean": (mean[..., 0], big[..., 0]),
               "invstd": (inv[..., 0], (inv * rel)[..., 0])}
        if dy is not None:
            dy = dy.astype("float64")
            a = dy * g
            lead = tuple(range(x.ndim - 1))
            out["dx"] = (inv * (a - a.mean(-1, keepdims=True) - xhat * (a * xhat).mean(-1, keepdims=True)),
                         inv * rel * (np.abs(a) + np.abs(a).mean(-1, keepdims=True) +
                                      2 * mag * (np.abs(a) * mag).mean(-1, keepdims=True)))
            out["dgamma"] = ((dy * xhat).sum(lead), (np.abs(dy) * mag * rel).sum(lead))
            out["dbeta"] = (dy.sum(lead), np.abs(dy).sum(lead))
        return out


def log_softmax(z):
    """Of the last axis in float64; -infinity where nothing is left, NaN where there is a NaN or +infinity."""
    with np.errstate(all="ignore"):
        m = z.max(-1, keepdims=True) if z.shape[-1] else np.full(z.shape[:-1] + (1,), -INF)
        none = (z == -INF).all(-1, keepdims=True)
        d = z - np.where(none, 0.0, m)
        return np.where(none, -INF, d - np.log(np.exp(d).sum(-1, keepdims=True))), none


def order_of(x, k):
    """Columns of the k largest logits of each row: NaN first, then by value, then by position."""
    key = np.where(np.isnan(x), INF, x.astype("float64"))
    nan = np.isnan(x)
    at = np.broadcast_to(np.arange(x.shape[-1]), x.shape)
    return np.lexsort((at, -key, ~nan), axis=-1)[..., :k]


def lp_ref(x, tokens, temperature=1.0, n_top=0, w=None, u=None, c=None):
    with np.errstate(all="ignore"):
        z = x.astype("float64") / temperature
        V = z.shape[-1]
        logp, none = log_softmax(z)
        p = np.exp(logp)
        fin = np.where(p > 0, logp, np.where(np.isnan(p), np.nan, 0.0))
        H = -(p * fin).sum(-1)
        have, far = tokens >= 0, tokens >= V
        at = np.where(have & ~far, tokens, 0)[..., None].astype("int64")
        lp = np.where(have, np.take_along_axis(logp, at, -1)[..., 0], 0.0)
        lp = np.where(far, np.nan, lp)
        out = {"log_prob": (lp, 1 + np.where(np.isfinite(lp), np.abs(lp), 0)), "entropy": (H, 1 + np.abs(H))}
        if n_top:
            top = order_of(x, n_top)
            tv = np.take_along_axis(logp, top, -1)
            out["top"] = (tv, 1 + np.where(np.isfinite(tv), np.abs(tv), 0))
            out["top_at"] = top
        if w is not None or u is not None or c is not None:
            zero = np.zeros(tokens.shape)
            wt = np.where(have, zero if w is None else w.astype("float64"), 0.0)
            ut = (zero if u is None else u.astype("float64"))[..., None]
            a, mag = wt[..., None], np.abs(wt)[..., None]
            if c is not None:
                a = a + c.astype("float64").sum(-1, keepdims=True)
                mag = mag + np.abs(c.astype("float64")).sum(-1, keepdims=True)
            dz = -p * (a + ut * (fin + H[..., None]))
            scale = p * (1 + np.abs(fin)) * (mag + np.abs(ut) * (1 + np.abs(fin) + np.abs(H[..., None])))
            for idx, v in [(at, wt[..., None])] + ([(top, c.astype("float64"))] if c is not None else []):
                for k in range(idx.shape[-1]):
                    i = idx[..., k:k + 1]
                    for arr, add in ((dz, v[..., k:k + 1]), (scale, np.abs(v[..., k:k + 1]))):
                        np.put_along_axis(arr, i, np.take_along_axis(arr, i, -1) + add, -1)
            dz = np.where(none, 0.0, dz / temperature)
            if w is not None:
                dz = np.where(far[..., None], np.nan, dz)
            out["dx"] = (dz, np.where(np.isfinite(scale), scale, 0) / temperature)
        return out


def kd_ref(x, teacher, ids, temperature=1.0, g=None):
    with np.errstate(all="ignore"):
        z = x.astype("float64") / temperature
        V, T_ = z.shape[-1], temperature
        logp, none = log_softmax(z)
        t = np.where(ids >= 0, teacher.astype("float64") / T_, -INF)
        logq, tnone = log_softmax(t)
        q = np.exp(logq)
        far = (ids >= V).any(-1) | np.isnan(z).any(-1) | (z == INF).any(-1)
        at = np.clip(ids, 0, V - 1).astype("int64")
        lp = np.take_along_axis(logp, at, -1)
        loss = T_ ** 2 * np.where(q > 0, q * (logq - lp), np.where(np.isnan(q), np.nan, 0.0)).sum(-1)
        mag = T_ ** 2 * (1 + np.where(q > 0, q * (2 + np.abs(logq) + np.where(np.isfinite(lp), np.abs(lp), 0)), 0).sum(-1))
        loss = np.where(far, np.nan, loss)
        out = {"loss": (loss, mag)}
        if g is not None:
            g = g.astype("float64")[..., None] * T_
            p = np.exp(logp)
            dz = p * q.sum(-1, keepdims=True)
            scale = p * (1 + np.where(p > 0, np.abs(logp), 0))
            for k in range(ids.shape[-1]):
                i = at[..., k:k + 1]
                for arr, add in ((dz, -q[..., k:k + 1]), (scale, (q * (1 + np.where(q > 0, np.abs(logq), 0)))[..., k:k + 1])):
                    np.put_along_axis(arr, i, np.take_along_axis(arr, i, -1) + add, -1)
            dz = np.where(none, 0.0, g * dz)
            out["dx"] = (np.where(far[..., None], np.nan, dz), np.where(np.isfinite(scale), scale, 0) * np.abs(g))
        return out


# ---- the functions under test ------------------------------------------------------------------------------

def tensor(dtype, nd, name=None):
    return T.TensorType(dtype, (False,) * nd)(name)


_cache = {}


def ln_function(dtype, pdtype, nd, n_params, eps, train, fuse=True):
    """``fuse``: the forward pass and the gradients in one launch, else two."""
    key = ("ln", dtype, pdtype, nd, n_params, eps, train, fuse)
    if key not in _cache:
        x, dy = tensor(dtype, nd), tensor(dtype, nd)
        ps = [tensor(pdtype, 1) for _ in range(n_params)]
        outs = list(T.nnet.layer_normalization(x, *ps, epsilon=eps))
        ins = [x] + ps
        if train:
            outs += th.grad(None, ins, known_grads={outs[0]: dy})
            ins = ins + [dy]
        _cache[key] = th.function(ins, [Out(o, device=True) for o in outs], fuse=fuse)
    return _cache[key]


def lp_function(dtype, idt, nd, n_top, temperature, given, fuse=True):
    """``fuse``: the forward pass and the gradient in one launch (without alternatives), else two."""
    key = ("lp", dtype, idt, nd, n_top, temperature, given, fuse)
    if key not in _cache:
        acc = acc_of(dtype)
        x, t = tensor(dtype, nd), tensor(idt, nd - 1)
        outs = list(T.nnet.token_log_probs(x, t, n_top=n_top, temperature=temperature))
        cot = [tensor(acc, nd - 1), tensor(acc, nd - 1), tensor(acc, nd)]
        known = dict((outs[k], cot[k]) for k in range(3) if given[k])
        ins = [x, t] + [cot[k] for k in range(3) if given[k]]
        if known:
            outs.append(th.grad(None, x, known_grads=known))
        _cache[key] = th.function(ins, [Out(o, device=True) for o in outs], fuse=fuse)
    return _cache[key]


def kd_function(dtype, tdt, idt, nd, temperature, train, fuse=True):
    key = ("kd", dtype, tdt, idt, nd, temperature, train, fuse)
    if key not in _cache:
        x, t, ids = tensor(dtype, nd), tensor(tdt, nd), tensor(idt, nd)
        g = tensor(acc_of(dtype), nd - 1)
        loss = T.nnet.topk_distillation_loss(x, t, ids, temperature=temperature)
        outs = [loss] + ([th.grad(None, x, known_grads={loss: g})] if train else [])
        _cache[key] = th.function([x, t, ids] + ([g] if train else []), [Out(o, device=True) for o in outs], fuse=fuse)
    return _cache[key]


def check_ln(x, gamma, beta, dy=None, eps=1e-5, dev=None, what=""):
    """``dev``: device arrays that hold the same values in another layout, by position of the argument."""
    ref = ln_ref(x, gamma, beta, eps, dy)
    for fuse in ([True, False] if dy is not None else [False]):
        check_ln_call(x, gamma, beta, dy, eps, dev, ref, fuse, what)


def check_ln_call(x, gamma, beta, dy, eps, dev, ref, fuse, what):
    ps = [p for p in (gamma, beta) if p is not None]
    f = ln_function(str(x.dtype), str(ps[0].dtype) if ps else "float32", x.ndim, len(ps), eps, dy is not None, fuse)
    assert any(type(n.op).__name__ == "HipLayerNormalizationTrain" for n in f.toposort()) == fuse
    args = [x] + ps + ([dy] if dy is not None else [])
    for k, v in (dev or {}).items():
        args[k] = v
    got = [o.to_numpy() for o in f(*args)]
    names = ["y", "mean", "invstd"] + (["dx", "dgamma", "dbeta"][:1 + len(ps)] if dy is not None else [])
    acc = acc_of(str(x.dtype))
    assert len(got) == len(names)
    rows = int(np.prod(x.shape[:-1]))
    for g, name in zip(got, names):
        assert str(g.dtype) == (str(x.dtype) if name in ("y", "dx") else acc if name in ("mean", "invstd") else str(ps[0].dtype))
        n = chain(x.shape[-1], rows if name in ("dgamma", "dbeta") else 0)
        close(g, ref[name][0], ref[name][1], n, "%s %s" % (what, name), acc)


def check_lp(x, tokens, temperature=1.0, n_top=0, w=None, u=None, c=None, dev=None, what=""):
    given = tuple(v is not None for v in (w, u, c))
    ref = lp_ref(x, tokens, temperature, n_top, w, u, c)
    for fuse in ([True, False] if any(given) and not n_top else [False]):
        check_lp_call(x, tokens, temperature, n_top, given, [v for v in (w, u, c) if v is not None], dev, ref, fuse, what)


def check_lp_call(x, tokens, temperature, n_top, given, cotangents, dev, ref, fuse, what, flush=0.0):
    f = lp_function(str(x.dtype), str(tokens.dtype), x.ndim, n_top, temperature, given, fuse)
    assert any(type(n.op).__name__ == "HipTokenLogProbsTrain" for n in f.toposort()) == fuse
    args = [x, tokens] + cotangents
    for k, v in (dev or {}).items():
        args[k] = v
    got = [o.to_numpy() for o in f(*args)]
    acc, n = acc_of(str(x.dtype)), chain(x.shape[-1])
    close(got[0], *ref["log_prob"], n, what + " log_prob", acc)
    close(got[1], *ref["entropy"], n, what + " entropy", acc)
    assert got[0].dtype == got[1].dtype == np.dtype(acc)
    if n_top:
        assert got[3].dtype == np.int64
        np.testing.assert_array_equal(got[3], ref["top_at"], err_msg=what)
        close(got[2], *ref["top"], n, what + " top_log_probs", acc)
    if any(given):
        assert got[-1].dtype == x.dtype
        close(got[-1], *ref["dx"], n, what + " dlogits", acc, flush)


def check_kd(x, teacher, ids, temperature=1.0, g=None, dev=None, what=""):
    ref = kd_ref(x, teacher, ids, temperature, g)
    for fuse in ([True, False] if g is not None else [False]):
        check_kd_call(x, teacher, ids, temperature, g, dev, ref, fuse, what)


def check_kd_call(x, teacher, ids, temperature, g, dev, ref, fuse, what, flush=0.0):
    f = kd_function(str(x.dtype), str(teacher.dtype), str(ids.dtype), x.ndim, temperature, g is not None, fuse)
    assert any(type(n.op).__name__ == "HipTopKDistillationTrain" for n in f.toposort()) == fuse
    args = [x, teacher, ids] + ([g] if g is not None else [])
    for k, v in (dev or {}).items():
        args[k] = v
    got = [o.to_numpy() for o in f(*args)]
    acc, n = acc_of(str(x.dtype)), chain(x.shape[-1]) + ids.shape[-1]
    assert got[0].dtype == np.dtype(acc)
    close(got[0], *ref["loss"], n, what + " loss", acc)
    if g is not None:
        assert got[1].dtype == x.dtype
        close(got[1], *ref["dx"], n, what + " dlogits", acc, flush)


def logits(rng, shape, dtype, spread=3.0):
    return (spread * rng.standard_normal(shape)).astype(dtype)


# ---- layer normalisation -----------------------------------------------------------------------------------

LN_SHAPES = [(1, 1), (1, 1024), (3, 2), (7, 63), (5, 64), (4, 65), (300, 33), (2, 3, 129), (2, 1, 3, 40), (64, 768), (13, 769),
             (9, 1023), (33, 2048), (5, 2049), (3, 4097), (2, 8191), (3, 8192), (2, 16384), (2, 16385), (2, 40001), (1500, 16),
             (700, 1000), (130, 5000)]


@pytest.mark.parametrize("dtype,pdtype", [("float16", "float16"), ("float16", "float32"), ("float32", "float32"),
                                          ("float64", "float64")])
@pytest.mark.parametrize("shape", LN_SHAPES, ids=str)
def test_layer_normalization_and_its_gradients(shape, dtype, pdtype):
    rng = np.random.default_rng(sum(shape) * 7 + len(dtype + pdtype))
    x = (2 * rng.standard_normal(shape) + rng.standard_normal(shape[:-1] + (1,))).astype(dtype)
    gamma, beta = [(1 - k + 0.2 * rng.standard_normal(shape[-1])).astype(pdtype) for k in range(2)]
    dy = rng.standard_normal(shape).astype(dtype)
    check_ln(x, gamma, beta, dy, what=str(shape))


@pytest.mark.parametrize("n_params", [0, 1])
@pytest.mark.parametrize("dtype", ["float16", "float32", "float64"])
def test_layer_normalization_without_parameters(dtype, n_params):
    rng = np.random.default_rng(5)
    for shape in [(6, 100), (40, 1024), (3, 9000)]:
        x, dy = [rng.standard_normal(shape).astype(dtype) for _ in range(2)]
        gamma = rng.standard_normal(shape[-1]).astype(dtype) if n_params else None
        check_ln(x, gamma, None, dy, what="%s %d" % (shape, n_params))


def test_layer_normalization_of_rows_far_from_zero():
    """The variance is taken around the mean: rows at 1000 with a spread of 1 keep their digits."""
    rng = np.random.default_rng(6)
    for dtype, at in (("float32", 1000.0), ("float16", 100.0), ("float64", 1e6)):
        x = (at + rng.standard_normal((20, 1536))).astype(dtype)
        one = np.ones(1536, dtype)
        check_ln(x, one, one, rng.standard_normal(x.shape).astype(dtype), what=dtype)
    x = np.full((4, 512), 3.0, "float32")       # no spread at all: invstd = 1 / sqrt(epsilon)
    check_ln(x, None, None, rng.standard_normal(x.shape).astype("float32"))
    x = np.full((3, 4096), 60000.0, "float16")  # squares and sums beyond the type's range
    x[:, ::2] = -60000.0
    check_ln(x, None, None, rng.standard_normal(x.shape).astype("float16"))


def test_layer_normalization_with_nan_and_infinity():
    """They stay in their own row of the result and of dx, and reach the gradients of the parameters of their column."""
    x = np.random.default_rng(7).standard_normal((5, 300)).astype("float32")
    x[1, 17], x[3, 2] = np.nan, INF
    dy = np.ones_like(x)
    f = ln_function("float32", "float32", 2, 2, 1e-5, True)
    y, mean, inv, dx, dg, db = [o.to_numpy() for o in f(x, np.ones(300, "float32"), np.ones(300, "float32"), dy)]
    for bad in (1, 3):
        assert np.isnan(y[bad]).all() and np.isnan(dx[bad]).all()
    for r in (0, 2, 4):
        assert np.isfinite(y[r]).all() and np.isfinite(dx[r]).all() and np.isfinite(mean[r]) and np.isfinite(inv[r])
    assert np.isnan(dg).all() and (db == 5).all()


def test_layer_normalization_of_nothing():
    f = ln_function("float32", "float32", 2, 2, 1e-5, True)
    v = np.ones(40, "float32")
    got = [o.to_numpy() for o in f(np.zeros((0, 40), "float32"), v, v, np.zeros((0, 40), "float32"))]
    assert got[0].shape == got[3].shape == (0, 40) and got[1].shape == (0,)
    assert (got[4] == 0).all() and (got[5] == 0).all() and got[4].shape == (40,)
    e = np.ones(0, "float32")
    got = [o.to_numpy() for o in f(np.zeros((3, 0), "float32"), e, e, np.zeros((3, 0), "float32"))]
    assert got[0].shape == (3, 0) and got[4].shape == (0,) and np.isnan(got[1]).all() and np.isnan(got[2]).all()
    x = tensor("float32", 1)
    out, mean, inv = th.function([x], list(T.nnet.layer_normalization(x)))(np.arange(7, dtype="float32"))
    ref = ln_ref(np.arange(7, dtype="float32"), None, None, 1e-5)
    close(out, *ref["y"], chain(7), "vector", "float32")
    assert np.asarray(mean).shape == () and abs(float(mean) - 3) < 1e-6


def layouts(a, rng):
    """Device arrays with the values of ``a`` in other layouts: (name, array)."""
    nd = a.ndim

    def put(base, view_of):
        """A device copy of ``base`` and the view of it that ``view_of`` takes of a host array."""
        d = HipArray.from_numpy(np.ascontiguousarray(base))
        v = view_of(base)
        off = (v.__array_interface__["data"][0] - base.__array_interface__["data"][0])
        return d.view(v.shape, v.strides, d.offset + off)

    def holes(pad, extra):
        base = rng.integers(1, 100, a.shape[:-1] + (a.shape[-1] + pad + extra,)).astype(a.dtype)
        base[..., pad:pad + a.shape[-1]] = a
        return put(base, lambda b: b[..., pad:pad + a.shape[-1]])

    yield "rows apart", holes(0, 7)
    yield "off by one", holes(1, 0)
    yield "off by three, rows apart", holes(3, 6)
    yield "column-major", put(np.ascontiguousarray(a.T), lambda b: b.T)
    if nd == 2:
        yield "rows backwards", put(np.ascontiguousarray(a[::-1]), lambda b: b[::-1])
        base = rng.integers(1, 100, (2 * a.shape[0], a.shape[1])).astype(a.dtype)
        base[::2] = a
        yield "every second row", put(base, lambda b: b[::2])
    if nd == 3:
        yield "axes swapped", put(np.ascontiguousarray(a.swapaxes(0, 1)), lambda b: b.swapaxes(0, 1))


@pytest.mark.parametrize("dtype", ["float16", "float32", "float64"])
def test_layouts_of_the_operands(dtype):
    rng = np.random.default_rng(8)
    for shape in [(6, 500), (40, 129), (3, 4, 260)]:
        x, dy = [rng.standard_normal(shape).astype(dtype) for _ in range(2)]
        gamma, beta = [rng.standard_normal(shape[-1]).astype(dtype) for _ in range(2)]
        for (name, xd), (_, dyd) in zip(layouts(x, rng), reversed(list(layouts(dy, rng)))):
            check_ln(x, gamma, beta, dy, dev={0: xd, 3: dyd}, what="ln " + name)
        wide = HipArray.from_numpy(np.repeat(gamma, 3))
        check_ln(x, gamma, beta, dy, dev={1: wide.view((shape[-1],), (3 * wide.strides[0],))}, what="ln gamma apart")
        lead, acc = shape[:-1], acc_of(dtype)
        tokens = rng.integers(0, shape[-1], lead)
        w, u = [rng.standard_normal(lead).astype(acc) for _ in range(2)]
        c = rng.standard_normal(lead + (4,)).astype(acc)
        for name, xd in layouts(x, rng):
            check_lp(x, tokens, n_top=4, w=w, u=u, c=c, dev={0: xd}, what="lp " + name)
            check_lp(x, tokens, w=w, u=u, dev={0: xd}, what="lp " + name)
        teacher, ids = rng.standard_normal(lead + (5,)).astype("float32"), rng.integers(0, shape[-1], lead + (5,)).astype("int32")
        for (name, xd), (_, td), (_, idd) in zip(layouts(x, rng), reversed(list(layouts(teacher, rng))), layouts(ids, rng)):
            check_kd(x, teacher, ids, g=w, dev={0: xd, 1: td, 2: idd}, what="kd " + name)


def test_one_row_for_all():
    """A row that is broadcast over the batch (a stride of 0) is read as it lies."""
    rng = np.random.default_rng(9)
    row = rng.standard_normal(700).astype("float32")
    x = np.repeat(row[None], 5, axis=0)
    d = HipArray.from_numpy(row).view((5, 700), (0, 4))
    dy = rng.standard_normal(x.shape).astype("float32")
    check_ln(x, row, row, dy, dev={0: d})
    check_lp(x, np.arange(5), n_top=3, w=dy[:, 0].copy(), dev={0: d})
    check_kd(x, dy[:, :6].copy(), np.arange(30).reshape(5, 6), g=dy[:, 0].copy(), dev={0: d})


# ---- log probabilities -------------------------------------------------------------------------------------

# held by one block of every size (up to 256 to 20480 vectors of 16 bytes), and beyond
LP_SHAPES = [(3, 9000), (2, 20000), (3, 70000), (2, 150000), (2, 170001), (1, 1), (1, 2), (2, 7), (3, 64), (5, 65), (1, 513), (4, 1000), (2, 3, 257), (300, 100), (17, 4097), (1, 16384),
             (3, 32000), (1, 50257), (2, 131072), (700, 515), (70, 9001)]


@pytest.mark.parametrize("dtype", ["float16", "float32", "float64"])
@pytest.mark.parametrize("shape", LP_SHAPES, ids=str)
def test_token_log_probs(shape, dtype):
    rng = np.random.default_rng(sum(shape))
    lead, V, acc = shape[:-1], shape[-1], acc_of(dtype)
    x = logits(rng, shape, dtype)
    tokens = rng.integers(0, V, lead)
    w, u = [rng.standard_normal(lead).astype(acc) for _ in range(2)]
    check_lp(x, tokens, what="plain")
    check_lp(x, tokens.astype("int32"), temperature=0.7, n_top=1, w=w, what="one")
    k = min(V, 20)
    check_lp(x, tokens, n_top=k, u=u, what="entropy alone")
    check_lp(x, tokens, temperature=2.0, n_top=k, w=w, u=u, c=rng.standard_normal(lead + (k,)).astype(acc), what="all")
    check_lp(x, tokens, temperature=1.5, w=w, u=u, what="both gradients")
    check_lp(x, tokens, n_top=min(V, 64), what="most")


@pytest.mark.parametrize("dtype", ["float16", "float32", "float64"])
def test_ties_go_to_the_lowest_column(dtype):
    rng = np.random.default_rng(11)
    for shape in [(3, 40), (4, 5000), (1, 60000), (600, 700)]:
        k = min(64, shape[1])
        t = np.zeros(shape[:1], "int64")
        check_lp(np.zeros(shape, dtype), t, n_top=k, what="equal")
        check_lp(rng.integers(0, 3, shape).astype(dtype), t, n_top=k, what="three values")
        x = np.sort(logits(rng, shape, dtype), axis=1)
        check_lp(x, t, n_top=k, what="rising")
        check_lp(np.ascontiguousarray(x[:, ::-1]), t, n_top=k, what="falling")
        z = np.where(rng.random(shape) < 0.5, 0.0, -0.0).astype(dtype)
        check_lp(z, t, n_top=k, what="both zeros")
        x = np.full(shape, -INF, dtype)
        x[:, -3:] = 1
        check_lp(x, t + shape[1] - 1, n_top=k, what="three left")


@pytest.mark.parametrize("dtype", ["float16", "float32", "float64"])
def test_masked_logits(dtype):
    rng = np.random.default_rng(12)
    lowest = np.finfo(dtype).min
    for shape in [(9, 50), (9, 3000), (9, 33333)]:
        lead, acc = shape[:1], acc_of(dtype)
        tokens = rng.integers(0, shape[1], lead)
        teacher, ids = rng.standard_normal(lead + (6,)).astype("float32"), rng.integers(0, shape[1], lead + (6,))
        w, u = [rng.standard_normal(lead).astype(acc) for _ in range(2)]
        c = rng.standard_normal(lead + (7,)).astype(acc)
        for mask in (-INF, lowest):
            x = logits(rng, shape, dtype)
            x[rng.random(shape) < 0.6] = mask
            x[1] = mask                               # nothing but masked
            x[2, :] = mask
            x[2, 13] = 0.5                            # one left
            x[3, :] = -INF
            x[3, 7] = lowest                          # the lowest value beside nothing
            x[4, :] = lowest
            x[4, ::3] = -INF
            check_lp(x, tokens, n_top=7, w=w, u=u, c=c, what="%s %s" % (shape, mask))
            check_lp(x, tokens, w=w, u=u, what="%s %s" % (shape, mask))
            check_kd(x, teacher, ids, g=w, temperature=1.5, what="%s %s" % (shape, mask))


@pytest.mark.parametrize("dtype", ["float16", "float32", "float64"])
def test_nan_and_infinity_among_the_logits(dtype):
    rng = np.random.default_rng(13)
    for shape in [(8, 60), (8, 5000)]:
        lead, acc = shape[:1], acc_of(dtype)
        x = logits(rng, shape, dtype)
        x[1, 3] = np.nan
        x[2, 4] = INF
        x[3, :] = -INF
        x[3, 5] = np.nan
        x[4, :] = np.nan
        x[5, 7:9] = INF
        x[6, 0], x[6, 59], x[6, 30] = np.nan, np.nan, INF
        tokens = rng.integers(0, shape[1], lead)
        w, u = [rng.standard_normal(lead).astype(acc) for _ in range(2)]
        check_lp(x, tokens, n_top=9, w=w, u=u, what=str(shape))
        check_lp(x, tokens, w=w, u=u, what=str(shape))
        check_kd(x, rng.standard_normal(lead + (6,)).astype("float32"), rng.integers(0, shape[1], lead + (6,)), g=w,
                 what=str(shape))


def test_tokens_that_are_none_or_beyond_the_last_column():
    rng = np.random.default_rng(14)
    x = logits(rng, (6, 3000), "float32")
    w, u = [rng.standard_normal(6).astype("float32") for _ in range(2)]
    for idt in ("int32", "int64"):
        tokens = np.array([5, -1, 2999, 3000, -100, np.iinfo(idt).max], idt)
        check_lp(x, tokens, n_top=3, w=w, u=u, what=idt)
        check_lp(x, tokens, w=w, u=u, what=idt)
        check_lp(x, tokens, u=u, what=idt + " entropy alone")     # the row's gradient does not go through the token
        ids = np.tile(np.array([5, 7, -1, 9, -3], idt), (6, 1))
        ids[1] = -1
        ids[2, 2] = 3000
        ids[3] = 11                                               # one token, named five times
        ids[4, 3] = np.iinfo(idt).max
        ids[5, :4] = -1
        check_kd(x, rng.standard_normal((6, 5)).astype("float32"), ids, g=w, temperature=0.5, what=idt)


def test_large_logits_keep_their_digits():
    """Rows far from zero: probabilities depend on differences alone."""
    rng = np.random.default_rng(15)
    for dtype, at in (("float16", 5000.0), ("float32", 1e4), ("float32", -3e38), ("float64", 1e9)):
        x = (at + 8 * rng.standard_normal((4, 2000))).astype(dtype)
        w, u = [rng.standard_normal(4).astype(acc_of(dtype)) for _ in range(2)]
        check_lp(x, rng.integers(0, 2000, 4), n_top=5, w=w, u=u, what="%s %g" % (dtype, at))
        check_lp(x, rng.integers(0, 2000, 4), w=w, u=u, what="%s %g" % (dtype, at))
        check_kd(x, rng.standard_normal((4, 6)).astype("float32"), rng.integers(0, 2000, (4, 6)), g=w, what="%s %g" % (dtype, at))
    x = logits(rng, (3, 700), "float16")
    for t in (1e-3, 50.0):
        check_lp(x, rng.integers(0, 700, 3), n_top=5, temperature=t, w=np.ones(3, "float32"), what="temperature %g" % t)


def beside_largest(x):
    """The differences to the largest of each row, in float64."""
    x = x.astype("float64")
    m = x.max(-1, keepdims=True)
    return x - np.where(np.isfinite(m), m, 0.0)


@pytest.mark.parametrize("temperature", [1e-6, 1e-5, 1e-4, 5.6e-3, 5.7e-3])
@pytest.mark.parametrize("dtype", ["float16", "float32", "float64"])
def test_large_logits_at_low_temperatures(dtype, temperature):
    """The largest logit's probability is no smaller than 1 / columns, however large logit / temperature is.  Gradients
    are weighted so that the results are of order 1.

    Of exponentials below the smallest normal number (2^-126; 2^-1022) the device's single precision gives 0 and the double
    precision fewer digits, so a probability may be off by that number, and the gradient by that times what p is multiplied
    with, (w + sum c + u (ln p + H)) / temperature: weights over temperature of at most 5 each, 5 + 5 * 5 of them, ln p
    down to -89 (-709), H up to ln 20001 < 10.  Distillation: g * temperature, at most 5, times p and q."""
    rng = np.random.default_rng(16)
    acc, lowest = acc_of(dtype), float(np.finfo("float16").min)
    tiny = float(np.finfo(acc).tiny)
    flush = tiny * (5 + 5 * 5 + 5 * (-np.log(tiny) + 10))
    for V in (700, 20001):
        x = np.full((10, V), 10.0)
        x[0, :2] = 8000, 7000
        x[1] = 65504 - 32 * rng.integers(0, 100, V)
        x[2] = lowest
        x[3] = lowest
        x[3, ::3] = -INF
        x[4] = -lowest
        x[5] = temperature * 3 * rng.standard_normal(V)         # probabilities of many columns
        x[6] = 3 * rng.standard_normal(V)
        x[7] = lowest
        x[7, 5:9] = -8000
        x[8, [3, 600, V - 1]] = 30000, 30000, 60000
        x[9] = 10000
        x[9, 1::2] = 9992
        x = x.astype(dtype)
        tokens = rng.integers(0, V, 10)
        tokens[[0, 5]] = 0, V - 1
        w, u = [(temperature * rng.standard_normal(10)).astype(acc) for _ in range(2)]
        c = (temperature * rng.standard_normal((10, 5))).astype(acc)
        what = "%d columns" % V
        # logits / temperature would carry a rounding of its own size; of the differences here the plain forms get all digits
        far = beside_largest(x)
        ref = lp_ref(far, tokens, temperature, 5, w, u, c)
        check_lp_call(x, tokens, temperature, 5, (True,) * 3, [w, u, c], None, ref, False, what, flush)
        ref = lp_ref(far, tokens, temperature, w=w, u=u)
        for fuse in (True, False):
            check_lp_call(x, tokens, temperature, 0, (True, True, False), [w, u], None, ref, fuse, what, flush)
        teacher, ids = x[:, :6].copy(), rng.integers(0, V, (10, 6))
        ids[:, 0] = np.argmax(x, axis=1)
        g = (rng.standard_normal(10) / temperature).astype(acc)
        ref = kd_ref(far, beside_largest(teacher), ids, temperature, g)
        for fuse in (True, False):
            check_kd_call(x, teacher, ids, temperature, g, None, ref, fuse, what, 10 * tiny)


def test_no_rows():
    for dtype in ("float16", "float64"):
        acc = acc_of(dtype)
        z = np.zeros((0,), acc)
        check_lp(np.zeros((0, 50), dtype), np.zeros((0,), "int64"), n_top=3, w=z, u=z, c=np.zeros((0, 3), acc))
        check_lp(np.zeros((0, 50), dtype), np.zeros((0,), "int64"), w=z, u=z)
        check_kd(np.zeros((0, 50), dtype), np.zeros((0, 4), "float32"), np.zeros((0, 4), "int64"), g=z)


# ---- distillation ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,tdt,idt", [("float16", "float16", "int32"), ("float16", "float32", "int64"),
                                           ("float32", "float32", "int32"), ("float32", "float64", "int64"),
                                           ("float64", "float64", "int64"), ("float64", "float16", "int32")])
@pytest.mark.parametrize("shape,k", [((1, 1), 1), ((1, 2), 3), ((5, 64), 8), ((3, 1000), 1), ((2, 3, 515), 17), ((300, 100), 5),
                                     ((9, 32000), 64), ((1, 50257), 100), ((2, 131072), 300), ((3, 4099), 1024)], ids=str)
def test_topk_distillation(shape, k, dtype, tdt, idt):
    rng = np.random.default_rng(sum(shape) + k)
    lead, V = shape[:-1], shape[-1]
    x = logits(rng, shape, dtype)
    teacher = (2 * rng.standard_normal(lead + (k,))).astype(tdt)
    ids = rng.integers(0, V, lead + (k,)).astype(idt)
    ids[..., k // 2:][rng.random(ids[..., k // 2:].shape) < 0.2] = -1
    g = rng.standard_normal(lead).astype(acc_of(dtype))
    check_kd(x, teacher, ids, temperature=2.0, g=g, what="hot")
    teacher.reshape(-1)[::5] = -INF
    check_kd(x, teacher, ids, what="forward, some masked")
    check_kd(x, teacher, ids, g=g, what="some masked")


@pytest.mark.parametrize("vectors", [256, 512, 1024, 2048, 4096, 8192, 10240, 16384, 20480])
@pytest.mark.parametrize("dtype", ["float16", "float32", "float64"])
def test_rows_as_long_as_a_block_holds(dtype, vectors):
    """A loss with its gradient in one launch keeps a row in a block's registers: the last row that a block of each size
    holds, and the first that it does not."""
    rng = np.random.default_rng(vectors)
    width = 16 // np.dtype(dtype).itemsize
    for cols in (vectors * width, vectors * width + width):
        x = logits(rng, (2, cols), dtype)
        tokens = np.array([cols - 1, 0])
        w, u = [rng.standard_normal(2).astype(acc_of(dtype)) for _ in range(2)]
        check_lp(x, tokens, w=w, u=u, what=str(cols))
        ids = rng.integers(0, cols, (2, 70))
        ids[:, :4] = cols - 1, 0, cols - 1, cols - 2
        ids[0, 69] = 0
        check_kd(x, rng.standard_normal((2, 70)).astype("float32"), ids, g=w, temperature=1.5, what=str(cols))


@pytest.mark.parametrize("entries", [3, 4, 5, 255, 256, 257, 1024])
def test_entries_that_name_the_same_columns(entries):
    """Many entries to a column, at both ends of the list and of a block's turns through it."""
    rng = np.random.default_rng(entries)
    for dtype, cols in (("float16", 40), ("float32", 2100), ("float16", 33000)):
        ids = rng.integers(0, 6, (3, entries)).astype("int32")      # six columns share the entries
        ids[1] = cols - 1
        ids[2, 1:-1] = -1
        ids[2, -1] = ids[2, 0]
        check_kd(logits(rng, (3, cols), dtype), rng.standard_normal((3, entries)).astype("float16"), ids,
                 g=rng.standard_normal(3).astype("float32"), what="%s %d" % (dtype, cols))


# ---- gradients against differences, and the operators together ---------------------------------------------

@pytest.mark.parametrize("pdtype", [None, "float16", "float32"])
@pytest.mark.parametrize("stats", [(True, False), (False, True), (True, True)])
def test_gradients_through_statistics_are_rounded_once(pdtype, stats):
    """dx of float16 rows is the sum of what arrives through the result and through the statistics, rounded once: half a
    step of the sum, whatever the size of its parts."""
    rng = np.random.default_rng(31)
    shape = (60, 333)
    x, dy = [rng.standard_normal(shape).astype("float16") for _ in range(2)]
    gamma, beta = [rng.standard_normal(333).astype(pdtype or "float16") for _ in range(2)]
    # of the size of dx in each element, so that parts cancel
    dmean, dinv = [(333 * rng.standard_normal(60) * there).astype("float32") for there in stats]
    xt, dyt, mt, it = tensor("float16", 2), tensor("float16", 2), T.fvector(), T.fvector()
    ps = [tensor(pdtype, 1) for _ in range(2)] if pdtype else []
    y, mean, inv = T.nnet.layer_normalization(xt, *ps)
    known = {y: dyt}
    known.update((v, g) for v, g, there in ((mean, mt, stats[0]), (inv, it, stats[1])) if there)
    f = th.function([xt, dyt, mt, it] + ps, th.grad(None, [xt] + ps, known_grads=known), on_unused_input="ignore")
    got = f(x, dy, dmean, dinv, *([gamma, beta] if pdtype else []))
    ref = ln_ref(x, gamma if pdtype else None, beta if pdtype else None, 1e-5, dy)
    m, i = ref["mean"][0][:, None], ref["invstd"][0][:, None]
    parts = [dmean[:, None] / 333.0, -dinv[:, None] * i ** 3 / 333.0 * (x.astype("float64") - m)]
    value = ref["dx"][0] + parts[0] + parts[1]
    # x - mean is off by roundings of the largest |x|, and of invstd the cube is taken
    big = np.abs(x.astype("float64")).max(-1, keepdims=True)
    scale = ref["dx"][1] + np.abs(parts[0]) + 4 * np.abs(dinv[:, None]) * (ref["invstd"][1][:, None]) ** 3 / 333.0 * 2 * big
    close(got[0], value, scale, chain(333), "dx", "float32")
    if pdtype:
        for g, name in zip(got[1:], ("dgamma", "dbeta")):
            assert str(g.dtype) == pdtype
            close(g, *ref[name], chain(333, 60), name, "float32")


def differences(f, args, k, h):
    """Central differences of the scalar function ``f`` with respect to its argument ``k``."""
    out = np.zeros(args[k].shape)
    for i in np.ndindex(*args[k].shape):
        vals = []
        for s in (h, -h):
            moved = [a.copy() for a in args]
            moved[k][i] += s
            vals.append(float(f(*moved)))
        out[i] = (vals[0] - vals[1]) / (2 * h)
    return out


def test_gradients_are_those_of_differences():
    """In float64 with a step of 1e-6: the second-order term and the rounding of the cost are both far below 1e-7 of
    gradients of order 1."""
    rng = np.random.default_rng(21)
    x, gamma, beta, t, z = T.dmatrix(), T.dvector(), T.dvector(), T.lvector(), T.dmatrix()
    ids, teacher = T.lmatrix(), T.dmatrix()
    a, m, i = T.nnet.layer_normalization(x, gamma, beta)
    vals = [rng.standard_normal((3, 5)), 1 + rng.standard_normal(5), rng.standard_normal(5), rng.standard_normal((3, 5))]
    for cost in (T.sum(T.sqr(a) * z) / 2 + T.sum(a * z), T.sum(a * z) + T.sum(T.sqr(m)) + T.sum(i * z[:, 0]),
                 T.sum(m * z[:, 1]), T.sum(T.sqr(i))):
        ins = [x, gamma, beta, z]
        f = th.function(ins, cost, on_unused_input="ignore")
        gs = th.function(ins, th.grad(cost, [x, gamma, beta], disconnected_inputs="ignore"), on_unused_input="ignore")(*vals)
        for k, g in enumerate(gs):
            np.testing.assert_allclose(g, differences(f, vals, k, 1e-6), rtol=1e-6, atol=1e-7)
    lp, h, tv, ti = T.nnet.token_log_probs(x, t, n_top=3, temperature=0.8)
    kd = T.nnet.topk_distillation_loss(x, teacher, ids, temperature=1.7)
    vals = [rng.standard_normal((4, 9)), np.array([1, 8, -1, 3]), rng.integers(0, 9, (4, 3)), rng.standard_normal((4, 3))]
    for cost in (T.sum(T.exp(lp) * h) + T.sum(T.sqr(tv) * teacher), T.sum(T.sqr(h)), T.sum(T.sqr(kd) + lp * kd)):
        ins = [x, t, ids, teacher]
        f = th.function(ins, cost, on_unused_input="ignore")
        g = th.function(ins, th.grad(cost, x), on_unused_input="ignore")(*vals)
        np.testing.assert_allclose(g, differences(f, vals, 0, 1e-6), rtol=1e-6, atol=1e-7)


def test_one_weight_for_all_rows():
    """The weight of a mean is read as one value, in one launch and in two."""
    rng = np.random.default_rng(28)
    x, t, teacher, ids = tensor("float16", 2), T.lvector(), T.fmatrix(), T.imatrix()
    lp, h = T.nnet.token_log_probs(x, t)
    kd = T.nnet.topk_distillation_loss(x, teacher, ids)
    cost = T.mean(np.float32(64) * kd) - T.mean(lp)
    vals = [logits(rng, (11, 777), "float16"), rng.integers(0, 777, 11), rng.standard_normal((11, 5)).astype("float32"),
            rng.integers(0, 777, (11, 5)).astype("int32")]
    one = np.ones(11)
    a, b = lp_ref(vals[0], vals[1], w=-one / 11), kd_ref(vals[0], vals[2], vals[3], g=64 * one / 11)
    for fuse in (True, False):
        got = th.function([x, t, teacher, ids], th.grad(cost, x), fuse=fuse)(*vals)
        # each gradient is rounded to float16, then their sum
        off = 2.0 ** -11 * (np.abs(a["dx"][0]) + np.abs(b["dx"][0])) + 2 * 2.0 ** -25
        close(got, a["dx"][0] + b["dx"][0], a["dx"][1] + b["dx"][1] + off / (chain(777) * 2.0 ** -24), chain(777), "dx", "float32")


def test_two_results_that_are_each_others_gradients():
    rng = np.random.default_rng(30)
    a, b = T.fmatrix(), T.fmatrix()
    ya, yb = T.nnet.layer_normalization(a)[0], T.nnet.layer_normalization(b)[0]
    va, vb = [rng.standard_normal((5, 70)).astype("float32") for _ in range(2)]
    f = th.function([a, b], [th.grad(None, a, known_grads={ya: yb}), th.grad(None, b, known_grads={yb: ya})])
    got = f(va, vb)
    la, lb = [ln_ref(v, None, None, 1e-5)["y"][0].astype("float32") for v in (va, vb)]
    for g, v, dy in zip(got, (va, vb), (lb, la)):
        # dy is a result itself, off by the same number of roundings of its own scale m (|xhat| + largest |x| * invstd, 2 to
        # 7 here), where dx counts its value: (m + mean(m) + m mean(m^2)) / (mean|dy| + 2 m mean(|dy| m)) is below 4
        value, scale = ln_ref(v, None, None, 1e-5, dy)["dx"]
        close(g, value, scale, 5 * chain(70), "dx", "float32")


def test_second_derivatives_of_layer_normalization():
    rng = np.random.default_rng(22)
    x, gamma, beta, z = T.dmatrix(), T.dvector(), T.dvector(), T.dmatrix()
    y = T.nnet.layer_normalization(x, gamma, beta)[0]
    dx, dg, db = th.grad(T.sum(T.sqr(y) * z), [x, gamma, beta])
    cost = T.sum(dx * z) + T.sum(T.sqr(dg)) + T.sum(dg * db)
    vals = [rng.standard_normal((3, 4)), 1 + rng.standard_normal(4), rng.standard_normal(4), rng.standard_normal((3, 4))]
    f = th.function([x, gamma, beta, z], cost)
    gs = th.function([x, gamma, beta, z], th.grad(cost, [x, gamma, beta]))(*vals)
    for k, g in enumerate(gs):
        ref = differences(f, vals, k, 1e-6)
        np.testing.assert_allclose(g, ref, rtol=1e-5, atol=1e-6 * (1 + np.abs(ref).max()))


def head_graph():
    """The end of a model: normalised activations as logits, a policy loss on the given tokens with an entropy bonus,
    and distillation from a teacher, on the same logits."""
    h, gamma, beta = tensor("float16", 3, "h"), tensor("float32", 1, "gamma"), tensor("float32", 1, "beta")
    t, adv = T.TensorType("int64", (False, False))("t"), tensor("float32", 2, "adv")
    teacher, ids = tensor("float16", 3, "teacher"), T.TensorType("int32", (False,) * 3)("ids")
    y = T.nnet.layer_normalization(h, gamma, beta)[0]
    lp, ent, tv, ti = T.nnet.token_log_probs(y, t, n_top=4, temperature=0.9)
    kd = T.nnet.topk_distillation_loss(y, teacher, ids, temperature=2.0)
    cost = T.sum(-adv * lp - np.float32(0.01) * ent + np.float32(0.5) * kd)
    return [h, gamma, beta, t, adv, teacher, ids], [cost, lp, ent, ti] + th.grad(cost, [h, gamma, beta]), y, lp


def head_values(rng, lead=(2, 37), V=1111, k=9):
    return [rng.standard_normal(lead + (V,)).astype("float16"), (1 + 0.1 * rng.standard_normal(V)).astype("float32"),
            rng.standard_normal(V).astype("float32"), rng.integers(-1, V, lead), rng.standard_normal(lead).astype("float32"),
            rng.standard_normal(lead + (k,)).astype("float16"), rng.integers(-1, V, lead + (k,)).astype("int32")]


def test_the_operators_together_as_a_training_step():
    rng = np.random.default_rng(23)
    ins, outs, y, lp = head_graph()
    f = th.function(ins, outs + [y])
    vals = head_values(rng)
    cost, lp, ent, ti, dh, dg, db, yv = f(*vals)
    h, gamma, beta, t, adv, teacher, ids = vals
    # the operators' own logits go into the plain forms, so that a rounding of theirs is not counted again
    one = np.ones(t.shape)
    lpr, kdr = lp_ref(yv, t, 0.9, 4, w=-adv, u=-0.01 * one), kd_ref(yv, teacher, ids, 2.0, g=0.5 * one)
    close(lp, *lpr["log_prob"], chain(1111), "log_prob", "float32")
    close(ent, *lpr["entropy"], chain(1111), "entropy", "float32")
    np.testing.assert_array_equal(ti, lpr["top_at"])
    total = -adv * lpr["log_prob"][0] - 0.01 * lpr["entropy"][0] + 0.5 * kdr["loss"][0]
    size = np.abs(adv) * lpr["log_prob"][1] + 0.01 * lpr["entropy"][1] + 0.5 * kdr["loss"][1]
    close(np.asarray(cost), np.asarray(total.sum()), size.sum(), chain(1111, t.size), "cost", "float32")
    # dy is rounded to float16 three times (each operator's gradient, and their sum): three half steps of its parts
    dy = lpr["dx"][0] + kdr["dx"][0]
    off = 3 * 2.0 ** -11 * (np.abs(lpr["dx"][0]) + np.abs(kdr["dx"][0])) + 3 * 2.0 ** -25
    ref = ln_ref(h, gamma, beta, 1e-5, dy)
    xhat = np.abs((ref["y"][0] - beta) / gamma)
    inv = ref["invstd"][0][..., None]
    a = off * np.abs(gamma)
    slack = inv * (a + a.mean(-1, keepdims=True) + xhat * (a * xhat).mean(-1, keepdims=True))
    lead = (0, 1)
    for got, name, more in ((dh, "dx", slack), (dg, "dgamma", (off * xhat).sum(lead)), (db, "dbeta", off.sum(lead))):
        value, scale = ref[name]
        u = 2.0 ** -24
        close(got, value, scale + more / (chain(1111, t.size) * u), chain(1111, t.size), name, "float32")


def test_modes_and_shared_updates():
    """The same step with the arguments' contents and rewrites checked, and as an update of shared parameters."""
    rng = np.random.default_rng(24)
    ins, outs, y, lp = head_graph()
    vals = head_values(rng)
    plain = th.function(ins, outs)(*vals)
    for mode in ("check", "nan_guard"):
        got = th.function(ins, outs, mode=mode)(*vals)
        for a, b in zip(plain, got):
            np.testing.assert_array_equal(a, b)
    w = th.shared(vals[1])
    x = tensor("float16", 3)
    yy = T.nnet.layer_normalization(x, w)[0]
    c = T.sum(T.cast(yy, "float32"))
    step = th.function([x], c, updates=[(w, w - np.float32(0.5) * th.grad(c, w))])
    step(vals[0])
    ref = ln_ref(vals[0], vals[1], None, 1e-5, np.ones_like(vals[0]))
    close(w.get_value(), vals[1] - 0.5 * ref["dgamma"][0], np.abs(vals[1]) + ref["dgamma"][1], chain(1111, 74), "update", "float32")


def test_recorded_and_replayed():
    """Two recordings that are alive together, each replayed with other contents and eager work between."""
    rng = np.random.default_rng(25)
    ins, outs, y, lp = head_graph()
    dev = [Out(o, device=True) for o in outs]
    f, eager = th.function(ins, dev), th.function(ins, dev)
    sizes = [dict(lead=(2, 37), V=1111, k=9), dict(lead=(1, 3), V=40000, k=70)]
    graphs = []
    for kw in sizes:
        args = [HipArray.from_numpy(v) for v in head_values(rng, **kw)]
        graphs.append((args, kw) + f.capture(*args))
    for replay in range(4):
        for args, kw, results, graph in graphs:
            for a, v in zip(args, head_values(rng, **kw)):
                copy_into(HipArray.from_numpy(v), a)
            eager(*[HipArray.from_numpy(v) for v in head_values(rng)])
        for args, kw, results, graph in graphs:
            graph.launch()
        for args, kw, results, graph in graphs:
            want = [w.to_numpy() for w in eager(*args)]
            for g, w in zip(results, want):
                np.testing.assert_array_equal(g.to_numpy(), w)


def test_the_same_call_gives_the_same_bits():
    rng = np.random.default_rng(26)
    for shape in [(1, 50257), (3000, 700)]:
        x = HipArray.from_numpy(logits(rng, shape, "float16"))
        t = HipArray.from_numpy(rng.integers(0, shape[1], shape[:1]))
        w = HipArray.from_numpy(rng.standard_normal(shape[:1]).astype("float32"))
        f = lp_function("float16", "int64", 2, 20, 1.0, (True, True, False))
        first = [o.to_numpy() for o in f(x, t, w, w)]
        for _ in range(3):
            for a, b in zip(first, f(x, t, w, w)):
                np.testing.assert_array_equal(a, b.to_numpy())


def test_offsets_past_32_bits():
    """More than 2^31 elements, and rows further apart than 2^31: the rows at both ends and on both sides of the border,
    the others holding whatever the memory held."""
    rng = np.random.default_rng(29)

    def rows_of(a, ids):
        return np.stack([HipArray(a.buffer, a.offset + r * a.strides[0], a.shape[1:], a.strides[1:], a.dtype).to_numpy()
                         for r in ids])

    def put(a, ids, values):
        for r, v in zip(ids, values):
            copy_into(HipArray.from_numpy(v), HipArray(a.buffer, a.offset + r * a.strides[0], a.shape[1:], a.strides[1:], a.dtype))

    def compare(got, ref, ids, names, n):
        for g, name in zip(got, names):
            v = rows_of(g, ids)
            if name == "top_at":
                np.testing.assert_array_equal(v, ref[name])
            elif name in ref:
                close(v, *ref[name], n, name, "float32")

    big = HipArray.empty(((1 << 31) + 40 * 131073,), "float16")
    for V in (131073, 999):
        rows = big.size // V if V > 1000 else 3
        step = V if V > 1000 else (big.size - V) // 2 // 8 * 8 - 5      # 999: three rows a thousand million apart
        x = HipArray(big.buffer, 0, (rows, V), (2 * step, 2), "float16")
        ids = sorted(set([0, 1, (1 << 31) // step - 1, (1 << 31) // step, rows - 2, rows - 1]) & set(range(rows)))
        v = logits(rng, (len(ids), V), "float16")
        put(x, ids, v)
        tokens = rng.integers(0, V, rows)
        w, u = [rng.standard_normal(rows).astype("float32") for _ in range(2)]
        ref = lp_ref(v, tokens[ids], w=w[ids], u=u[ids])
        for fuse in (True, False):
            got = lp_function("float16", "int64", 2, 0, 1.0, (True, True, False), fuse)(x, tokens, w, u)
            compare(got, ref, ids, ["log_prob", "entropy", "dx"], chain(V))
            del got
        got = lp_function("float16", "int64", 2, 5, 1.0, (False,) * 3)(x, tokens)
        compare(got, lp_ref(v, tokens[ids], n_top=5), ids, ["log_prob", "entropy", "top", "top_at"], chain(V))
        teacher, at = rng.standard_normal((rows, 3)).astype("float32"), rng.integers(0, V, (rows, 3))
        ref = kd_ref(v, teacher[ids], at[ids], g=w[ids])
        for fuse in (True, False):
            got = kd_function("float16", "float32", "int64", 2, 1.0, True, fuse)(x, teacher, at, w)
            compare(got, ref, ids, ["loss", "dx"], chain(V) + 3)
            del got
    for V in (4097, 70000):          # rows in registers, and the kernels for any row
        rows = big.size // V
        x = HipArray(big.buffer, 0, (rows, V), (2 * V, 2), "float16")
        ids = [0, 1, (1 << 31) // V - 1, (1 << 31) // V, rows - 1]
        v = rng.standard_normal((len(ids), V)).astype("float16")
        put(x, ids, v)
        gamma, beta = [rng.standard_normal(V).astype("float32") for _ in range(2)]
        ref = ln_ref(v, gamma, beta, 1e-5, v)
        for fuse in (True, False):
            got = ln_function("float16", "float32", 2, 2, 1e-5, True, fuse)(x, gamma, beta, x)
            compare(got, ref, ids, ["y", "mean", "invstd", "dx"], chain(V))
            del got


# ---- arrays of other libraries -----------------------------------------------------------------------------

def test_views_of_and_for_other_libraries():
    class Other(object):
        """What another library's array shows of itself."""
        def __init__(self, a):
            self.a = a
            self.__cuda_array_interface__ = dict(a.__cuda_array_interface__)

    rng = np.random.default_rng(27)
    v = rng.standard_normal((6, 40)).astype("float32")
    a = HipArray.from_numpy(v)
    d = a.__cuda_array_interface__
    assert d["shape"] == (6, 40) and d["typestr"] == "<f4" and d["strides"] == (160, 4) and d["data"] == (a.ptr, False)
    assert d["stream"] == hip.stream() and d["stream"]
    b = HipArray.from_cuda_array_interface(Other(a))
    assert b.ptr == a.ptr and b.shape == a.shape and b.strides == a.strides and b.dtype == a.dtype
    t = HipArray.from_cuda_array_interface(Other(a.transpose()))
    np.testing.assert_array_equal(t.to_numpy(), v.T)
    x = T.fmatrix()
    np.testing.assert_allclose(th.function([x], x * 2)(b), v * 2)
    host = Other(a)
    host.__cuda_array_interface__["data"] = (v.ctypes.data, False)
    with pytest.raises(ValueError, match="not device memory"):
        HipArray.from_cuda_array_interface(host)
    wrong = Other(a)
    wrong.__cuda_array_interface__["typestr"] = "<U4"
    with pytest.raises(TypeError):
        HipArray.from_cuda_array_interface(wrong)
    empty = HipArray.from_cuda_array_interface(Other(HipArray.empty((0, 3), "float16")))
    assert empty.shape == (0, 3)
