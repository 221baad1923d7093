"""The training operators (layer norm, token log probabilities, gradient
norm and clipping) against plain 64-bit implementations of their formulas,
at the sizes, strides and masks where they can go wrong.

Tolerances: u is the rounding of the result's type (half a step of its 24, 11 and 8
bits: 2^-24, 2^-11, 2^-8), e = 2^-24 that of the f32 arithmetic.  Each is a bound on the formula's own
rounding, stated where it is used."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import oracle as O
from tensorcrate_b200 import _native as N
from tensorcrate_b200 import nn
from tensorcrate_b200.cuda import CudaStorage, Tensor, TensorView, f32_to_bits
from util import DTYPES, normal

pytestmark = pytest.mark.gpu

U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}  # the smallest values: below them all is rounded off
e = 2.0 ** -24


def put(values, dtype):
    return CudaStorage.store(f32_to_bits(np.asarray(values, np.float32).ravel(), dtype), dtype)


def tensor(values, dtype="f32"):
    return Tensor(put(values, dtype), np.shape(values))


def as_type(values, dtype):
    """The values that `dtype` holds of them, in f64."""
    return O.widen(f32_to_bits(np.asarray(values, np.float32), dtype), dtype).astype(np.float64)


def matrix(values, dtype, pad=0, offset=0):
    """A view of `values` whose rows are cols + pad elements apart, `offset`
    elements into its storage; what lies between is NaN."""
    rows, cols = values.shape
    whole = np.full(offset + rows * (cols + pad), np.nan, np.float32)
    for r in range(rows):
        at = offset + r * (cols + pad)
        whole[at:at + cols] = values[r]
    return TensorView(put(whole, dtype), [rows, cols], [cols + pad, 1], offset)


def blank(rows, cols, dtype, pad=0, offset=0):
    return matrix(np.full((rows, cols), 7.0, np.float32), dtype, pad, offset)


def read(view):
    """A view's values in f64, and whether what lies between its rows is
    still NaN."""
    flat = O.widen(view.storage.as_slice(), view.dtype).astype(np.float64)
    rows, cols = view.shape
    keep = np.ones(flat.size, bool)
    out = np.empty((rows, cols))
    for r in range(rows):
        at = view.offset + r * view.strides[0]
        out[r] = flat[at:at + cols]
        keep[at:at + cols] = False
    return out, bool(np.all(np.isnan(flat[keep])))


def within(got, want, tol):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        bad = ~same & ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), got[bad][:4], want[bad][:4], np.broadcast_to(tol, got.shape)[bad][:4])


# ---------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------
def norm64(x, w, b, eps):
    mean = x.mean(1, keepdims=True)
    rstd = 1.0 / np.sqrt(((x - mean) ** 2).mean(1, keepdims=True) + eps)
    h = (x - mean) * rstd
    return h * w + b, mean, rstd, h


def norm_grad64(g, x, w, mean, rstd):
    h = (x - mean) * rstd
    gw = g * w
    dx = rstd * (gw - gw.mean(1, keepdims=True) - h * (gw * h).mean(1, keepdims=True))
    return dx, (g * h).sum(0), g.sum(0), h, gw


NORM_SHAPES = [(1, 1, 0, 0), (1, 7, 0, 0), (3, 8, 0, 0), (5, 100, 3, 1), (70, 256, 0, 0), (4, 1001, 0, 0), (9, 1024, 0, 0),
               (7, 1032, 8, 8), (130, 1536, 0, 0), (2, 4096, 0, 0), (33, 4099, 0, 0), (3, 5000, 5, 0), (3, 8200, 0, 0),
               (2, 16384, 0, 0), (3, 16392, 8, 0), (5, 9001, 0, 0), (90, 16408, 0, 0), (50, 20003, 0, 1), (2, 33001, 0, 3), (1, 70000, 0, 0)]


@pytest.mark.parametrize("params", ["same", "f32", "none"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols,pad,offset", NORM_SHAPES)
def test_layer_norm_and_its_gradients(device, rows, cols, pad, offset, dtype, params):
    eps = 1e-5
    kind = dtype if params == "same" else "f32"
    x = as_type(normal((rows, cols), 1) * 2 + 0.5, dtype)
    g = as_type(normal((rows, cols), 2), dtype)
    w, b = (as_type(1 + 0.3 * normal(cols, 3), kind), as_type(normal(cols, 4), kind)) if params != "none" else (1.0, 0.0)
    W, B = (tensor(w, kind), tensor(b, kind)) if params != "none" else (None, None)
    X, Y = matrix(x, dtype, pad, offset), blank(rows, cols, dtype, pad, offset)
    y, st = nn.layer_norm(X, W, B, eps, out=Y)
    want, mean, rstd, h = norm64(x, w, b, eps)
    got, kept = read(Y)
    # mean: the sum's rounding, at most 24 levels and terms deep, e |x| each;
    # its error and that of x - mean enter h times rstd
    off = 32 * e * (np.abs(x).mean(1, keepdims=True) + np.abs(mean) + np.abs(x - mean))
    within(got, want, U[dtype] * np.abs(want) + TINY[dtype] + (off * rstd + 40 * e * np.abs(h)) * np.abs(w) + 4 * e * np.abs(b))
    assert kept and y is Y
    s = st.to_f32().astype(np.float64)
    within(s[:, :1], mean, off.max(1, keepdims=True))
    if cols > 1:  # a single element's variance is eps alone
        within(s[:, 1:], rstd, rstd * (40 * e + 2 * off.max(1, keepdims=True) * rstd))
    # the gradients, from the statistics as the forward pass left them
    mean, rstd = s[:, :1], s[:, 1:]
    G, D = matrix(g, dtype, pad, offset), blank(rows, cols, dtype, pad, offset)
    _, dw, db = nn.layer_norm_backward(G, X, st, W, out=D)
    want, want_w, want_b, h, gw = norm_grad64(g, x, w, mean, rstd)
    got, kept = read(D)
    # the two means' sums: 32 terms and levels deep at most, e of the terms' magnitudes
    deep = 48 * e * rstd * (np.abs(gw) + np.abs(gw).mean(1, keepdims=True) + np.abs(h) * np.abs(gw * h).mean(1, keepdims=True))
    near = 4 * e * rstd * np.abs(mean) * rstd * (np.abs(gw * h).mean(1, keepdims=True) + np.abs(gw).mean(1, keepdims=True) * np.abs(h))
    within(got, want, U[dtype] * np.abs(want) + TINY[dtype] + deep + near)
    assert kept
    # sums over the rows: at most 128 additions deep
    assert dw.dtype == db.dtype == (kind if params != "none" else dtype)
    kind = dw.dtype
    within(dw.to_f32(), want_w, U[kind] * np.abs(want_w) + TINY[kind] + 128 * e * (np.abs(g * h) + np.abs(g * mean * rstd)).sum(0))
    within(db.to_f32(), want_b, U[kind] * np.abs(want_b) + TINY[kind] + 128 * e * np.abs(g).sum(0))


def test_layer_norm_gradients_agree_with_differences(device):
    """The kernels' f32 gradients of sum(c y) against central differences of
    the definition in 64 bits (error h^2 with h = 1e-5, far below the f32
    rounding's 1e-5 of the largest)."""
    rng = np.random.default_rng(0)
    rows, cols, eps, h = 5, 37, 1e-3, 1e-5
    x, c = as_type(rng.standard_normal((rows, cols)), "f32"), as_type(rng.standard_normal((rows, cols)), "f32")
    w, b = as_type(rng.standard_normal(cols), "f32"), as_type(rng.standard_normal(cols), "f32")
    X = tensor(x)
    _, st = nn.layer_norm(X, tensor(w), tensor(b), eps)
    got = [t.to_f32() for t in nn.layer_norm_backward(tensor(c), X, st, tensor(w))]

    def loss(x, w, b):
        return (c * norm64(x, w, b, eps)[0]).sum()

    for k, at in enumerate([x, w, b]):
        want = np.empty(at.shape)
        for i in np.ndindex(at.shape):
            two = []
            for s in (h, -h):
                v = [x, w, b]
                v[k] = at.copy()
                v[k][i] += s
                two.append(loss(*v))
            want[i] = (two[0] - two[1]) / (2 * h)
        within(got[k], want, 1e-5 * np.abs(want).max())


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_in_place_and_repeated(device, dtype):
    """y over x, grad_x over grad or over x: the same bits as into buffers of
    their own; and the same bits on every call (the sums' order is fixed)."""
    for rows, cols in [(300, 96), (64, 2048), (37, 1003), (5, 17000)]:
        x, g = normal((rows, cols), 1), normal((rows, cols), 2)
        w = tensor(normal(cols, 3))
        X, G = tensor(x, dtype), tensor(g, dtype)
        y, st = nn.layer_norm(X, w)
        own = tensor(x, dtype)
        nn.layer_norm(own, w, out=own)
        assert np.array_equal(own.to_numpy(), y.to_numpy())
        first = [t.to_numpy() for t in nn.layer_norm_backward(G, X, st, w)]
        again = [t.to_numpy() for t in nn.layer_norm_backward(G, X, st, w)]
        over_g, over_x = tensor(g, dtype), tensor(x, dtype)
        a = nn.layer_norm_backward(over_g, X, st, w, out=over_g)
        b = nn.layer_norm_backward(G, over_x, st, w, out=over_x)
        for i in range(3):
            assert np.array_equal(first[i], again[i])
            assert np.array_equal(first[i], a[i].to_numpy()) and np.array_equal(first[i], b[i].to_numpy())


def test_layer_norm_of_a_constant_row_and_of_no_rows(device):
    x = np.full((3, 64), 3.0, np.float32)
    y, st = nn.layer_norm(tensor(x), eps=1e-5)
    assert np.all(y.to_f32() == 0.0)
    within(st.to_f32(), [[3.0, 1e-5 ** -0.5]] * 3, 1e-5 ** -0.5 * 4 * e)
    none = Tensor(CudaStorage("f32", 0), [0, 64])
    y, st = nn.layer_norm(none)
    dx, dw, db = nn.layer_norm_backward(none, none, st)
    assert y.to_numpy().shape == (0, 64) and not dw.to_f32().any() and not db.to_f32().any()


def test_layer_norm_only_what_is_asked_for(device):
    """Null outputs are not computed, and the others keep their bits."""
    x, g, w = tensor(normal((40, 600), 1)), tensor(normal((40, 600), 2)), tensor(normal(600, 3))
    _, st = nn.layer_norm(x, w)
    whole = nn.layer_norm_backward(g, x, st, w)
    dx, dw, db = tensor(np.zeros((40, 600))), tensor(np.zeros(600)), tensor(np.zeros(600))
    for o in ((dx, None, None), (None, dw, None), (None, None, db)):
        p = [None if t is None else t.storage.ptr for t in o]
        N.call("tc_layer_norm_backward", N.F32, N.F32, 40, 600, g.storage.ptr, 600, x.storage.ptr, 600, st.storage.ptr,
               w.storage.ptr, p[0], 600, p[1], p[2], None)
    for got, want in zip((dx, dw, db), whole):
        assert np.array_equal(got.to_numpy(), want.to_numpy())


# ---------------------------------------------------------------------------
# token log probabilities
# ---------------------------------------------------------------------------
def tokens64(x, token):
    """(logprob, entropy, max, log sum, log p) by the definitions."""
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        m = np.max(np.where(np.isnan(x), -np.inf, x), 1)
        empty = np.all(x == -np.inf, 1)
        base = np.where(m == -np.inf, 0.0, m)
        d = x - base[:, None]
        s = np.where(empty, 1.0, np.exp(d).sum(1))
        ls = np.log(s)
        a = d - ls[:, None]
        p = np.exp(a)
        ent = -np.where(x == -np.inf, 0.0, p * a).sum(1)
        lp = np.array([0.0 if t == N.NO_TOKEN else a[r, t] if t < x.shape[1] else np.nan for r, t in enumerate(token)])
    ent[empty] = 0.0
    return lp, ent, m, ls, a, p, empty


def slope64(x, token, u, v):
    lp, ent, m, ls, a, p, empty = tokens64(x, token)
    known = np.array([t < x.shape[1] for t in token]) & ~empty
    u = np.where(known, u, 0.0)[:, None]
    one = np.zeros_like(x)
    for r, t in enumerate(token):
        if t < x.shape[1]:
            one[r, t] = 1.0
    with np.errstate(invalid="ignore"):
        grad = u * (one - p) - v[:, None] * np.where(x == -np.inf, 0.0, p * (a + ent[:, None]))
    quiet = (u[:, 0] == 0) & ((v == 0) | empty)
    grad[quiet | empty] = 0.0
    return grad, p, a, ent, u, one


def masked(x, how, dtype, rng):
    if how == "none":
        return x
    low = -np.inf if how == "inf" else {"f32": np.finfo(np.float32).min, "f16": -65504.0,
                                        "bf16": -float(2 ** 128 - 2 ** 120)}[dtype]
    x = np.where(rng.random(x.shape) < 0.7, low, x)
    x[1::5] = low  # rows that are left nothing
    return x


SHAPES = [(1, 1, 0), (5, 2, 0), (7, 33, 0), (6, 100, 3), (40, 513, 0), (6, 1024, 8), (6, 1031, 0), (3, 4096, 0), (6, 5003, 0),
          (3, 50257, 0), (2, 131072, 0), (1, 262144, 0)]


@pytest.mark.parametrize("mask", ["none", "inf", "lowest"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,pad", SHAPES)
def test_token_logprobs_and_their_gradients(device, rows, vocab, pad, dtype, mask):
    rng = np.random.default_rng(rows * vocab)
    x = as_type(masked(rng.standard_normal((rows, vocab)) * 3 + 20, mask, dtype, rng), dtype)
    token = rng.integers(0, vocab, rows).astype(np.uint32)
    if rows > 3:
        token[2], token[3] = N.NO_TOKEN, vocab + 5  # none, and one past the vocabulary
    tok = Tensor(CudaStorage.store(token, "u32"), [rows])
    X = matrix(x, dtype, pad, pad)
    top = min(20, vocab)
    got = nn.token_logprobs(X, tok, top=top)
    lp, ent, m, ls, a, p, empty = tokens64(x, token)
    # S: 2^-21 of each exp, and sums at most 600 additions deep, of a
    # distribution of rounding errors that grows as its root: 2^-18 in all;
    # the differences x - m and what is taken from them round by themselves
    with np.errstate(invalid="ignore"):
        soft = 2.0 ** -18 + 4 * e * (np.abs(np.where(np.isfinite(lp), lp, 0.0)) + 2 * ls)
    within(got.logprobs.to_f32(), lp, soft)
    st = got.statistics.to_f32().astype(np.float64)
    assert np.array_equal(st[:, 0], m)
    within(st[:, 1], ls, 2.0 ** -18 + 2 * e * ls)
    within(got.entropy.to_f32(), ent, 2.0 ** -17 * (1 + ent + ls))
    # the top ones, exactly: by value, then by index
    order = np.argsort(-x, axis=1, kind="stable")[:, :top]
    assert np.array_equal(got.top_tokens.to_numpy(), order)
    want = np.take_along_axis(a, order, 1)
    with np.errstate(invalid="ignore"):
        within(got.top_logprobs.to_f32(), want, 2.0 ** -18 + 4 * e * (np.abs(np.where(np.isfinite(want), want, 0)) + 2 * ls[:, None]))
    # the gradients, both ways
    u, v = as_type(rng.standard_normal(rows), "f32"), as_type(rng.standard_normal(rows), "f32")
    if rows > 5:
        u[5] = v[5] = 0.0
    for with_entropy in (False, True):
        v_ = v if with_entropy else np.zeros(rows)
        want, p, a, ent, u_, one = slope64(x, token, u, v_)
        D = blank(rows, vocab, dtype, pad, pad)
        nn.token_logprobs_backward(X, tok, got.statistics, tensor(u), got.entropy if with_entropy else None,
                                   tensor(v) if with_entropy else None, out=D)
        with np.errstate(invalid="ignore", over="ignore"):
            size = p * (np.abs(u_) + np.abs(v_[:, None]) * (1 + np.where(p > 0, np.abs(a), 0.0) + ent[:, None])) + np.abs(u_) * one
        tol = U[dtype] * np.abs(want) + TINY[dtype] + 2.0 ** -16 * size + 1e-37
        back, kept = read(D)
        within(back, want, tol)
        assert kept
        F = blank(rows, vocab, dtype, pad, pad)
        loss, _ = nn.token_loss(X, tok, tensor(u), tensor(v) if with_entropy else None, grad=F)
        fused, kept = read(F)
        within(fused, want, tol)
        assert kept
        within(loss.logprobs.to_f32(), lp, soft)
        within(loss.entropy.to_f32(), ent, 2.0 ** -17 * (1 + ent + ls))
        assert np.array_equal(loss.statistics.to_f32()[:, 0], m)


def test_token_gradients_agree_with_differences(device):
    rng = np.random.default_rng(1)
    rows, vocab, h = 3, 41, 1e-5
    x = as_type(rng.standard_normal((rows, vocab)) * 2, "f32")
    token = rng.integers(0, vocab, rows).astype(np.uint32)
    u, v = as_type(rng.standard_normal(rows), "f32"), as_type(rng.standard_normal(rows), "f32")
    X, tok = tensor(x), CudaStorage.store(token, "u32")
    _, grad = nn.token_loss(X, tok, tensor(u), tensor(v))
    want = np.empty(x.shape)
    for i in np.ndindex(x.shape):
        two = []
        for s in (h, -h):
            y = x.copy()
            y[i] += s
            lp, ent = tokens64(y, token)[:2]
            two.append((u * lp + v * ent).sum())
        want[i] = (two[0] - two[1]) / (2 * h)
    within(grad.to_f32(), want, 1e-5 * np.abs(want).max())


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_with_nan_and_infinity(device, dtype):
    """A NaN or +inf makes its row's results NaN (not its neighbours'); NaNs
    rank last among the top; a row whose gradients are zero is written as
    zeros all the same."""
    for vocab in (40, 3000):
        x = as_type(normal((6, vocab), 3), dtype)
        x[1, 7] = np.nan
        x[2, 11] = np.inf
        x[3, :] = np.nan
        x[4, :] = np.nan
        x[4, 20], x[4, 30] = -np.inf, 1.0
        token = np.array([1, 2, 3, 4, N.NO_TOKEN, 5], np.uint32)
        tok = CudaStorage.store(token, "u32")
        X = tensor(x, dtype)
        got = nn.token_logprobs(X, tok, top=5)
        lp, ent = got.logprobs.to_f32(), got.entropy.to_f32()
        assert np.array_equal(np.isnan(lp), [0, 1, 1, 1, 0, 0]) and lp[4] == 0.0
        assert np.array_equal(np.isnan(ent), [0, 1, 1, 1, 1, 0])
        t = got.top_tokens.to_numpy()
        order = np.argsort(-x[1], kind="stable")  # NaNs sort last
        assert np.array_equal(t[1], order[:5])
        assert t[2][0] == 11
        assert np.array_equal(t[3], np.arange(5)) and np.array_equal(t[4], [30, 20, 0, 1, 2])
        u = tensor(np.array([1, 1, 1, 1, 1, 0], np.float32))
        for grad in (nn.token_loss(X, tok, u)[1], nn.token_logprobs_backward(X, tok, got.statistics, u)):
            g = grad.to_f32()
            assert np.isnan(g[1:4]).all() and np.isfinite(g[0]).all()
            assert not g[4].any() and not g[5].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_top_tokens_of_rows_with_structure(device, dtype):
    """Ties, rows of one value, large values that lie close together or a
    fixed distance apart, more of them than there is room for at once."""
    vocab = 200003
    rng = np.random.default_rng(2)
    rows = [np.zeros(vocab), np.full(vocab, -np.inf), rng.integers(0, 3, vocab).astype(float),
            np.arange(vocab) * 1e-3, -np.arange(vocab) * 1e-3, np.zeros(vocab), rng.standard_normal(vocab)]
    for start in range(0, vocab, 4096):  # more than 2048, in one group of threads
        rows[5][start:start + 64] = 1 + rng.random(min(64, vocab - start))
    rows[6][100:4000] += 10
    few = np.full(vocab, -np.inf)
    few[[5, 77777, vocab - 1]] = [1.0, -0.0, 0.0]  # zeros of either sign are equal
    rows.append(few)
    x = as_type(np.array(rows), dtype)
    for top in (1, 20, 32):
        got = nn.token_logprobs(tensor(x, dtype), top=top, entropy=False)
        assert got.logprobs is None and got.entropy is None
        assert np.array_equal(got.top_tokens.to_numpy(), np.argsort(-x, axis=1, kind="stable")[:, :top])


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_over_the_logits(device, dtype):
    for rows, vocab in [(9, 700), (4, 5001), (3, 70000)]:
        x, token = normal((rows, vocab), 5), np.arange(rows, dtype=np.uint32)
        tok, u, v = CudaStorage.store(token, "u32"), tensor(normal(rows, 6)), tensor(normal(rows, 7))
        X = tensor(x, dtype)
        out, grad = nn.token_loss(X, tok, u, v)
        again, _ = nn.token_loss(X, tok, u, v)
        own = tensor(x, dtype)
        nn.token_loss(own, tok, u, v, grad=own)
        assert np.array_equal(own.to_numpy(), grad.to_numpy())
        assert np.array_equal(out.entropy.to_numpy(), again.entropy.to_numpy())
        back = nn.token_logprobs_backward(X, tok, out.statistics, u, out.entropy, v)
        own = tensor(x, dtype)
        nn.token_logprobs_backward(own, tok, out.statistics, u, out.entropy, v, out=own)
        assert np.array_equal(own.to_numpy(), back.to_numpy())


def test_rows_further_apart_than_32_bits_count(device):
    """Two rows 2^32 + 8 elements apart (bf16, 8.6 GB)."""
    far, cols = 2 ** 32 + 8, 1000
    s, d = CudaStorage("bf16", far + cols), CudaStorage("bf16", far + cols)
    x = normal((2, cols), 1)
    bits = f32_to_bits(x, "bf16")
    for r in range(2):
        N.call("tc_memcpy_h2d", s.ptr + 2 * r * far, bits[r].ctypes.data, 2 * cols, None)
    N.call("tc_stream_sync", None)
    X, Y = TensorView(s, [2, cols], [far, 1]), TensorView(d, [2, cols], [far, 1])
    near = Tensor(CudaStorage.store(bits, "bf16"), [2, cols])

    def rows_of(view):
        out = np.empty((2, cols), np.uint16)
        N.call("tc_stream_sync", None)
        for r in range(2):
            N.call("tc_memcpy_d2h", out[r].ctypes.data, view.storage.ptr + 2 * r * far, 2 * cols, None)
        return out

    _, st = nn.layer_norm(X, out=Y)
    assert np.array_equal(rows_of(Y), nn.layer_norm(near)[0].to_numpy())
    back = nn.layer_norm_backward(X, X, st, out=Y)
    want = nn.layer_norm_backward(near, near, st)
    assert np.array_equal(rows_of(Y), want[0].to_numpy())
    assert np.array_equal(back[1].to_numpy(), want[1].to_numpy())
    tok, u = CudaStorage.store(np.array([3, 4], np.uint32), "u32"), tensor(np.ones(2, np.float32))
    a, _ = nn.token_loss(X, tok, u, grad=Y)
    b, want = nn.token_loss(near, tok, u)
    assert np.array_equal(rows_of(Y), want.to_numpy())
    assert np.array_equal(a.logprobs.to_numpy(), b.logprobs.to_numpy())
    # and a gradient of more than 2^32 elements
    N.call("tc_memset", d.ptr, 0, d.nbytes, None)
    N.call("tc_memcpy_d2d", d.ptr + 2 * far, near.storage.ptr, 2 * cols, None)
    grads = nn.GradList([d])
    norm = nn.grad_norm(grads)
    first = as_type(x[0], "bf16")
    within(norm.to_f32(), [np.sqrt((first ** 2).sum())], 2 * e * 100)
    nn.clip_grads(grads, norm, 1.0)
    tail = np.empty(cols, np.uint16)
    N.call("tc_stream_sync", None)
    N.call("tc_memcpy_d2h", tail.ctypes.data, d.ptr + 2 * far, 2 * cols, None)
    want = first / np.sqrt((first ** 2).sum())
    within(O.widen(tail, "bf16"), want, (U["bf16"] + 4 * e) * np.abs(want))


# ---------------------------------------------------------------------------
# gradient norm and clipping
# ---------------------------------------------------------------------------
def clipped64(values, limit):
    norm = np.sqrt(sum((v ** 2).sum() for v in values))
    with np.errstate(invalid="ignore", divide="ignore"):
        by = 1.0 if norm <= limit else limit / norm
    return norm, [v * by for v in values]


@pytest.mark.parametrize("limit", [0.5, 1e6])
@pytest.mark.parametrize("kinds", [("f32",), ("f16",), ("bf16",), ("bf16", "f32", "f16")])
def test_clipping_many_tensors(device, kinds, limit):
    """Lengths from none to several chunks, off the 16-byte grid, of mixed
    types, more than one launch holds (512); into buffers of their own (some
    aligned otherwise than their gradient) and in place."""
    lengths = [1, 0, 7, 8, 13, 4096, 4099, 100003, 31, 64] + [3] * 520 + [40000]
    values, grads, outs, own = [], [], [], []
    for i, n in enumerate(lengths):
        dtype, shift = kinds[i % len(kinds)], i % 3
        v = as_type(normal(n, i) * 0.1, dtype)
        host = np.concatenate([np.full(shift, np.nan, np.float32), v.astype(np.float32)])
        values.append(v)
        grads.append(TensorView(put(host, dtype), [n], [1], shift))
        own.append(TensorView(put(host, dtype), [n], [1], shift))
        outs.append(TensorView(CudaStorage(dtype, n + 1), [n], [1], (shift + i // 3) % 2))
    norm, want = clipped64(values, limit)
    for into in (outs, None):
        held = nn.GradList(grads if into else own, into)
        got = nn.grad_norm(held)
        within(got.to_f32(), [norm], 2 * e * norm)
        nn.clip_grads(held, got, limit)
        for o, g, w in zip(into or own, grads, want):
            back = O.widen(o.storage.as_slice()[o.offset:o.offset + o.shape[0]], o.dtype)
            within(back, w, (U[o.dtype] + 4 * e) * np.abs(w) + TINY[o.dtype])


def test_norms_that_f32_squares_cannot_hold(device):
    for scale in (1e30, 1e-30):
        v = as_type(normal(1000, 1) * scale, "f32")
        got = nn.grad_norm([tensor(v)]).to_f32()
        within(got, [np.sqrt((v ** 2).sum())], 2 * e * got)
        b = as_type(v, "bf16")
        got = nn.grad_norm([tensor(b, "bf16")]).to_f32()
        within(got, [np.sqrt((b ** 2).sum())], 2 * e * got)


def test_norm_of_nothing_of_zeros_and_of_nan(device):
    assert nn.grad_norm([]).to_f32()[0] == 0.0
    nn.clip_grads([], nn.grad_norm([]), 1.0)
    zeros = tensor(np.zeros(100, np.float32))
    norm = nn.grad_norm([zeros])
    assert norm.to_f32()[0] == 0.0
    nn.clip_grads([zeros], norm, 0.0)
    assert not zeros.to_f32().any()
    for bad, rest in ((np.nan, np.nan), (np.inf, 0.0)):
        v = np.ones(100, np.float32)
        v[3] = bad
        a, b = tensor(v), tensor(np.ones(9, np.float32), "bf16")
        norm = nn.grad_norm([a, b])
        within(norm.to_f32(), [bad], 0)
        nn.clip_grads([a, b], norm, 1.0)
        assert np.isnan(a.to_f32()[3])
        within(b.to_f32(), np.full(9, rest), 0)


def test_norm_is_the_same_on_every_call(device):
    g = [tensor(normal(n, n)) for n in (100003, 7, 250000)]
    assert len({nn.grad_norm(g).to_f32().tobytes() for _ in range(5)}) == 1


# ---------------------------------------------------------------------------
# streams, and what is refused
# ---------------------------------------------------------------------------
def test_on_a_stream_of_its_own(device):
    """Every operator on a stream other than the default one, whose inputs
    were uploaded on it: the same results."""
    ctx, stream = C.c_void_p(), C.c_void_p()
    N.call("tc_ctx_create", 0, C.byref(ctx))
    N.call("tc_ctx_stream", ctx, C.byref(stream))
    on = stream.value
    x, w = tensor(normal((300, 4104), 1), "bf16"), tensor(normal(4104, 2))
    tok, u = CudaStorage.store(np.arange(300, dtype=np.uint32), "u32"), tensor(normal(300, 3))

    def all_of(s):
        y, st = nn.layer_norm(x, w, w, stream=s)
        d = nn.layer_norm_backward(y, x, st, w, stream=s)
        out = nn.token_logprobs(y, tok, top=4, stream=s)
        loss, grad = nn.token_loss(y, tok, u, u, stream=s)
        back = nn.token_logprobs_backward(y, tok, out.statistics, u, out.entropy, u, stream=s)
        norm = nn.grad_norm([*d, grad], stream=s)
        nn.clip_grads([*d, grad], norm, 1e-3, stream=s)
        N.call("tc_stream_sync", s)
        return [t.to_numpy() for t in (y, *d, out.logprobs, out.top_tokens, out.entropy, loss.logprobs, grad, back, norm)]

    N.call("tc_stream_sync", None)
    for a, b in zip(all_of(None), all_of(on)):
        assert np.array_equal(a, b)
    N.call("tc_ctx_destroy", ctx)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [9, 169, 337, 1001, 1003, 5003])
def test_top_tokens_among_nans(device, vocab, dtype):
    """NaNs rank last wherever they are: in all of a thread's 16-byte runs, in
    the single elements before and after them, in all of the row."""
    rng = np.random.default_rng(vocab)
    x = np.full((8, vocab), np.nan)
    x[1, -1], x[2, 0], x[3, vocab // 2] = 1.5, -2.0, 0.5
    x[4, -1], x[4, -2] = -np.inf, -3.0
    x[5] = np.where(rng.random(vocab) < 0.9, np.nan, rng.standard_normal(vocab))
    x[6, -5:] = [2.0, 1.0, 2.0, 3.0, -np.inf]
    x[7, :5] = [2.0, 1.0, 2.0, 3.0, -np.inf]
    x = as_type(x, dtype)
    for pad, offset in ((0, 0), (0, 1), (3, 5)):
        X = matrix(x, dtype, pad, offset)
        for top in (1, 5, 32):
            top = min(top, vocab)
            got = nn.token_logprobs(X, top=top)
            want = np.argsort(-x, axis=1, kind="stable")[:, :top]  # NaNs sort last
            assert np.array_equal(got.top_tokens.to_numpy(), want)
            assert np.isnan(got.top_logprobs.to_f32()).all()


@pytest.mark.parametrize("side", [1.0, -1.0])
def test_a_maximum_that_passes_1024(device, side):
    """Rows whose running maximum passes |x| = 1024 after many elements just
    short of it: the weights are relative to a rounded multiple of the
    maximum on one side and to the maximum itself on the other.  `to` is where
    that rounding is largest.  Tolerance: as for all rows."""
    vocab = 5003
    near = np.float32(-1024.5 if side < 0 else 1023.0) + np.arange(64, dtype=np.float32) * np.float32(2.0 ** -13)
    log2e = np.float32(1.4426950408889634)

    def left(v):  # what rounding v * log2(e) to f32 leaves out
        return np.abs(v.astype(np.float64) * np.float64(log2e) - (v * log2e).astype(np.float64))

    at = near[np.argmax(left(near))]
    later = np.float32(-1023.9) + np.arange(64, dtype=np.float32) * np.float32(2.0 ** -13)
    to = later[np.argmax(left(later))] if side < 0 else at + np.float32(8.5)
    four = np.full((4, vocab), at)
    for r, first in enumerate((2200, 3000, 4000, 4900)):
        four[r, first:] = to
    four, token = as_type(four, "f32"), np.array([0, 4950, 1, 2], np.uint32)
    lp, ent, m, ls = (np.tile(v, 300) for v in tokens64(four, token)[:4])
    # so many rows that none is shared by blocks: each thread meets both values
    X, tok = tensor(np.tile(four, (300, 1))), CudaStorage.store(np.tile(token, 300), "u32")
    u = tensor(np.ones(1200))
    for got in (nn.token_logprobs(X, tok), nn.token_loss(X, tok, u)[0]):
        st = got.statistics.to_f32().astype(np.float64)
        assert np.array_equal(st[:, 0], m)
        within(st[:, 1], ls, 2.0 ** -18 + 2 * e * ls)
        within(got.logprobs.to_f32(), lp, 2.0 ** -18 + 4 * e * (np.abs(lp) + 2 * ls))
        within(got.entropy.to_f32(), ent, 2.0 ** -17 * (1 + ent + ls))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(2, 64), (3, 256), (2, 33), (3, 16384)])
def test_layer_norm_gradients_where_the_mean_is_near_the_largest_value(device, rows, cols, dtype):
    """Rows of one value near the type's largest: their deviations are zero, so
    grad_x = rstd (g w - mean(g w)), grad_weight is zero and all is finite.
    What a thread holds beside the row's columns, or of a row past the last,
    must not enter: (0 - mean) rstd is infinite there."""
    value, eps = float(2.0 ** 121), 1e-5  # times rstd = 316: past 2^128
    x, g = np.full((rows, cols), value), as_type(normal((rows, cols), 2), dtype)
    st = tensor(np.tile([value, eps ** -0.5], (rows, 1)))
    rstd = float(np.float32(eps ** -0.5))
    dx, dw, db = nn.layer_norm_backward(tensor(g, dtype), tensor(x, dtype), st)
    want = rstd * (g - g.mean(1, keepdims=True))
    # as in test_layer_norm_and_its_gradients, with h = 0
    within(dx.to_f32(), want, U[dtype] * np.abs(want) + 48 * e * rstd * (np.abs(g) + np.abs(g).mean(1, keepdims=True)))
    assert not dw.to_f32().any()
    want = g.sum(0)
    within(db.to_f32(), want, U[dtype] * np.abs(want) + 128 * e * np.abs(g).sum(0))


# ---------------------------------------------------------------------------
# results on a stream of the caller's
# ---------------------------------------------------------------------------
def _busy(stream, room):
    """Some 50 ms of work on `stream`: 100 passes over 3 GB."""
    for _ in range(100):
        N.call("tc_memset", room.ptr, 0, room.nbytes, stream)


def test_results_are_made_in_their_streams_order(device):
    """Results that a call on another stream makes come from that stream's
    order: a block whose last use is queued on the default stream is not
    written before that use, and one dropped early is not handed to the
    default stream before the call has written it."""
    ctx, stream = C.c_void_p(), C.c_void_p()
    N.call("tc_ctx_create", 0, C.byref(ctx))
    N.call("tc_ctx_stream", ctx, C.byref(stream))
    on, shape = stream.value, (2048, 1536)  # 12 MB of f32: a pool class that nothing else here uses
    room = CudaStorage("bf16", 3 << 29)
    x = normal(shape, 1)
    X = tensor(x)
    want = nn.layer_norm(X)[0].to_numpy()
    # 1: the default stream is yet to copy from a block that has been dropped
    old = tensor(normal(shape, 2))
    kept = old.to_numpy()
    _busy(None, room)
    late = old.storage.duplicate()
    del old
    y, st = nn.layer_norm(X, stream=on)
    N.call("tc_stream_sync", on)
    N.call("tc_stream_sync", None)
    assert np.array_equal(late.as_slice().reshape(shape), kept)
    assert np.array_equal(y.to_numpy(), want)
    # 2: the call's stream is yet to write a result that has been dropped
    del y, late
    N.call("tc_stream_sync", None)
    _busy(on, room)
    for _ in range(4):
        nn.layer_norm(X, stream=on)
    fresh = [CudaStorage.zeros("f32", x.size) for _ in range(4)]
    N.call("tc_stream_sync", None)
    N.call("tc_stream_sync", on)
    for s in fresh:
        assert not s.as_slice().any()
    del st, fresh
    N.call("tc_ctx_destroy", ctx)


def test_a_result_may_outlive_its_stream(device):
    """tc_ctx_destroy waits for the stream; what was made on it stays valid, and
    goes back to the pool when it is dropped."""
    ctx, stream = C.c_void_p(), C.c_void_p()
    N.call("tc_ctx_create", 0, C.byref(ctx))
    N.call("tc_ctx_stream", ctx, C.byref(stream))
    X = tensor(normal((300, 700), 1))
    N.call("tc_stream_sync", None)
    y, st = nn.layer_norm(X, stream=stream.value)
    N.call("tc_ctx_destroy", ctx)
    assert np.array_equal(y.to_numpy(), nn.layer_norm(X)[0].to_numpy())
    at = y.storage.ptr
    del y
    assert CudaStorage("f32", 300 * 700).ptr == at


# ---------------------------------------------------------------------------
# several turns a block: rows loaded ahead, stages filled again, remainders
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("rows,cols,dtype,pad", [
    (20011, 64, "bf16", 8), (20011, 64, "f32", 0), (3001, 1001, "f16", 0), (3001, 1001, "f32", 3), (3001, 1001, "bf16", 7),
    (3001, 4096, "bf16", 0), (1501, 4096, "f32", 4), (1203, 8192, "f16", 8), (1203, 8192, "f32", 0), (701, 16384, "bf16", 0),
    (301, 16384, "f32", 0), (1203, 5001, "bf16", 0), (603, 5001, "f32", 0), (301, 20001, "bf16", 3)])
def test_layer_norm_over_many_rows(device, rows, cols, dtype, pad):
    """More rows than the blocks take in four turns, and no whole number of
    turns.  Tolerances as in test_layer_norm_and_its_gradients; a column's sum
    is still less than 128 additions deep: a thread's rows (at most 3001 / 148
    / 2), its block's groups (15), 148 partial sums over 32 lanes."""
    eps = 1e-5
    x = as_type(normal((rows, cols), 1) * 2 + 0.5, dtype)
    g = as_type(normal((rows, cols), 2), dtype)
    w, b = as_type(1 + 0.3 * normal(cols, 3), "f32"), as_type(normal(cols, 4), "f32")
    W, B = tensor(w), tensor(b)
    X, G, Y = matrix(x, dtype, pad), matrix(g, dtype, pad), blank(rows, cols, dtype, pad)
    _, st = nn.layer_norm(X, W, B, eps, out=Y)
    want, mean, rstd, h = norm64(x, w, b, eps)
    got, kept = read(Y)
    off = 32 * e * (np.abs(x).mean(1, keepdims=True) + np.abs(mean) + np.abs(x - mean))
    within(got, want, U[dtype] * np.abs(want) + TINY[dtype] + (off * rstd + 40 * e * np.abs(h)) * np.abs(w) + 4 * e * np.abs(b))
    assert kept
    s = st.to_f32().astype(np.float64)
    within(s[:, :1], mean, off.max(1, keepdims=True))
    within(s[:, 1:], rstd, rstd * (40 * e + 2 * off.max(1, keepdims=True) * rstd))
    mean, rstd = s[:, :1], s[:, 1:]
    D = blank(rows, cols, dtype, pad)
    _, dw, db = nn.layer_norm_backward(G, X, st, W, out=D)
    want, want_w, want_b, h, gw = norm_grad64(g, x, w, mean, rstd)
    got, kept = read(D)
    deep = 48 * e * rstd * (np.abs(gw) + np.abs(gw).mean(1, keepdims=True) + np.abs(h) * np.abs(gw * h).mean(1, keepdims=True))
    near = 4 * e * rstd * np.abs(mean) * rstd * (np.abs(gw * h).mean(1, keepdims=True) + np.abs(gw).mean(1, keepdims=True) * np.abs(h))
    within(got, want, U[dtype] * np.abs(want) + TINY[dtype] + deep + near)
    assert kept
    within(dw.to_f32(), want_w, U["f32"] * np.abs(want_w) + 128 * e * (np.abs(g * h) + np.abs(g * mean * rstd)).sum(0))
    within(db.to_f32(), want_b, U["f32"] * np.abs(want_b) + 128 * e * np.abs(g).sum(0))


@pytest.mark.parametrize("rows,vocab,dtype,mask,pad", [
    (80003, 33, "f16", "none", 0), (80003, 33, "f32", "inf", 3), (3001, 4104, "bf16", "inf", 0), (3001, 4104, "f16", "lowest", 8),
    (1801, 8200, "f32", "none", 0), (1801, 8200, "f32", "lowest", 4), (2003, 5003, "f16", "inf", 0), (1601, 16411, "bf16", "none", 0)])
def test_token_loss_over_many_rows(device, rows, vocab, dtype, mask, pad):
    """More rows than are resident at once: a warp or a block goes on to
    others, the next row copied while this one's gradient is written.
    Tolerances as in test_token_logprobs_and_their_gradients."""
    rng = np.random.default_rng(vocab)
    x = as_type(masked(rng.standard_normal((rows, vocab)).astype(np.float32) * 3 + 20, mask, dtype, rng), dtype)
    token = rng.integers(0, vocab, rows).astype(np.uint32)
    token[2::7] = N.NO_TOKEN
    tok = CudaStorage.store(token, "u32")
    u, v = as_type(rng.standard_normal(rows), "f32"), as_type(rng.standard_normal(rows), "f32")
    u[5::9] = v[5::9] = 0.0
    X = matrix(x, dtype, pad)
    lp, ent, m, ls = tokens64(x, token)[:4]
    for with_entropy in (True, False):
        v_ = v if with_entropy else np.zeros(rows)
        want, p, a, ent_, u_, one = slope64(x, token, u, v_)
        with np.errstate(invalid="ignore", over="ignore"):
            size = p * (np.abs(u_) + np.abs(v_[:, None]) * (1 + np.where(p > 0, np.abs(a), 0.0) + ent_[:, None])) + np.abs(u_) * one
        F = blank(rows, vocab, dtype, pad)
        out, _ = nn.token_loss(X, tok, tensor(u), tensor(v) if with_entropy else None, grad=F,
                               out=None if with_entropy else nn.TokenLogprobs(tensor(np.zeros(rows))))
        got, kept = read(F)
        within(got, want, U[dtype] * np.abs(want) + TINY[dtype] + 2.0 ** -16 * size + 1e-37)
        assert kept
        with np.errstate(invalid="ignore"):
            within(out.logprobs.to_f32(), lp, 2.0 ** -18 + 4 * e * (np.abs(np.where(np.isfinite(lp), lp, 0.0)) + 2 * ls))
        if with_entropy:
            within(out.entropy.to_f32(), ent, 2.0 ** -17 * (1 + ent + ls))
            assert np.array_equal(out.statistics.to_f32()[:, 0], m)
    if vocab < 100:
        got = nn.token_logprobs(X, tok, top=3)
        assert np.array_equal(got.top_tokens.to_numpy(), np.argsort(-x, axis=1, kind="stable")[:, :3])


def test_results_made_while_the_stream_is_captured(device):
    """A call on a stream that is captured into a CUDA graph makes its results
    as any other, where a call of the same size went before: from the pool or
    anew, without waiting for or asking after work outside the capture."""
    import torch

    X, W = tensor(normal((40, 600), 1)), tensor(normal(600, 2))
    other = tensor(normal((40, 600), 3))
    want = [t.to_numpy() for t in nn.layer_norm(other, W)]
    cap, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    nn.layer_norm(X, W, stream=cap)
    torch.cuda.synchronize()
    # the pool's blocks of these sizes: last used on the stream, on the default one, none
    for freed_on in (cap, None, "nothing"):
        graph = torch.cuda.CUDAGraph()
        if freed_on == "nothing":
            hold = [CudaStorage("f32", n) for n in (24000, 80) for _ in range(20)]
        elif freed_on is None:
            _ = [nn.layer_norm(X, W) for _ in range(8)]
            del _
        with torch.cuda.graph(graph, stream=cap):
            y, st = nn.layer_norm(X, W, stream=cap)
            nn.layer_norm(y, W, stream=cap)  # a result dropped at once
            nn.layer_norm(X, W, out=y, statistics=st, stream=cap)
        N.call("tc_memcpy_d2d", X.storage.ptr, other.storage.ptr, X.storage.nbytes, None)
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(y.to_numpy(), want[0]) and np.array_equal(st.to_numpy(), want[1])
        del graph, y, st
