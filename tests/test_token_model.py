"""The tape's layer norm and token loss against f64 gradients of the same
expression, and the small model that trains through them, the clipping and
Adam."""
from __future__ import annotations

import numpy as np
import pytest

import oracle as O
from tensorcrate_b200 import _native as N
from tensorcrate_b200 import cuda
from tensorcrate_b200.tape import Tape
from tensorcrate_b200.token_model import TokenModel
from util import normal


def _leaf(tape, values, dtype="f32"):
    values = np.asarray(values, np.float32)
    return tape.leaf(cuda.CudaStorage.store(O.narrow(values.ravel(), dtype), dtype), list(values.shape))


def _network64(x, w1, b1, gain, shift, w2, token, scale):
    """(loss, gradients of the five parameters) of the model in 64 bits."""
    a = x @ w1 + b1
    h = np.maximum(a, 0)
    mean, var = h.mean(1, keepdims=True), h.var(1, keepdims=True)
    r = 1 / np.sqrt(var + 1e-5)
    n = (h - mean) * r
    y = n * gain + shift
    z = y @ w2
    z -= z.max(1, keepdims=True)
    p = np.exp(z) / np.exp(z).sum(1, keepdims=True)
    live = token != N.NO_TOKEN
    rows = np.arange(len(token))[live]
    loss = -scale * np.log(p[rows, token[live]]).sum()
    gz = p * live[:, None] * scale
    gz[rows, token[live]] -= scale
    gy = gz @ w2.T
    gn = gy * gain
    gh = r * (gn - gn.mean(1, keepdims=True) - n * (gn * n).mean(1, keepdims=True))
    ga = gh * np.where(a > 0, 1.0, np.where(a == 0, 0.5, 0.0))
    return loss, [x.T @ ga, ga.sum(0, keepdims=True), (gy * n).sum(0), gy.sum(0), y.T @ gz]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,inputs,width,vocab", [(37, 24, 48, 101), (64, 32, 300, 1031), (5, 16, 64, 9000)])
def test_the_models_gradients(device, rows, inputs, width, vocab):
    """f32 products within the products' own contract (1e-5 sqrt K) of the f64
    gradients, through four of them: 1e-4 of each gradient's largest value."""
    model = TokenModel(inputs, width, vocab, seed=3)
    rng = np.random.default_rng(4)
    token = rng.integers(0, vocab, rows).astype(np.uint32)
    token[1] = N.NO_TOKEN
    x = normal((rows, inputs), 5)
    tape = Tape("f32")
    loss, variables = model.loss(tape, cuda.CudaStorage.store(x.ravel(), "f32"), cuda.CudaStorage.store(token, "u32"), rows - 1)
    tape.backward(loss)
    values = [p.to_f32().astype(np.float64).reshape(s) for p, s in zip(model.params, model.shapes)]
    want_loss, want = _network64(x.astype(np.float64), *values, token, 1.0 / (rows - 1))
    assert abs(tape.value(loss)[0] - want_loss) <= 1e-5 * abs(want_loss)
    for v, g in zip(variables, want):
        got = tape.grad(v).astype(np.float64)
        assert got.shape == g.shape
        assert np.abs(got - g).max() <= 1e-4 * np.abs(g).max(), v
    tape.close()


@pytest.mark.gpu
def test_a_var_used_twice_gets_both_contributions(device):
    tape = Tape("f32")
    x, w, b = _leaf(tape, normal((6, 20), 1)), _leaf(tape, 1 + 0.1 * normal(20, 2)), _leaf(tape, normal(20, 3))
    y = tape.add(tape.layer_norm(x, w, b), tape.layer_norm(x, w, b))
    tape.backward(tape.sum(tape.mul(y, y)))
    twice = [tape.grad(v) for v in (x, w, b)]
    once = Tape("f32")
    x, w, b = _leaf(once, normal((6, 20), 1)), _leaf(once, 1 + 0.1 * normal(20, 2)), _leaf(once, normal(20, 3))
    y = once.scale(once.layer_norm(x, w, b), 2.0)
    once.backward(once.sum(once.mul(y, y)))
    for v, g in zip((x, w, b), twice):
        want = once.grad(v)
        assert np.abs(g - want).max() <= 1e-5 * np.abs(want).max()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_the_model_learns(device, dtype):
    """40 steps on one batch: the loss falls from log(vocab) to less than half
    of it; the clipped gradients' norm is at most the limit."""
    rng = np.random.default_rng(2)
    vocab, rows = 257, 64
    model = TokenModel(32, 128, vocab, dtype=dtype, limit=0.5, rate=1e-2)
    token = rng.integers(0, vocab, rows).astype(np.uint32)
    x = cuda.CudaStorage.store(O.narrow(rng.standard_normal(rows * 32).astype(np.float32), dtype), dtype)
    tokens = cuda.CudaStorage.store(token, "u32")
    first = model.step(x, tokens).to_f32()[0]
    assert abs(first - np.log(vocab)) < 1.5
    for _ in range(40):
        last = model.step(x, tokens).to_f32()[0]
    assert np.isfinite(last) and last < first / 2
    assert np.isfinite(model.norm.to_f32()[0])


def test_tape_rules_refuse():
    """Before any device call: a tape with leaves over made-up addresses."""
    import ctypes as C
    out, v = C.c_void_p(), C.c_uint32()
    N.call("tc_tape_create", N.F32, None, C.byref(out))

    def leaf(*shape):
        N.call("tc_tape_leaf", out, C.c_void_p(0x1000), len(shape), N.sizes(shape), C.byref(v))
        return v.value

    x, w, short, none, scalar = leaf(2, 4), leaf(4), leaf(3), leaf(2, 0), leaf()
    norm = N.lib().tc_tape_layer_norm
    assert norm(out, x, short, w, 1e-5, C.byref(v)) == N.EINVAL and "columns" in N.last_error()
    assert norm(out, x, w, 99, 1e-5, C.byref(v)) == N.EINVAL
    assert norm(out, x, w, w, -1.0, C.byref(v)) == N.EINVAL
    assert norm(out, none, w, w, 1e-5, C.byref(v)) == N.EINVAL
    assert norm(out, scalar, w, w, 1e-5, C.byref(v)) == N.EINVAL
    loss = N.lib().tc_tape_token_loss
    assert loss(out, x, None, 1.0, C.byref(v)) == N.EINVAL
    assert loss(out, none, C.c_void_p(0x1000), 1.0, C.byref(v)) == N.EINVAL
    assert loss(out, 99, C.c_void_p(0x1000), 1.0, C.byref(v)) == N.EINVAL
    N.call("tc_tape_destroy", out)




@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_the_models_clipped_gradients_are_within_the_limit(device, dtype, monkeypatch):
    """In every step of the model: the norm of what Adam is given is at most
    the limit, and the limit itself where the norm before was above it.  Each
    gradient is rounded once to its type, the factor and the norm to f32."""
    from tensorcrate_b200 import token_model

    seen, clip = [], token_model.nn.clip_grads

    def watched(grads, norm, limit, stream=None):
        clip(grads, norm, limit, stream)
        clipped = [g.to_f32().astype(np.float64) for g in grads._keep[0]]
        seen.append((float(norm.to_f32()[0]), np.sqrt(sum((g ** 2).sum() for g in clipped))))

    monkeypatch.setattr(token_model.nn, "clip_grads", watched)
    rng = np.random.default_rng(7)
    limit, vocab, rows = 0.05, 257, 64
    model = TokenModel(32, 128, vocab, dtype=dtype, limit=limit, rate=1e-2)
    x = cuda.CudaStorage.store(O.narrow(rng.standard_normal(rows * 32).astype(np.float32), dtype), dtype)
    tokens = cuda.CudaStorage.store(rng.integers(0, vocab, rows).astype(np.uint32), "u32")
    for _ in range(6):
        model.step(x, tokens)
    near = 4 * 2.0 ** -24 + {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}[dtype]
    assert len(seen) == 6 and any(before > limit for before, _ in seen)
    for before, after in seen:
        assert abs(after - min(before, limit)) <= near * limit
