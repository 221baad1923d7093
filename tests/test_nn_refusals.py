"""What the training operators refuse, on the host and before any device
call: by the C entry points, and by the Python functions over them."""
from __future__ import annotations

import ctypes as C

import pytest

from tensorcrate_b200 import _native as N
from tensorcrate_b200 import nn
from tensorcrate_b200.cuda import CudaStorage, Tensor, TensorView

P = C.c_void_p(0x1000)
ODD = C.c_void_p(0x1004)  # off the 8-byte grid that statistics need


def status(name, *args):
    return getattr(N.lib(), name)(*args)


def norm(**k):
    a = dict(dtype=N.F32, param=N.F32, rows=2, cols=4, x=P, xs=4, w=P, b=P, eps=1e-5, y=P, ys=4, st=P) | k
    return status("tc_layer_norm", *a.values(), None)


def norm_back(**k):
    a = dict(dtype=N.F32, param=N.F32, rows=2, cols=4, g=P, gs=4, x=P, xs=4, st=P, w=P, dx=P, dxs=4, dw=P, db=P) | k
    return status("tc_layer_norm_backward", *a.values(), None)


@pytest.mark.parametrize("call", [norm, norm_back])
def test_layer_norm_refuses(call):
    assert call(dtype=9) == N.EINVAL
    assert call(dtype=N.U32, param=N.U32) == N.EINVAL
    assert call(param=N.BF16) == N.EINVAL  # f32 rows, bf16 parameters
    assert call(dtype=N.F16, param=N.BF16) == N.EINVAL
    assert call(cols=0) == N.EINVAL
    assert call(xs=3) == N.EINVAL and "apart" in N.last_error()
    assert call(x=None) == N.EINVAL
    assert call(st=ODD) == N.EINVAL
    assert call(rows=2 ** 40, xs=2 ** 40) == N.ERANGE


def test_layer_norm_refuses_more():
    assert norm(eps=-1.0) == N.EINVAL and norm(eps=float("nan")) == N.EINVAL
    assert norm(ys=3) == N.EINVAL and norm(y=None) == N.EINVAL
    assert norm_back(gs=3) == N.EINVAL and norm_back(dxs=3) == N.EINVAL
    assert norm_back(g=None) == N.EINVAL and norm_back(st=None) == N.EINVAL
    assert norm(rows=0) == N.OK
    assert norm_back(dx=None, dw=None, db=None) == N.OK


def logprobs(**k):
    a = dict(dtype=N.F32, rows=2, vocab=8, x=P, xs=8, tok=P, lp=P, ent=P, st=P, top=2, tt=P, tl=P) | k
    return status("tc_token_logprobs", *a.values(), None)


def back(**k):
    a = dict(dtype=N.F32, rows=2, vocab=8, x=P, xs=8, tok=P, st=P, ent=P, u=P, v=P, d=P, ds=8) | k
    return status("tc_token_logprobs_backward", *a.values(), None)


def loss(**k):
    a = dict(dtype=N.F32, rows=2, vocab=8, x=P, xs=8, tok=P, u=P, v=P, lp=P, ent=P, st=P, d=P, ds=8) | k
    return status("tc_token_loss", *a.values(), None)


@pytest.mark.parametrize("call", [logprobs, back, loss])
def test_token_operators_refuse(call):
    assert call(dtype=N.U32) == N.EINVAL
    assert call(vocab=0) == N.EINVAL
    assert call(vocab=2 ** 32 - 1, xs=2 ** 32, **({} if call is logprobs else {"ds": 2 ** 32})) == N.ERANGE
    assert call(xs=7) == N.EINVAL
    assert call(x=None) == N.EINVAL
    assert call(tok=None) == N.EINVAL
    assert call(st=ODD) == N.EINVAL
    assert call(rows=2 ** 40, xs=2 ** 40) == N.ERANGE
    assert call(rows=0) == N.OK


def test_token_operators_refuse_more():
    assert logprobs(top=9) == N.EINVAL  # of 8
    assert logprobs(vocab=100, xs=100, top=N.MAX_TOP + 1) == N.EINVAL
    assert logprobs(tt=None) == N.EINVAL and logprobs(tl=None) == N.EINVAL
    assert logprobs(lp=None, ent=None, st=None, top=0, tt=None, tl=None) == N.OK
    assert back(ent=None) == N.EINVAL  # the entropy's gradient without the entropy
    assert back(d=None) == N.EINVAL and back(ds=7) == N.EINVAL and back(st=None) == N.EINVAL
    assert loss(d=None) == N.EINVAL and loss(ds=7) == N.EINVAL


def test_clipping_refuses():
    one = (N.Gradient * 1)()
    one[0].g, one[0].out, one[0].n, one[0].dtype = 0x1000, 0x1000, 4, N.F32
    assert status("tc_grad_norm", None, 1, P, None) == N.EINVAL
    assert status("tc_grad_norm", one, 1, None, None) == N.EINVAL
    assert status("tc_clip_grads", one, 1, None, 1.0, None) == N.EINVAL
    assert status("tc_clip_grads", one, 1, P, -1.0, None) == N.EINVAL
    assert status("tc_clip_grads", one, 1, P, float("nan"), None) == N.EINVAL
    one[0].out = None
    assert status("tc_clip_grads", one, 1, P, 1.0, None) == N.EINVAL
    one[0].dtype = N.U32
    assert status("tc_grad_norm", one, 1, P, None) == N.EINVAL
    one[0].dtype, one[0].n = N.F32, 2 ** 50
    assert status("tc_grad_norm", one, 1, P, None) == N.ERANGE
    assert status("tc_clip_grads", None, 0, P, 1.0, None) == N.OK


def held(shape, dtype="f32", strides=None, room=None):
    n = 1
    for e in shape:
        n *= e
    s = CudaStorage(dtype, n if room is None else room, ptr=0x1000)
    return Tensor(s, shape) if strides is None else TensorView(s, list(shape), list(strides))


def test_python_functions_refuse():
    x, w = held([2, 4]), held([4])
    with pytest.raises(ValueError, match="last axis"):
        nn.layer_norm(held([2, 4], strides=[1, 2]))
    with pytest.raises(ValueError, match="do not step as one"):
        nn.layer_norm(held([2, 3, 4], strides=[100, 4, 1], room=200))
    with pytest.raises(ValueError, match="past"):
        nn.layer_norm(held([2, 4], strides=[100, 1]))
    with pytest.raises(ValueError, match="no rows"):
        nn.layer_norm(held([]))
    with pytest.raises(ValueError, match="elements, expected 4"):
        nn.layer_norm(x, held([5]))
    with pytest.raises(ValueError, match="element type"):
        nn.layer_norm(x, held([4], "bf16"))
    with pytest.raises(ValueError, match="weight is bf16, bias f32"):
        nn.layer_norm(held([2, 4], "bf16"), held([4], "bf16"), w)
    with pytest.raises(ValueError, match="differ"):
        nn.layer_norm(x, out=held([4, 2]))
    with pytest.raises(ValueError, match="differ"):
        nn.layer_norm_backward(held([4, 2]), x, held([2, 2]))
    with pytest.raises(ValueError, match="statistics"):
        nn.layer_norm_backward(x, x, held([3, 2]))
    with pytest.raises(ValueError, match="tokens"):
        nn.token_logprobs(x, held([3], "u32"), out=nn.TokenLogprobs(held([2])))
    with pytest.raises(ValueError, match="tokens"):
        nn.token_logprobs(x, held([2]), out=nn.TokenLogprobs(held([2])))
    with pytest.raises(ValueError, match="go together"):
        nn.token_logprobs(x, out=nn.TokenLogprobs(top_tokens=held([2, 1], "u32")))
    with pytest.raises(ValueError, match="token_logprobs'"):
        nn.token_loss(x, held([2], "u32"), held([2]), out=nn.TokenLogprobs(top_tokens=held([2, 1], "u32")), grad=x)
    with pytest.raises(ValueError, match="1 gradients, 2 outputs"):
        nn.GradList([x], [x, x])
    with pytest.raises(ValueError, match="not contiguous"):
        nn.GradList([held([2, 4], strides=[8, 1], room=20)])
    with pytest.raises(ValueError, match="element type"):
        nn.GradList([held([4], "u32")])
    with pytest.raises(ValueError, match="expected 1"):
        nn.clip_grads([x], held([2]), 1.0)


def test_what_lies_outside_a_storage_is_refused():
    """By the host, as the layout checks of the other operators do: a tensor
    whose shape has more elements than its storage, a view that begins before
    its storage."""
    short = Tensor(CudaStorage("f32", 7, ptr=0x1000), [2, 4])
    before = TensorView(CudaStorage("f32", 64, ptr=0x1000), [2, 4], [4, 1], -8)
    vector = TensorView(CudaStorage("f32", 64, ptr=0x1000), [4], [1], -1)
    x, st, tok, u = held([2, 4]), held([2, 2]), held([2], "u32"), held([2])
    for bad, why in ((short, "past 7 elements"), (before, "before")):
        for call in (lambda: nn.layer_norm(bad), lambda: nn.layer_norm(x, out=bad), lambda: nn.layer_norm_backward(bad, x, st),
                     lambda: nn.layer_norm_backward(x, x, st, out=bad), lambda: nn.token_logprobs(bad, tok),
                     lambda: nn.token_logprobs_backward(x, tok, st, u, out=bad),
                     lambda: nn.token_loss(x, tok, u, out=nn.TokenLogprobs(), grad=bad)):
            with pytest.raises(ValueError, match=why):
                call()
    with pytest.raises(ValueError, match="before"):
        nn.layer_norm(x, vector)
    with pytest.raises(ValueError, match="before"):
        nn.GradList([vector])
