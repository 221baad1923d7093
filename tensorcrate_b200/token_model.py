"""A small model over a vocabulary, trained step by step: features through a
dense layer, a layer norm and the output product to logits, the mean log
probability of the given tokens as the loss, its gradients clipped by their
global norm, Adam.  It runs the training operators together as a program
would use them, on the tape.

    python -m tensorcrate_b200.token_model [--steps 200] [--width 512] [--vocab 8192] [--batch 1024]
"""
from __future__ import annotations

import argparse
import time

import numpy as np

from . import _native as N
from . import nn
from .cuda import CudaStorage, f32_to_bits, synchronize
from .mlp import xavier
from .tape import Tape


class TokenModel:
    """logits = layer_norm(relu(x W1 + b1)) W2, rows of x the positions."""

    def __init__(self, inputs: int, width: int, vocab: int, dtype: str = "f32", limit: float = 1.0, rate: float = 1e-3,
                 seed: int = 0):
        rng = np.random.default_rng(seed)
        self.dtype, self.limit, self.rate, self.steps = dtype, limit, rate, 0
        self.beta1, self.beta2, self.eps = 0.9, 0.99, 1e-8 if dtype == "f32" else 1e-6
        values = [xavier(inputs, width, rng), np.zeros(width, np.float32), np.ones(width, np.float32),
                  np.zeros(width, np.float32), xavier(width, vocab, rng)]
        self.shapes = [[inputs, width], [1, width], [width], [width], [width, vocab]]
        self.params = [CudaStorage.store(f32_to_bits(v.ravel(), dtype), dtype) for v in values]
        self.moments = [(CudaStorage.zeros(dtype, p.len), CudaStorage.zeros(dtype, p.len)) for p in self.params]
        self.norm = CudaStorage("f32", 1)

    def loss(self, tape: Tape, x: CudaStorage, tokens: CudaStorage, count: int | None = None):
        """(loss var, parameter vars): the mean over `count` tokens (all rows
        unless some hold nn.NO_TOKEN)."""
        rows = tokens.len
        w1, b1, gain, shift, w2 = v = [tape.leaf(p, s) for p, s in zip(self.params, self.shapes)]
        hidden = tape.relu(tape.add(tape.matmul(tape.leaf(x, [rows, self.shapes[0][0]]), w1), b1))
        logits = tape.matmul(tape.layer_norm(hidden, gain, shift), w2)
        return tape.token_loss(logits, tokens, 1.0 / (count or rows)), v

    def step(self, x: CudaStorage, tokens: CudaStorage, count: int | None = None) -> CudaStorage:
        """One training step; the loss (one element on the device).  The
        gradients' norm before clipping is left in self.norm."""
        tape = Tape(self.dtype)
        loss, variables = self.loss(tape, x, tokens, count)
        tape.backward(loss)
        grads = [tape.grad_storage(v) for v in variables]
        held = nn.GradList(grads)
        nn.grad_norm(held, out=self.norm)
        nn.clip_grads(held, self.norm, self.limit)
        self.steps += 1
        entries = (N.AdamTensor * len(grads))()
        for e, p, g, (m, v) in zip(entries, self.params, grads, self.moments):
            e.p, e.g, e.m, e.v, e.n = p.ptr, g.ptr, m.ptr, v.ptr, p.len
        N.call("tc_adam_multi", N.DTYPES[self.dtype], entries, len(grads), int(self.steps > 1), self.rate, self.beta1,
               self.beta2, self.eps, 1.0 / (1.0 - self.beta1 ** self.steps), 1.0 / (1.0 - self.beta2 ** self.steps), None)
        out = tape.value_storage(loss).duplicate()
        tape.close()
        return out


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--width", type=int, default=512)
    ap.add_argument("--vocab", type=int, default=8192)
    ap.add_argument("--batch", type=int, default=1024)
    a = ap.parse_args()
    N.call("tc_set_device", 0)
    rng = np.random.default_rng(1)
    # each token has a feature vector of its own, seen with noise
    features = rng.standard_normal((a.vocab, 64)).astype(np.float32)
    model = TokenModel(64, a.width, a.vocab)
    start = time.perf_counter()
    for step in range(a.steps):
        tokens = rng.integers(0, a.vocab, a.batch).astype(np.uint32)
        x = features[tokens] + 0.1 * rng.standard_normal((a.batch, 64)).astype(np.float32)
        loss = model.step(CudaStorage.store(x.ravel(), "f32"), CudaStorage.store(tokens, "u32"))
        if step % 20 == 0 or step == a.steps - 1:
            print(f"step {step:4d}  loss {loss.to_f32()[0]:.4f}  gradient norm {model.norm.to_f32()[0]:.4f}")
    synchronize()
    print(f"{(time.perf_counter() - start) / a.steps * 1e3:.2f} ms a step")


if __name__ == "__main__":
    main()
