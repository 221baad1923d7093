"""Blocks of a cluster that share a row store into one another's shared
memory.  CUDA allows that only once the other block has started, so each such
kernel has the cluster's blocks meet before its first store.

Nothing on a GPU shows reliably that the meeting is missing, so the sources are
read for it; the GPU test runs many such calls close together."""
from __future__ import annotations

import re
from pathlib import Path

import numpy as np
import pytest

from tensorcrate_b200 import nn
from tensorcrate_b200.cuda import CudaStorage, Tensor
from test_gpu_nn import as_type, e, put, slope64, tokens64, within

CSRC = Path(__file__).resolve().parent.parent / "tensorcrate_b200" / "csrc"


def _body(text: str, at: int) -> str:
    """From the first brace after `at` to the one that closes it."""
    start = text.index("{", at)
    depth = 0
    for i in range(start, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[start:i]
    raise AssertionError("unbalanced braces")


def _functions():
    """(name, body) of every kernel."""
    for path in sorted(CSRC.glob("*.cu")):
        text = re.sub(r"//[^\n]*", "", path.read_text())
        for m in re.finditer(r"__global__\s+void\s+(?:__launch_bounds__\([^)]*\)\s*)?(\w+)\(", text):
            yield m[1], _body(text, m.end())


def test_blocks_meet_before_their_first_store_to_one_another():
    seen = []
    for name, body in _functions():
        if "cluster_parts()" not in body:
            continue
        stores = [body.index(s) for s in ("store_at(", "row_join<") if s in body]
        if not stores:
            continue
        seen.append(name)
        before = body[:min(stores)]
        assert "cluster_sync()" in before or "cluster_arrive()" in before, name
    assert {"token_rows", "token_loss_twice", "norm_grad_rows"} <= set(seen)
    # where a kernel only arrives at its start, the join waits before it stores
    text = (CSRC / "logprob.cu").read_text()
    join = _body(text, text.index("Sums row_join("))
    assert 0 <= join.index("cluster_wait()") < join.index("store_at(")


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,dtype", [(1, 9001, "f32"), (3, 50257, "bf16"), (1, 131072, "f16"), (2, 262144, "bf16")])
def test_rows_shared_by_a_cluster_many_calls_together(device, rows, vocab, dtype):
    """Calls queued one after another on different logits: every one has the
    results of its own logits, the first row of each kernel among them."""
    rng = np.random.default_rng(vocab)
    token = rng.integers(0, vocab, rows).astype(np.uint32)
    tok, u = CudaStorage.store(token, "u32"), np.ones(rows)
    up = Tensor(put(u, "f32"), [rows])
    host = [as_type(rng.standard_normal((rows, vocab)) * 3 + 5 * k, dtype) for k in range(4)]
    logits = [Tensor(put(x, dtype), [rows, vocab]) for x in host]
    got = [(k, nn.token_logprobs(logits[k], tok, top=3), nn.token_loss(logits[k], tok, up)) for _ in range(12) for k in range(4)]
    first = {}
    for k, told, (loss, grad) in got:
        mine = [t.to_numpy() for t in (told.logprobs, told.entropy, told.statistics, told.top_tokens, told.top_logprobs,
                                       loss.logprobs, loss.entropy, loss.statistics, grad)]
        if k not in first:
            first[k] = mine
            lp, ent, m, ls = tokens64(host[k], token)[:4]
            # as in test_token_logprobs_and_their_gradients
            within(told.logprobs.to_f32(), lp, 2.0 ** -18 + 4 * e * (np.abs(lp) + 2 * ls))
            within(told.entropy.to_f32(), ent, 2.0 ** -17 * (1 + ent + ls))
            assert np.array_equal(told.statistics.to_f32()[:, 0], m)
            assert np.array_equal(told.top_tokens.to_numpy(), np.argsort(-host[k], axis=1, kind="stable")[:, :3])
            want, p = slope64(host[k], token, u, np.zeros(rows))[:2]
            step = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype]
            tiny = {"f32": 0.0, "f16": 2.0 ** -24, "bf16": 0.0}[dtype]
            one = np.zeros_like(p)
            one[np.arange(rows), token] = 1.0
            within(grad.to_f32(), want, step * np.abs(want) + tiny + 2.0 ** -16 * (p + one) + 1e-37)
        for a, b in zip(first[k], mine):
            assert np.array_equal(a, b)
