"""What is measured of the training operators: layer norm and its gradients, the log
probabilities of given tokens (with entropy, alternatives, gradient) and the gradients' global
norm with clipping.  A training step over a vocabulary runs all three: the norm before the
output product, the loss after it, the clipping before the optimizer.

Each case is one call of one operator on inputs that such a step has in hand.  `run` gives the
operators' plain form in 32 bits, or, where `own` is set, the framework's calls."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5
NO_TOKEN = -1  # 0xFFFFFFFF as the u32 that the framework reads: a position without a token


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def norm(rows, cols, dtype, params="same", pad=0, grad=False):
    return {"op": "norm_grad" if grad else "norm", "rows": rows, "cols": cols, "dtype": dtype, "params": params, "pad": pad}


def tokens(op, rows, vocab, dtype, entropy=True, top=0, mask="none", pad=0):
    return {"op": op, "rows": rows, "vocab": vocab, "dtype": dtype, "entropy": entropy, "top": top, "mask": mask, "pad": pad}


def clip(layers, width, dtype, limit="over", mixed=True):
    return {"op": "clip", "layers": layers, "width": width, "dtype": dtype, "limit": limit, "mixed": mixed}


def listed():
    return [
        # a few positions of a served sequence: a call whose latency counts
        {"name": "norm, 4 rows", **norm(4, 4096, "bf16", "f32")},
        # the broadcast workload's tensor [64, 512, 1024], normalised over its last axis
        {"name": "norm, 32768 x 1024 f32", **norm(32768, 1024, "f32")},
        # the gradient at the dense network's batch and hidden width
        {"name": "norm gradient, 2048 x 4096", **norm(2048, 4096, "bf16", grad=True)},
        # the gradient over a long batch of tokens and a wide model, weights kept in 32 bits
        {"name": "norm gradient, 16384 x 8192", **norm(16384, 8192, "bf16", "f32", grad=True)},
        # an odd width: no row but the first starts on a 16-byte boundary
        {"name": "norm gradient, 4099 x 1001", **norm(4099, 1001, "f16", grad=True)},
        # one served token: its log probability, its alternatives
        {"name": "token, 1 x 131072, top 20", **tokens("logprobs", 1, 131072, "bf16", top=20)},
        # a prompt scored with alternatives over an odd vocabulary, some of it masked
        {"name": "tokens, 2048 x 50257, top 8", **tokens("logprobs", 2048, 50257, "bf16", top=8, mask="inf")},
        # the loss's gradient from kept statistics, logits in 32 bits
        {"name": "token gradient, 4096 x 32768", **tokens("logprobs_grad", 4096, 32768, "f32")},
        # a training batch: loss and gradient in one call
        {"name": "token loss, 4096 x 131072", **tokens("loss", 4096, 131072, "bf16", entropy=False)},
        # a small network's gradients, clipped: latency
        {"name": "clip, 1 layer of 64", **clip(1, 64, "f32")},
        # the dense network's widths (1024 and 4096)
        {"name": "clip, 4 layers of 1024", **clip(4, 1024, "bf16")},
        # a large model's: many tensors, no power of two among them
        {"name": "clip, 24 layers of 2001", **clip(24, 2001, "bf16")},
    ]


def between(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def odd_or_round(rng, n, low):
    """Half of the sizes as drawn, half on a multiple of 64 (where one is near)."""
    return n if n < 128 or rng.random() < 0.5 else max(low, n // 64 * 64)


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "logprobs", "logprobs_grad", "loss", "clip"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    pad = rng.choice([0, 0, 0, 8, 3])
    if op in ("norm", "norm_grad"):
        cols = odd_or_round(rng, between(rng, 8, 16384), 8)
        rows = between(rng, 1, min(65536, (1 << 26) // cols))
        return norm(rows, cols, dtype, rng.choice(["same", "f32"]), pad, op == "norm_grad")
    if op == "clip":
        width = odd_or_round(rng, between(rng, 16, 2048), 16)
        layers = between(rng, 1, max(1, min(64, (1 << 28) // (8 * width * width))))
        return clip(layers, width, dtype, rng.choice(["over", "over", "under"]), rng.random() < 0.5)
    vocab = odd_or_round(rng, between(rng, 64, 262144), 64)
    top = rng.choice([0, 1, 5, 20]) if op == "logprobs" else 0
    rows = between(rng, 1, min(16384, (1 << (26 if top else 28)) // vocab))
    return tokens(op, rows, vocab, dtype, rng.random() < 0.5, top, rng.choice(["none", "inf", "lowest"]), pad)


# ---------------------------------------------------------------------------
# the inputs
# ---------------------------------------------------------------------------
def matrix(rows, cols, pad, dtype, gen=None, scale=1.0):
    """[rows, cols] whose rows are cols + pad elements apart; filled from `gen` where it is given."""
    whole = torch.empty((rows, cols + pad), dtype=TYPES[dtype], device="cuda")
    if gen is not None:
        whole.normal_(0.0, scale, generator=gen)
    return whole[:, :cols]


def clip_shapes(case):
    """A layer's tensors: two products' weights, their biases, a norm's weight and bias."""
    w = case["width"]
    small = "f32" if case["mixed"] else case["dtype"]
    one = [(w * 4 * w, case["dtype"]), (4 * w, small), (4 * w * w, case["dtype"]), (w, small), (w, small), (w, small)]
    return one * case["layers"]


def cut(flat, sizes):
    """Consecutive runs of `flat`, as a program's flat gradient buffer of each type holds its tensors."""
    return list(torch.split(flat, sizes))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, state = case["op"], {"case": case}
    if op in ("norm", "norm_grad"):
        rows, cols, pad, dtype = (case[k] for k in ("rows", "cols", "pad", "dtype"))
        kind = TYPES["f32" if case["params"] == "f32" else dtype]
        x = matrix(rows, cols, pad, dtype, gen, 2.0)
        x += 0.5  # activations are not centred
        state["x"] = x
        state["weight"] = (1.0 + 0.2 * torch.randn(cols, generator=gen, device="cuda")).to(kind)
        state["bias"] = (0.2 * torch.randn(cols, generator=gen, device="cuda")).to(kind)
        state["statistics"] = torch.empty((rows, 2), device="cuda")
        if op == "norm":
            state["y"] = matrix(rows, cols, pad, dtype)
        else:
            # what the forward call left: each row's mean and 1 / sqrt(variance + eps)
            mean = x.double().mean(1)
            state["statistics"][:, 0] = mean
            state["statistics"][:, 1] = torch.rsqrt((x.double() - mean[:, None]).square().mean(1) + EPS)
            state["grad"] = matrix(rows, cols, pad, dtype, gen, 0.01)
            state["grad_x"] = matrix(rows, cols, pad, dtype)
            state["grad_weight"], state["grad_bias"] = torch.empty_like(state["weight"]), torch.empty_like(state["bias"])
        return state
    if op == "clip":
        shapes = clip_shapes(case)
        grads, outs = [None] * len(shapes), [None] * len(shapes)
        state["flat"], state["clipped"], square = [], [], 0.0
        for dtype in sorted({d for _, d in shapes}):
            at = [i for i, (_, d) in enumerate(shapes) if d == dtype]
            sizes = [shapes[i][0] for i in at]
            flat = torch.empty(sum(sizes), dtype=TYPES[dtype], device="cuda").normal_(0.0, 1e-2, generator=gen)
            square += sum(sizes) * 1e-4
            state["flat"].append(flat)
            state["clipped"].append(torch.empty_like(flat))
            for i, g, o in zip(at, cut(flat, sizes), cut(state["clipped"][-1], sizes)):
                grads[i], outs[i] = g, o
        # the limit lies well to one side of the norm that such values have
        state["limit"] = math.sqrt(square) * (0.3 if case["limit"] == "over" else 4.0)
        state["grads"], state["outs"], state["norm"] = grads, outs, torch.empty(1, device="cuda")
        return state
    rows, vocab, pad, dtype = (case[k] for k in ("rows", "vocab", "pad", "dtype"))
    x = matrix(rows, vocab, pad, dtype, gen, 2.5)
    token = torch.randint(0, vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    likely = 6.0 + torch.randn(rows, generator=gen, device="cuda")
    value = -math.inf if case["mask"] == "inf" else torch.finfo(TYPES[dtype]).min
    if case["mask"] != "none":
        # a grammar leaves about a tenth of the vocabulary
        x[:, torch.rand(vocab, generator=gen, device="cuda") > 0.1] = value
    # a trained model gives the tokens that follow more than the others
    x[torch.arange(rows, device="cuda"), token.long()] = likely.to(x.dtype)
    if case["mask"] != "none":
        x[5::97] = value  # some positions are left nothing
    if rows > 1:
        token[torch.rand(rows, generator=gen, device="cuda") < 0.1] = NO_TOKEN
    state["logits"], state["tokens"] = x, token
    if op != "logprobs":
        state["grad_logprobs"] = torch.randn(rows, generator=gen, device="cuda") / rows
        state["grad_entropy"] = torch.randn(rows, generator=gen, device="cuda") * (0.01 / rows) if case["entropy"] else None
        state["grad_logits"] = matrix(rows, vocab, pad, dtype)
    if op == "logprobs_grad":
        # what the forward call left: each row's maximum, the log of the sum beside it, its entropy
        statistics, entropy = [], []
        for part in x.split(max(1, (1 << 26) // vocab)):
            m, s, t = sums(part.double())
            statistics.append(torch.stack([m, s.log()], 1).float())
            entropy.append((s.log() - t / s).float())
        state["statistics"] = torch.cat(statistics)
        state["entropy"] = torch.cat(entropy) if case["entropy"] else None
        return state
    state["logprobs"] = torch.empty(rows, device="cuda")
    state["entropy"] = torch.empty(rows, device="cuda") if case["entropy"] else None
    state["statistics"] = torch.empty((rows, 2), device="cuda")
    if op == "logprobs" and case["top"]:
        k = min(case["top"], vocab)
        state["top_tokens"] = torch.empty((rows, k), dtype=torch.int32, device="cuda")
        state["top_logprobs"] = torch.empty((rows, k), device="cuda")
    return state


def sums(x):
    """Each row's maximum, the sum of exp(x - maximum) and of that times (x - maximum); a row
    of minus infinities has the sums 1 and 0, so that what is taken from them is finite."""
    m = x.amax(1)
    d = x - torch.where(m == -math.inf, 0.0, m)[:, None]
    e = d.exp()
    t = torch.where(d == -math.inf, 0.0, e * d).sum(1)
    return m, torch.where(m == -math.inf, 1.0, e.sum(1)), t


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def plain_norm(s):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = 1.0 / (d.square().mean(1, keepdim=True) + EPS).sqrt()
    y = d * rstd * s["weight"].float() + s["bias"].float()
    return {"y": y.to(s["x"].dtype), "statistics": torch.cat([mean, rstd], 1)}


def plain_norm_grad(s):
    x, g, w = s["x"].float(), s["grad"].float(), s["weight"]
    mean, rstd = s["statistics"][:, :1], s["statistics"][:, 1:]
    h = (x - mean) * rstd
    gw = g * w.float()
    dx = rstd * (gw - gw.mean(1, keepdim=True) - h * (gw * h).mean(1, keepdim=True))
    return {"grad_x": dx.to(s["x"].dtype), "grad_weight": (g * h).sum(0).to(w.dtype), "grad_bias": g.sum(0).to(w.dtype)}


def plain_logprobs(s):
    x, case = s["logits"].float(), s["case"]
    m, e, t = sums(x)
    log_sum = e.log()
    present = s["tokens"] != NO_TOKEN
    at = x.gather(1, torch.where(present, s["tokens"], 0).long()[:, None])[:, 0]
    safe = torch.where(m == -math.inf, 0.0, m)
    out = {"logprobs": torch.where(present, at - safe - log_sum, 0.0), "statistics": torch.stack([m, log_sum], 1)}
    if case["entropy"]:
        out["entropy"] = log_sum - t / e
    if case["top"]:
        value, index = torch.sort(x, dim=1, descending=True, stable=True)
        k = min(case["top"], case["vocab"])
        out["top_tokens"] = index[:, :k].int()
        out["top_logprobs"] = value[:, :k] - safe[:, None] - log_sum[:, None]
    return out


def plain_logits_grad(s, statistics, entropy):
    x = s["logits"].float()
    m, log_sum = statistics[:, :1], statistics[:, 1:]
    d = x - torch.where(m == -math.inf, 0.0, m) - log_sum
    p = d.exp()
    g = -s["grad_logprobs"] * (s["tokens"] != NO_TOKEN)
    grad = p * g[:, None]
    if s["grad_entropy"] is not None:
        grad = grad - torch.where(d == -math.inf, 0.0, p * (d + entropy[:, None])) * s["grad_entropy"][:, None]
    alive = (s["tokens"] != NO_TOKEN) & (m[:, 0] != -math.inf)
    at = torch.where(alive, s["tokens"], 0).long()[:, None]
    grad = grad.scatter_add(1, at, torch.where(alive, s["grad_logprobs"], 0.0)[:, None])
    return grad.to(s["logits"].dtype)


def plain_logprobs_grad(s):
    return {"grad_logits": plain_logits_grad(s, s["statistics"], s["entropy"])}


def plain_loss(s):
    out = plain_logprobs(s)
    return {**out, "grad_logits": plain_logits_grad(s, out["statistics"], out.get("entropy"))}


def plain_clip(s):
    norm = torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()
    by = torch.clamp(s["limit"] / norm, max=1.0)
    return {"norm": norm[None], "grads": [(f.float() * by).to(f.dtype) for f in s["flat"]]}


PLAIN = {"norm": plain_norm, "norm_grad": plain_norm_grad, "logprobs": plain_logprobs, "logprobs_grad": plain_logprobs_grad,
         "loss": plain_loss, "clip": plain_clip}


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def handles(s):
    """The state's buffers as the framework's tensors, which a program that uses it holds."""
    from tensorcrate_b200 import nn
    from tensorcrate_b200.cuda import CudaStorage, TensorView

    names = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16", torch.int32: "u32"}

    def view(t):
        reach = 1 + sum((e - 1) * st for e, st in zip(t.shape, t.stride()))
        return TensorView(CudaStorage(names[t.dtype], reach, ptr=t.data_ptr()), list(t.shape), list(t.stride()))

    h = {k: view(v) for k, v in s.items() if isinstance(v, torch.Tensor)}
    if s["case"]["op"] == "clip":
        h["grads"] = nn.GradList([view(g) for g in s["grads"]], [view(o) for o in s["outs"]])
    if s["case"]["op"] in ("logprobs", "loss"):
        h["out"] = nn.TokenLogprobs(**{k: h.get(k) for k in ("logprobs", "entropy", "statistics", "top_tokens", "top_logprobs")})
    return nn, h


def run(state):
    op = state["case"]["op"]
    if not own:
        return PLAIN[op](state)
    if "handles" not in state:
        state["handles"] = handles(state)
    nn, h = state["handles"]
    on = torch.cuda.current_stream().cuda_stream
    if op == "norm":
        nn.layer_norm(h["x"], h["weight"], h["bias"], EPS, out=h["y"], statistics=h["statistics"], stream=on)
        return {"y": state["y"], "statistics": state["statistics"]}
    if op == "norm_grad":
        nn.layer_norm_backward(h["grad"], h["x"], h["statistics"], h["weight"], out=h["grad_x"], grad_weight=h["grad_weight"],
                               grad_bias=h["grad_bias"], stream=on)
        return {k: state[k] for k in ("grad_x", "grad_weight", "grad_bias")}
    if op == "clip":
        nn.grad_norm(h["grads"], out=h["norm"], stream=on)
        nn.clip_grads(h["grads"], h["norm"], state["limit"], stream=on)
        return {"norm": state["norm"], "grads": state["clipped"]}
    if op == "logprobs_grad":
        nn.token_logprobs_backward(h["logits"], h["tokens"], h["statistics"], h["grad_logprobs"], h.get("entropy"),
                                   h.get("grad_entropy"), out=h["grad_logits"], stream=on)
        return {"grad_logits": state["grad_logits"]}
    if op == "logprobs":
        nn.token_logprobs(h["logits"], h["tokens"], out=h["out"], stream=on)
    else:
        nn.token_loss(h["logits"], h["tokens"], h["grad_logprobs"], h.get("grad_entropy"), out=h["out"], grad=h["grad_logits"],
                      stream=on)
    return {k: state[k] for k in ("logprobs", "statistics", "entropy", "top_tokens", "top_logprobs", "grad_logits")
            if state.get(k) is not None}


# ---------------------------------------------------------------------------
# what a pass cannot do without, and the results in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "clip":
        shapes = clip_shapes(case)
        return {"bytes": 2 * sum(n * BYTES[d] for n, d in shapes) + 4, "flops": 3 * sum(n for n, _ in shapes)}
    b = BYTES[case["dtype"]]
    if op in ("norm", "norm_grad"):
        n, vectors = case["rows"] * case["cols"], case["cols"] * (4 if case["params"] == "f32" else b)
        if op == "norm":
            return {"bytes": 2 * n * b + 2 * vectors + 8 * case["rows"], "flops": 8 * n}
        return {"bytes": 3 * n * b + 3 * vectors + 8 * case["rows"], "flops": 14 * n}
    n, rows = case["rows"] * case["vocab"], case["rows"]
    per_row = {"logprobs": 16, "logprobs_grad": 16, "loss": 20}[op] + (8 if case["entropy"] and op != "logprobs" else 4 if case["entropy"] else 0)
    return {"bytes": (n * b if op == "logprobs" else 2 * n * b) + rows * (per_row + 8 * case["top"]),
            "flops": n * ({"logprobs": 4, "logprobs_grad": 4, "loss": 8}[op] + (2 if case["entropy"] else 0))}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "clip":
        norm = math.sqrt(math.fsum(float((g.double() ** 2).sum()) for g in s["grads"]))
        by = min(1.0, s["limit"] / norm)
        return {"norm": torch.tensor([norm], dtype=torch.float64), "grads": [f.double() * by for f in s["flat"]]}
    if op in ("norm", "norm_grad"):
        return exact_norm(s) if op == "norm" else exact_norm_grad(s)
    parts = [exact_tokens(s, slice(i, i + step)) for step in [max(1, (1 << 26) // case["vocab"])]
             for i in range(0, case["rows"], step)]
    return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}


def exact_norm(s):
    x = s["x"].double()
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    rstd = torch.rsqrt(var + EPS)
    return {"y": torch.addcmul(s["bias"].double(), (x - mean) * rstd, s["weight"].double()), "statistics": torch.cat([mean, rstd], 1)}


def exact_norm_grad(s):
    """By the chain rule, a link at a time: y = h w + b, h = c r, c = x - mean, r = (mean(c^2) + eps)^(-1/2)."""
    n = s["x"].shape[1]
    grad, w = s["grad"].double(), s["weight"].double()
    mean, r = s["statistics"].double().split(1, 1)
    c = s["x"].double() - mean
    dh = grad * w
    dr = (dh * c).sum(1, keepdim=True)
    dc = dh * r + (-(r ** 3)) * dr * c / n
    return {"grad_x": dc - dc.mean(1, keepdim=True), "grad_weight": torch.einsum("ij,ij->j", grad, c * r),
            "grad_bias": torch.einsum("ij->j", grad)}


def exact_tokens(s, at):
    case = s["case"]
    x, token = s["logits"][at].double(), s["tokens"][at].long()
    rows = torch.arange(len(x), device=x.device)
    empty = (x == -math.inf).all(1)
    y = torch.where(empty[:, None], 0.0, x)  # the rows that hold nothing are set apart below
    lse = torch.logsumexp(y, 1)
    logp = torch.log_softmax(y, 1)
    p = logp.exp()
    entropy = torch.special.entr(p).sum(1)
    entropy[empty] = 0.0
    out = {}
    if case["op"] != "logprobs_grad":
        chosen = logp[rows, token.clamp(min=0)]
        chosen[empty] = -math.inf
        chosen[token < 0] = 0.0
        biggest = x.max(1).values
        log_sum = torch.where(empty, 0.0, lse - torch.where(empty, 0.0, biggest))
        out = {"logprobs": chosen, "statistics": torch.stack([biggest, log_sum], 1)}
        if case["entropy"]:
            out["entropy"] = entropy
    if case["op"] != "logprobs":
        up = s["grad_logprobs"][at].double()
        grad = -up[:, None] * p
        grad[rows, token.clamp(min=0)] += up
        grad[token < 0] = 0.0
        if case["entropy"]:
            grad -= s["grad_entropy"][at].double()[:, None] * p * torch.where(p > 0, logp + entropy[:, None], 0.0)
        grad[empty] = 0.0
        out["grad_logits"] = grad
    if case["top"]:
        k = min(case["top"], case["vocab"])
        # distinct keys: ties go to the lowest index
        order = torch.argsort(-x, dim=1, stable=True)[:, :k]
        out["top_tokens"] = order.int()
        out["top_logprobs"] = torch.where(empty[:, None], -math.inf, logp.gather(1, order))
    return out
