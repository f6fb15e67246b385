"""The vocabulary's two ends and the gradient norm of a training step: what
their cases are, their plain forms, and what they have to move.

Three operators, as the language models here use them in one step:

  embedding      token ids -> scaled rows of a table; its gradient sums the
                 rows of one token (axon.ops.embedding)
  cross entropy  logits and labels -> loss and the logits' gradient
                 (axon.ops.cross_entropy)
  clipping       the norm over all gradients, and the gradients scaled by it:
                 by itself (axon.optim.clip_grad_norm_), or inside the
                 optimizer's step (FusedAdamW(max_grad_norm=))
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
LR, BETAS, EPS, DECAY, STEP = 3e-4, (0.9, 0.95), 1e-8, 0.1, 10


def listed():
    return [
        # One decoding step of a batch of 8: a few rows of a large table.
        dict(name="embed decode bf16", op="embed", tokens=8, vocab=128256,
             dim=2048, dtype="bf16", scale=1.0, padded=0.0, train=False),
        # A small model of odd sizes, half of the batch padding.
        dict(name="embed odd fp32", op="embed", tokens=1999, vocab=5003,
             dim=509, dtype="fp32", scale=22.5, padded=0.5, train=True),
        # The encoder's pretraining batch: 64 sequences of 128 tokens.
        dict(name="embed encoder bf16", op="embed", tokens=8192, vocab=30522,
             dim=1024, dtype="bf16", scale=1.0, padded=0.1, train=True),
        # The large decoder's batch: 8 sequences of 4096 tokens.
        dict(name="embed decoder bf16", op="embed", tokens=32768,
             vocab=128256, dim=4096, dtype="bf16", scale=64.0, padded=0.0,
             train=True),
        # An image classifier's loss: short rows, smoothed labels.
        dict(name="loss classes fp32", op="loss", rows=256, classes=1000,
             dtype="fp32", ignored=0.0, smoothing=0.1, train=True),
        # Scoring one sequence: the loss of each token, nothing to train.
        dict(name="loss score fp16", op="loss", rows=511, classes=32003,
             dtype="fp16", ignored=0.02, smoothing=0.0, train=False),
        # The encoder's masked tokens: 85 of 100 rows carry no label.
        dict(name="loss masked bf16", op="loss", rows=8192, classes=30522,
             dtype="bf16", ignored=0.85, smoothing=0.0, train=True),
        # The large decoder's loss, two sequences of 4096 tokens.
        dict(name="loss decoder bf16", op="loss", rows=8192, classes=128256,
             dtype="bf16", ignored=0.0002, smoothing=0.0, train=True),
        # As many gradients and values as the digit classifier has: latency.
        dict(name="clip digits fp32", op="clip", tensors=8, values=21840,
             dtype="fp32", ratio=2.5),
        # As many as the image classifier has, below the norm's bound.
        dict(name="clip classifier fp32", op="clip", tensors=161,
             values=25557032, dtype="fp32", ratio=0.5),
        # As many as the encoder has.
        dict(name="clip encoder bf16", op="clip", tensors=298,
             values=335174458, dtype="bf16", ratio=4.0),
        # AdamW's step on clipped gradients, as many as the 1B decoder has.
        dict(name="step decoder bf16", op="step", tensors=147,
             values=1498482688, dtype="bf16", ratio=4.0),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["embed", "embed", "loss", "loss", "clip", "step"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "embed":
        train = rng.random() < 0.75
        return dict(op=op, tokens=_log(rng, 1, 32768),
                    vocab=_log(rng, 64, 128256),
                    dim=_log(rng, 16, 4096 if dtype != "fp32" else 2048),
                    dtype=dtype, scale=rng.choice([1.0, 8.0, 22.5]),
                    padded=rng.choice([0.0, 0.1, 0.6]), train=train)
    if op == "loss":
        classes = _log(rng, 10, 131072)
        rows = max(1, min(_log(rng, 1, 65536), (1 << 29) // classes))
        return dict(op=op, rows=rows, classes=classes, dtype=dtype,
                    ignored=rng.choice([0.0, 0.1, 0.85]),
                    smoothing=rng.choice([0.0, 0.0, 0.1]),
                    train=rng.random() < 0.75)
    if op == "step":
        dtype = rng.choice(["bf16", "fp32"])
    return dict(op=op, tensors=_log(rng, 1, 400),
                values=_log(rng, 1000, 300_000_000), dtype=dtype,
                ratio=rng.choice([0.5, 2.5, 20.0]))


def _shares(case):
    """How many values each tensor has: many small ones (norms, biases),
    some large ones, odd ones among them."""
    n, total = case["tensors"], case["values"]
    rng = random.Random(n * 1000003 + total)
    weights = [math.exp(rng.gauss(0.0, 2.5)) for _ in range(n)]
    all_ = sum(weights)
    sizes = [max(1, int(total * w / all_)) for w in weights]
    sizes[sizes.index(max(sizes))] += max(0, total - sum(sizes))
    return sizes


def _starts(sizes):
    """Where each tensor starts in one buffer: on borders of 16 values, as
    separate tensors would be aligned; what lies between holds zeros."""
    at, starts = 0, []
    for n in sizes:
        starts.append(at)
        at += -(-n // 16) * 16
    return starts, at


def _zipf(case):
    """The share of each token in a text, the most frequent one first."""
    rank = torch.arange(case["vocab"], dtype=torch.float64)
    p = 1.0 / (rank + 2.7)
    return p / p.sum()


def _texts(case, g):
    """Token ids as frequent as a text's words, padding (token 0) among
    them."""
    p = _zipf(case).to("cuda")
    u = torch.rand(case["tokens"], generator=g, device="cuda",
                   dtype=torch.float64)
    rank = torch.searchsorted(torch.cumsum(p, 0), u)
    rank = rank.clamp_(max=case["vocab"] - 1)
    token = torch.randperm(case["vocab"], generator=g, device="cuda")[rank]
    pad = torch.rand(case["tokens"], generator=g, device="cuda")
    return torch.where(pad < case["padded"], 0, token)


def _flat(n, std, dtype, g):
    return (torch.randn(n, generator=g, device="cuda", dtype=dtype)
            * std)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] == "embed":
        state["ids"] = _texts(case, g)
        table = torch.randn(case["vocab"], case["dim"], generator=g,
                            device="cuda", dtype=dtype).mul_(0.02)
        state["table"] = table.requires_grad_(case["train"])
        # Padding has a meaning only where it occurs.
        state["padding"] = 0 if case["padded"] else None
        if case["train"]:
            state["dout"] = _flat((case["tokens"], case["dim"]), 0.01, dtype,
                                  g)
        return state
    if case["op"] == "loss":
        rows, classes = case["rows"], case["classes"]
        logits = torch.randn(rows, classes, generator=g, device="cuda",
                             dtype=dtype).mul_(2.0)
        target = torch.randint(classes, (rows,), generator=g, device="cuda")
        # A trained model gives most labels a high score.
        known = torch.rand(rows, generator=g, device="cuda") < 0.7
        logits[torch.arange(rows, device="cuda"), target] += \
            torch.where(known, 8.0, 0.0).to(dtype)
        dropped = torch.rand(rows, generator=g, device="cuda")
        target = torch.where(dropped < case["ignored"], -100, target)
        state["target"] = target
        state["logits"] = logits.requires_grad_(case["train"])
        return state
    sizes = _shares(case)
    starts, end = _starts(sizes)
    # Gradients whose norm is `ratio` times the bound of 1.
    std = case["ratio"] / math.sqrt(sum(sizes))
    real = torch.zeros(end, dtype=torch.bool, device="cuda")
    for at, n in zip(starts, sizes):
        real[at:at + n] = True
    fresh = _flat(end, std, dtype, g).mul_(real)
    if case["op"] == "clip":
        # What the backward pass leaves in the gradients' buffers each step.
        state["fresh"] = fresh
        state["grads"] = torch.zeros_like(fresh)
        params = []
        for at, n in zip(starts, sizes):
            p = torch.nn.Parameter(torch.empty(n, device="cuda", dtype=dtype))
            p.grad = state["grads"][at:at + n]
            params.append(p)
        state["params"] = params
        return state
    state["grads"] = fresh
    state["weights"] = _flat(end, 0.02, dtype, g).mul_(real)
    state["m"] = _flat(end, std, dtype, g).mul_(real)
    state["v"] = _flat(end, std, dtype, g).square_().mul_(real)
    state["step"] = STEP
    if own:  # the optimizer that a program keeps from step to step
        from axon.optim import FusedAdamW

        params = []
        for at, n in zip(starts, sizes):
            p = torch.nn.Parameter(state["weights"][at:at + n])
            p.grad = state["grads"][at:at + n]
            params.append(p)
        opt = FusedAdamW(params, lr=LR, betas=BETAS, eps=EPS,
                         weight_decay=DECAY, max_grad_norm=1.0)
        for p, at, n in zip(params, starts, sizes):
            opt.state[p] = {"step": torch.tensor(float(STEP)),
                            "exp_avg": state["m"][at:at + n],
                            "exp_avg_sq": state["v"][at:at + n]}
        state["optimizer"] = opt
    return state


def _embed(state):
    case, ids, table = state["case"], state["ids"], state["table"]
    if own:
        from axon.ops import embedding

        out = embedding(ids, table, scale=case["scale"],
                        padding_idx=state["padding"])
        if not case["train"]:
            return {"out": out}
        (grad,) = torch.autograd.grad(out, table, state["dout"])
        return {"out": out.detach(), "grad": grad}
    table = table.detach()
    out = (table[ids].float() * case["scale"]).to(table.dtype)
    if not case["train"]:
        return {"out": out}
    grad = torch.zeros(table.shape, device="cuda")
    grad.index_add_(0, ids, state["dout"].float())
    grad *= case["scale"]
    if state["padding"] is not None:
        grad[state["padding"]] = 0
    return {"out": out, "grad": grad.to(table.dtype)}


def _loss(state):
    case, logits, target = state["case"], state["logits"], state["target"]
    eps, classes = case["smoothing"], case["classes"]
    if own:
        from axon.ops import cross_entropy

        if not case["train"]:
            return {"loss": cross_entropy(logits, target, reduction="none",
                                          label_smoothing=eps)}
        loss = cross_entropy(logits, target, label_smoothing=eps)
        (grad,) = torch.autograd.grad(loss, logits)
        return {"loss": loss.detach(), "grad": grad}
    x = logits.detach().float()
    valid = target != -100
    at = torch.where(valid, target, 0)[:, None]
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    lse = top + torch.log(total)
    loss = (1 - eps) * (lse - x.gather(1, at))
    if eps:
        loss = loss + eps * (lse - x.mean(1, keepdim=True))
    loss = torch.where(valid, loss[:, 0], 0.0)
    if not case["train"]:
        return {"loss": loss}
    count = valid.sum()
    grad = e / total
    if eps:
        grad -= eps / classes
    grad.scatter_add_(1, at, torch.full_like(total, eps - 1.0))
    grad *= torch.where(valid, 1.0 / count, 0.0)[:, None]
    return {"loss": loss.sum() / count, "grad": grad.to(logits.dtype)}


def _norm(grads):
    total = grads.float().square().sum(dtype=torch.float64).sqrt()
    return total.float()


def _clip(state):
    grads = state["grads"]
    grads.copy_(state["fresh"])
    if own:
        from axon.optim import clip_grad_norm_

        norm = clip_grad_norm_(state["params"], 1.0)
        return {"norm": norm, "grads": grads}
    norm = _norm(grads)
    factor = (1.0 / (norm + 1e-6)).clamp(max=1.0)
    grads.copy_(grads.float() * factor)
    return {"norm": norm, "grads": grads}


def _step(state):
    got = {k: state[k] for k in ("weights", "m", "v")}
    if own:
        opt = state["optimizer"]
        opt.step()
        return dict(got, norm=opt.grad_norm)
    grads = state["grads"]
    norm = _norm(grads)
    factor = (1.0 / (norm + 1e-6)).clamp(max=1.0)
    state["step"] += 1
    b1, b2 = BETAS
    c1, c2 = 1 - b1 ** state["step"], 1 - b2 ** state["step"]
    g = grads.float() * factor
    m = state["m"].float().mul_(b1).add_(g, alpha=1 - b1)
    state["m"].copy_(m)
    v = state["v"].float().mul_(b2).add_(g.square_(), alpha=1 - b2)
    state["v"].copy_(v)
    update = m.div_(c1).div_(v.sqrt_().div_(math.sqrt(c2)).add_(EPS))
    w = state["weights"].float().mul_(1 - LR * DECAY)
    state["weights"].copy_(w.sub_(update, alpha=LR))
    return dict(got, norm=norm)


def run(state):
    return {"embed": _embed, "loss": _loss, "clip": _clip,
            "step": _step}[state["case"]["op"]](state)


def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] == "embed":
        n, dim, vocab = case["tokens"], case["dim"], case["vocab"]
        # Each row of the table that the text names is read once.
        p = _zipf(case) * (1 - case["padded"])
        p[0] += case["padded"]
        named = float((1 - (1 - p) ** n).sum())
        moved = 8 * n + size * dim * (named + n)
        if case["train"]:
            moved += size * dim * (n + vocab)
        return {"bytes": moved, "flops": n * dim * (2 if case["train"] else 1)}
    if case["op"] == "loss":
        rows, classes = case["rows"], case["classes"]
        # A row without a label is not read; its gradient is zeros.
        read = rows * (1 - case["ignored"]) * classes
        moved = 8 * rows + size * read + 4 * (1 if case["train"] else rows)
        if case["train"]:
            moved += size * rows * classes
        return {"bytes": moved,
                "flops": read * (7 if case["train"] else 4)}
    n = sum(_shares(case))
    if case["op"] == "clip":
        # The fresh gradients arrive (read, written); the norm reads them;
        # only a norm above the bound reads and writes them again.
        passes = 3 if case["ratio"] < 1 else 5
        return {"bytes": passes * size * n, "flops": 3 * n}
    # The norm reads the gradients; the step reads them with the weights and
    # the two moments, and writes those three.
    return {"bytes": 8 * size * n, "flops": 16 * n}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "embed":
        ids = state["ids"]
        table = state["table"].detach()
        out = table[ids].double() * case["scale"]
        if not case["train"]:
            return {"out": out}
        d = state["dout"].double() * case["scale"]
        if state["padding"] is not None:
            d = d * (ids != state["padding"])[:, None]
        # The sum of a token's rows in the order of the text.
        order = torch.argsort(ids, stable=True)
        grad = torch.zeros(table.shape, dtype=torch.float64, device="cuda")
        grad.index_put_((ids[order],), d[order], accumulate=True)
        return {"out": out, "grad": grad}
    if case["op"] == "loss":
        x = state["logits"].detach().double()
        target, eps = state["target"], case["smoothing"]
        logp = x.sub_(torch.logsumexp(x, 1, keepdim=True))
        # The cross entropy of the smoothed label's distribution q with the
        # model's p, and its gradient p - q.
        valid = target >= 0
        rows = valid.nonzero()[:, 0]
        picked = logp[rows, target[rows]]
        loss = torch.zeros(len(target), dtype=torch.float64, device="cuda")
        loss[rows] = -((1 - eps) * picked + eps * logp[rows].mean(1)
                       if eps else picked)
        if not case["train"]:
            return {"loss": loss}
        grad = logp.exp_()
        if eps:
            grad -= eps / case["classes"]
        grad[rows, target[rows]] -= 1 - eps
        grad[~valid] = 0
        # Without any label the mean is 0/0; the gradient stays zeros.
        return {"loss": loss.sum() / len(rows),
                "grad": grad.div_(max(1, len(rows)))}
    fresh = state["fresh"] if case["op"] == "clip" else state["grads"]
    g = fresh.double()
    norm = torch.linalg.vector_norm(g)
    g *= min(1.0, 1.0 / (float(norm) + 1e-6))
    if case["op"] == "clip":
        return {"norm": norm, "grads": g}
    b1, b2 = BETAS
    m = torch.lerp(g, state["m"].double(), b1)
    v = torch.lerp(g.square(), state["v"].double(), b2)
    del g
    scale = math.sqrt(1 - b2 ** (STEP + 1)) / (1 - b1 ** (STEP + 1))
    w = state["weights"].double() * (1 - LR * DECAY)
    w -= LR * scale * m / (v.sqrt() + EPS * math.sqrt(1 - b2 ** (STEP + 1)))
    return {"weights": w, "m": m, "v": v, "norm": norm}
