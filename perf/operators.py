"""Cases of the language-model losses: what is measured, and their plain forms.

Three operators of ``pytorch_opt_b200.losses``, each with its gradient:

* ``linear_cross_entropy`` — softmax cross entropy of ``hidden @ weight.T`` over a large
  vocabulary, without the logits as a tensor of the caller's;
* ``linear_distillation`` — the divergence from a teacher's top logits, on the same product;
* ``distillation`` — the same divergence for student logits that are there already.

``own`` selects the side: False computes elementary torch operations in 32 bits (rounded once
to the output's type), True makes the calls a user makes. ``exact`` restates the definitions in
64 bits.

Definitions, for a row t with logits z (z = W h for the linear forms), lse(z) = log sum exp z:

* cross entropy with smoothing s and z-loss c: l = lse(z) - (1 - s) z_y - s mean(z) + c lse(z)^2,
  dl/dz = (1 + 2 c lse(z)) softmax(z) - (1 - s) onehot(y) - s/V; rows whose target is
  ``ignore_index`` count for nothing;
* distillation at temperature a over the entries k of the row whose index is not negative:
  q = softmax(teacher / a), l = a^2 sum_k q_k (log q_k - log softmax(z / a)_{i_k}),
  dl/dz = a (softmax(z / a) - q scattered to i); rows without an entry count for nothing.

``mean`` divides by the number of rows that count.
"""

import math

import torch

own = False

IGNORE = -100
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _case(name, op, grad, dtype, tokens, vocab, dim=0, top=1, masked=0.0, smoothing=0.0, z_loss=0.0, temperature=1.0,
          reduction="mean"):
    """``masked``: the share of rows that count for nothing. ``dim`` 0: logits given."""
    c = dict(op=op, grad=grad, dtype=dtype, tokens=tokens, vocab=vocab, dim=dim, top=top, masked=masked,
             smoothing=smoothing, z_loss=z_loss, temperature=temperature, reduction=reduction)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # Scoring the next token of one sequence with a small model's head: latency.
        _case("ce score 1 token", "ce", False, "bf16", 1, 50257, 768, reduction="none"),
        # Per-token losses of an evaluation batch on an 8B-sized head, a fifth of it padding.
        _case("ce eval 2047x128256", "ce", False, "bf16", 2047, 128256, 4096, masked=0.2, reduction="none"),
        # One training micro-batch of a small model: loss and both gradients.
        _case("ce train 1024x50257", "ce", True, "bf16", 1024, 50257, 768),
        # The head of an 8B-sized model in training.
        _case("ce train 4096x128256", "ce", True, "bf16", 4096, 128256, 4096),
        # Fine-tuning on answers only: over half of the packed tokens are prompt and carry no loss.
        _case("ce tune 8191x32000", "ce", True, "bf16", 8191, 32000, 1024, masked=0.6),
        # Mixed-precision fp16 training with smoothing and z-loss, no size a multiple of a tile.
        _case("ce fp16 1531x32003", "ce", True, "fp16", 1531, 32003, 1280, masked=0.1, smoothing=0.1, z_loss=1e-4),
        # A small model in fp32, as optimizer studies train it.
        _case("ce fp32 500x50257", "ce", True, "fp32", 500, 50257, 768, masked=0.1),
        # Distilling into an 8B-sized head from 64 stored teacher logits a token.
        _case("lin distil 2048x128256", "lin_distil", True, "bf16", 2048, 128256, 4096, top=64, masked=0.05,
              temperature=2.0),
        # The same for a small student, few tokens, more entries.
        _case("lin distil 300x50257", "lin_distil", True, "bf16", 300, 50257, 768, top=128, masked=0.05),
        # One token's divergence and gradient from logits at hand: latency.
        _case("distil 1x50257", "distil", True, "fp32", 1, 50257, top=16, reduction="none"),
        # Student logits of a training batch at hand, bandwidth.
        _case("distil 2048x128256", "distil", True, "bf16", 2048, 128256, top=64, masked=0.05, temperature=2.0),
        # Odd vocabulary and rows that start on no boundary, evaluation only.
        _case("distil eval 777x32003", "distil", False, "fp16", 777, 32003, top=100, masked=0.2, reduction="none"),
    ]


_MOST = 3 * 4096 * 128256 * 4096


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(("ce", "ce", "lin_distil", "distil"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    grad = rng.random() < 0.7
    vocab = _log_int(rng, 1000, 128256)
    dim = 0
    if op != "distil":
        dim = _log_int(rng, 64, 4096)
        if rng.random() < 0.7:
            dim = max(64, dim // 64 * 64)
    most = _MOST // (12 if dtype == "fp32" else 1) // (3 if grad else 1)
    tokens = _log_int(rng, 1, max(1, min(8192, most // (vocab * max(dim, 1)), (1 << 28) // vocab)))
    one_row = tokens == 1
    return _case(None, op, grad, dtype, tokens, vocab, dim, top=1 if op == "ce" else _log_int(rng, 1, 128),
                 masked=0.0 if one_row else rng.choice((0.0, 0.1, 0.5)),
                 smoothing=rng.choice((0.0, 0.1)) if op == "ce" else 0.0,
                 z_loss=rng.choice((0.0, 1e-4)) if op == "ce" else 0.0,
                 temperature=1.0 if op == "ce" else rng.choice((1.0, 2.0)),
                 reduction="mean" if grad and not one_row else "none")


def prepare(case, seed):
    """Inputs on the GPU from the seed. Hidden states lean towards their target's row of the head, so that
    targets are likely by anything between chance and near certainty, as in training."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype, T, V, D, K = TYPES[case["dtype"]], case["tokens"], case["vocab"], case["dim"], case["top"]
    rand = lambda *shape: torch.rand(*shape, generator=g, device=dev)
    randn = lambda *shape: torch.randn(*shape, generator=g, device=dev)
    target = torch.randint(0, V, (T,), generator=g, device=dev)
    counts = rand(T) >= case["masked"]
    counts[0] = True
    s = {"case": case}
    if D:
        weight = (randn(V, D) * 0.02).to(dtype)
        rows = weight[target].float()
        lean = 12 * rand(T, 1) / rows.square().sum(1, keepdim=True)
        hidden = (randn(T, D) + lean * rows).to(dtype)
        s["hidden"], s["weight"] = hidden.requires_grad_(case["grad"]), weight.requires_grad_(case["grad"])
        if case["op"] == "lin_distil":
            teacher = (hidden.detach() + 0.5 * randn(T, D).to(dtype)) @ weight.detach().t()
    else:
        logits = (1.5 * randn(T, V)).to(dtype)
        logits[torch.arange(T, device=dev), target] += (12 * rand(T)).to(dtype)
        s["logits"] = logits.requires_grad_(case["grad"])
        teacher = logits.detach() + 0.5 * randn(T, V).to(dtype)
    if case["op"] == "ce":
        s["target"] = torch.where(counts, target, IGNORE)
    else:
        top, index = teacher.topk(K, dim=1)
        kept = torch.randint((K + 1) // 2, K + 1, (T, 1), generator=g, device=dev)  # a nucleus may hold fewer than K
        gone = (torch.arange(K, device=dev) >= kept) | ~counts[:, None]
        s["index"] = torch.where(gone, -1, index)
        s["teacher"] = top.masked_fill(gone, math.nan)  # what is stored beside no entry is anything
    return s


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from pytorch_opt_b200 import losses

    c = s["case"]
    if c["op"] == "ce":
        inputs = {"dhidden": s["hidden"], "dweight": s["weight"]}
        loss = losses.linear_cross_entropy(s["hidden"], s["weight"], s["target"], ignore_index=IGNORE,
                                           label_smoothing=c["smoothing"], z_loss=c["z_loss"],
                                           reduction=c["reduction"])
    elif c["op"] == "lin_distil":
        inputs = {"dhidden": s["hidden"], "dweight": s["weight"]}
        loss = losses.linear_distillation(s["hidden"], s["weight"], s["index"], s["teacher"],
                                          temperature=c["temperature"], reduction=c["reduction"])
    else:
        inputs = {"dlogits": s["logits"]}
        loss = losses.distillation(s["logits"], s["index"], s["teacher"], temperature=c["temperature"],
                                   reduction=c["reduction"])
    if not c["grad"]:
        return {"loss": loss}
    up = torch.ones_like(loss) if c["reduction"] == "none" else None
    return {"loss": loss.detach(), **dict(zip(inputs, torch.autograd.grad(loss, tuple(inputs.values()), up)))}


@torch.no_grad()
def _run_plain(s):
    c = s["case"]
    linear = c["dim"] > 0
    if linear:
        h, w = s["hidden"].float(), s["weight"].float()
        z = h @ w.t()
    else:
        z = s["logits"].float()
    if c["op"] == "ce":
        loss, dz = _plain_ce(z, s["target"], c)
    else:
        loss, dz = _plain_distil(z, s["index"], s["teacher"].float(), c)
    if not c["grad"]:
        return {"loss": loss}
    if not linear:
        return {"loss": loss, "dlogits": dz.to(s["logits"].dtype)}
    return {"loss": loss, "dhidden": (dz @ w).to(s["hidden"].dtype), "dweight": (dz.t() @ h).to(s["weight"].dtype)}


def _softmax(z):
    """(log sum exp, softmax) over the last axis."""
    m = z.max(1, keepdim=True).values
    e = (z - m).exp_()
    total = e.sum(1, keepdim=True)
    return (m + total.log())[:, 0], e.div_(total)


def _reduced(loss, counts, reduction):
    """The loss, and what each row's gradient is multiplied by."""
    loss = torch.where(counts, loss, torch.zeros_like(loss))
    if reduction == "none":
        return loss, counts.float()
    n = counts.sum().clamp(min=1).float()
    return loss.sum() / n, counts.float() / n


def _plain_ce(z, target, c):
    counts = target != IGNORE
    at = target.clamp(min=0)[:, None]
    lse, p = _softmax(z)
    s, zc = c["smoothing"], c["z_loss"]
    loss = lse - (1 - s) * z.gather(1, at)[:, 0] - s * z.mean(1) + zc * lse * lse
    loss, each = _reduced(loss, counts, c["reduction"])
    if not c["grad"]:
        return loss, None
    dz = p.mul_((1 + 2 * zc * lse)[:, None]).sub_(s / z.shape[1])
    dz.scatter_add_(1, at, torch.full_like(at, -(1 - s), dtype=dz.dtype))
    return loss, dz.mul_(each[:, None])


def _plain_distil(z, index, teacher, c):
    a = c["temperature"]
    there = index >= 0
    counts = there.any(1)
    at = index.clamp(min=0)
    t = torch.where(there, teacher / a, torch.full_like(teacher, -torch.inf))
    m = torch.where(counts, t.max(1).values, torch.zeros_like(t[:, 0]))[:, None]
    e = (t - m).exp()
    total = torch.where(counts, e.sum(1), torch.ones_like(t[:, 0]))[:, None]
    q = e / total
    logq = torch.where(there, t - m - total.log(), torch.zeros_like(t))
    z = z / a
    lse, p = _softmax(z)
    loss = a * a * (q * (logq - z.gather(1, at) + lse[:, None])).sum(1)
    loss, each = _reduced(loss, counts, c["reduction"])
    if not c["grad"]:
        return loss, None
    dz = p.scatter_add_(1, at, -q)
    return loss, dz.mul_(a * each[:, None])


def work(case):
    T, V, D, K = case["tokens"], case["vocab"], case["dim"], case["top"]
    size = 4 if case["dtype"] == "fp32" else 2
    rows = max(1, round(T * (1 - case["masked"])))  # the others need not be read
    labels = 8 * T if case["op"] == "ce" else (8 + size) * T * K
    if D:
        data = size * (rows * D + V * D)  # read; the gradients have the same shapes, masked rows written too
        data += size * (T * D + V * D) if case["grad"] else 0
        flops = (3 if case["grad"] else 1) * 2 * rows * V * D
    else:
        data = size * rows * V + (size * T * V if case["grad"] else 0)
        flops = (6 if case["grad"] else 4) * rows * V
    return {"bytes": data + labels + 4 * (T if case["reduction"] == "none" else 1), "flops": flops}


@torch.no_grad()
def exact(case, seed):
    """The definitions in 64 bits, by log-probabilities and dense target distributions."""
    s = prepare(case, seed)
    linear = case["dim"] > 0
    z = s["hidden"].double() @ s["weight"].double().t() if linear else s["logits"].double()
    T, V = z.shape
    a = case["temperature"]
    goal = torch.zeros_like(z)  # the distribution that each row is held to
    if case["op"] == "ce":
        counts = s["target"] != IGNORE
        rows = counts.nonzero()[:, 0]
        goal[rows, s["target"][rows]] = 1 - case["smoothing"]
        if case["smoothing"]:
            goal[rows] += case["smoothing"] / V
        less = torch.zeros(T, dtype=torch.float64, device=z.device)
    else:
        counts = (s["index"] >= 0).any(1)
        rows, at = (s["index"] >= 0).nonzero(as_tuple=True)
        t = torch.full(s["index"].shape, -math.inf, dtype=torch.float64, device=z.device)
        t[rows, at] = s["teacher"].double()[rows, at] / a
        logq = t - torch.logsumexp(t, 1, keepdim=True)
        q = logq.exp()
        goal[rows, s["index"][rows, at]] = q[rows, at]
        less = torch.where(s["index"] >= 0, q * logq, torch.zeros_like(q)).sum(1)
    lse = torch.logsumexp(z / a, 1)
    logp = z / a - lse[:, None]
    loss = a * a * (less - (goal * logp).sum(1)) + case["z_loss"] * lse**2
    loss = torch.where(counts, loss, torch.zeros_like(loss))
    n = 1 if case["reduction"] == "none" else max(1, int(counts.sum()))
    out = {"loss": loss if case["reduction"] == "none" else loss.sum() / n}
    if not case["grad"]:
        return out
    dz = logp.exp_().mul_(1 + 2 * case["z_loss"] * lse[:, None]).sub_(goal).mul_(a / n)
    dz[~counts] = 0
    del goal
    if not linear:
        return {**out, "dlogits": dz}
    return {**out, "dhidden": dz @ s["weight"].double(), "dweight": dz.t() @ s["hidden"].double()}
