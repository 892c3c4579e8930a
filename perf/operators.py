"""The operators of a language model's output head that are measured, and what they are measured on.

* ``xent``: ``ops.loss.linear_cross_entropy`` -- softmax cross entropy of ``x @ w.T`` over a
  large vocabulary, and its gradients, without the logits ever being kept.
* ``distill``: ``ops.loss.linear_distill`` -- the divergence of the same softmax from a
  teacher's top logits, and its gradients.
* ``gemv``: ``ops.gemv.gemv_w4`` -- the products of one or a few token vectors with a 4-bit
  weight with group scales, as a node answers with such a head.

``run`` computes each in plain 32-bit torch operations, or calls the framework where ``own``
is true; ``exact`` computes them from their definitions in 64 bits.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
IGNORE = -100  # the target of a token that has no loss

# no drawn case costs more than the largest listed one
MOST_PRODUCTS = 8192 * 4096 * 131072  # tokens x hidden x vocab
MOST_WEIGHTS = 131072 * 8192          # out x inp of a 4-bit weight


def listed():
    return [
        # one small projection of one token: latency is all there is
        dict(name="gemv_token_small", op="gemv", dtype="bf16", rows=1, out=1024, inp=1024, group=128, zeros=False),
        # one token through a large square layer
        dict(name="gemv_token", op="gemv", dtype="bf16", rows=1, out=8192, inp=8192, group=128, zeros=False),
        # one token's logits over a large vocabulary, asymmetric codes
        dict(name="gemv_vocab", op="gemv", dtype="fp16", rows=1, out=131072, inp=4096, group=64, zeros=True),
        # a few tokens at once, sizes that fill no tile, the smallest group
        dict(name="gemv_few_ragged", op="gemv", dtype="fp16", rows=5, out=10001, inp=5152, group=32, zeros=True),
        # the largest decode batch
        dict(name="gemv_batch", op="gemv", dtype="bf16", rows=64, out=16384, inp=16384, group=128, zeros=False),
        # a step on a handful of tokens and a small vocabulary: launches count
        dict(name="xent_small", op="xent", dtype="bf16", tokens=48, hidden=512, vocab=1000, masked=0.0,
             reduction="mean", grad=True),
        # an ordinary training step
        dict(name="xent_step", op="xent", dtype="bf16", tokens=4096, hidden=4096, vocab=32768, masked=0.0,
             reduction="mean", grad=True),
        # a training step over a large vocabulary
        dict(name="xent_large", op="xent", dtype="bf16", tokens=8192, hidden=4096, vocab=131072, masked=0.0,
             reduction="mean", grad=True),
        # tuning on answers only: most tokens are prompt and have no loss; losses weighted by token
        dict(name="xent_answers", op="xent", dtype="fp16", tokens=6001, hidden=2560, vocab=50021, masked=0.6,
             reduction="none", grad=True),
        # evaluation: the loss of every token, no gradient, odd sizes
        dict(name="xent_eval", op="xent", dtype="fp16", tokens=1777, hidden=1536, vocab=50021, masked=0.1,
             reduction="none", grad=False),
        # distillation from a teacher's 64 top logits
        dict(name="distill_step", op="distill", dtype="bf16", tokens=2048, hidden=2048, vocab=65536, topk=64,
             temperature=2.0, absent=0.0, reduction="mean", grad=True),
        # lists of different lengths, some of them empty
        dict(name="distill_ragged", op="distill", dtype="fp16", tokens=333, hidden=1288, vocab=50021, topk=100,
             temperature=1.0, absent=0.3, reduction="sum", grad=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gemv", "xent", "distill"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "gemv":
        group = rng.choice([32, 64, 128])
        while True:
            out, inp = _log(rng, 256, 131072), max(1, _log(rng, 256, 16384) // group) * group
            if out * inp <= MOST_WEIGHTS:
                break
        return dict(op=op, dtype=dtype, rows=_log(rng, 1, 64), out=out, inp=inp, group=group,
                    zeros=rng.random() < 0.5)
    while True:
        tokens, vocab = _log(rng, 1, 8192), _log(rng, 500, 262144)
        hidden = _log(rng, 64, 8192)
        if rng.random() < 0.8:  # most widths are multiples of 8
            hidden = max(8, hidden // 8 * 8)
        if tokens * hidden * vocab <= MOST_PRODUCTS and vocab * hidden <= 131072 * 4096:
            break
    case = dict(op=op, dtype=dtype, tokens=tokens, hidden=hidden, vocab=vocab,
                reduction=rng.choice(["mean", "sum", "none"]), grad=rng.random() < 0.75)
    if op == "xent":
        case.update(masked=rng.choice([0.0, 0.1, 0.6]))
    else:
        case.update(topk=_log(rng, 1, 128), temperature=rng.choice([1.0, 2.0, 0.7]), absent=rng.choice([0.0, 0.3]))
    return case


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    if case["op"] == "gemv":
        m, n, k, group = case["rows"], case["out"], case["inp"], case["group"]
        # codes as a quantizer of normal weights gives them, two to a byte, the lower first
        code = (torch.randn((n, k), device="cuda", generator=g, dtype=torch.float16) * 2.7 + 8).round_().clamp_(0, 15)
        code = code.to(torch.uint8)
        zeros = torch.randint(5, 11, (n, k // group), device="cuda", generator=g, dtype=torch.uint8)
        scales = (k ** -0.5 / 2.7 * (0.5 + torch.rand((n, k // group), device="cuda", generator=g))).to(dt)
        return dict(case=case, x=randn(m, k).to(dt), codes=code[:, 0::2] | (code[:, 1::2] << 4), scales=scales,
                    zeros=zeros if case["zeros"] else None)

    n, d, v = case["tokens"], case["hidden"], case["vocab"]
    w = randn(v, d).mul_(d ** -0.5).to(dt)
    x = randn(n, d)
    # how sure the model is of the right token: from not at all to nearly certain
    sure = torch.rand((n, 1), device="cuda", generator=g) * (1.2 * math.log(v))
    state = dict(case=case, w=w, upstream=torch.rand(n, device="cuda", generator=g) + 0.5)
    if case["op"] == "xent":
        target = torch.randint(0, v, (n,), device="cuda", generator=g)
        x += sure * w[target].float()
        state["target"] = torch.where(torch.rand(n, device="cuda", generator=g) < case["masked"], IGNORE, target)
    else:
        topk = min(case["topk"], v)
        first = torch.randint(0, v, (n, 1), device="cuda", generator=g)
        gaps = torch.randint(1, max(2, v // topk), (n, topk), device="cuda", generator=g)
        ids = (first + gaps.cumsum(1)) % v  # distinct in a row
        state["logits"] = randn(n, topk).mul_(3).sort(1, descending=True).values
        x += sure * w[ids[:, 0]].float()
        length = torch.randint(0, topk + 1, (n, 1), device="cuda", generator=g)
        cut = torch.rand((n, 1), device="cuda", generator=g) < case["absent"]
        state["ids"] = torch.where(cut & (torch.arange(topk, device="cuda") >= length), -1, ids)
    state["x"] = x.to(dt)
    if case["grad"]:
        state["x"].requires_grad_()
        state["w"].requires_grad_()
    return state


def run(state):
    case = state["case"]
    if case["op"] == "gemv":
        return _gemv_own(state) if own else _gemv_plain(state)
    return _loss_own(state) if own else _loss_plain(state)


def _gemv_own(s):
    from triton_kubernetes_amd.ops.gemv import gemv_w4

    return gemv_w4(s["x"], s["codes"], s["scales"], s["zeros"])


def _loss_own(s):
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy, linear_distill

    case = s["case"]
    if case["op"] == "xent":
        loss = linear_cross_entropy(s["x"], s["w"], s["target"], ignore_index=IGNORE, reduction=case["reduction"])
    else:
        loss = linear_distill(s["x"], s["w"], s["ids"], s["logits"], temperature=case["temperature"],
                              reduction=case["reduction"])
    if not case["grad"]:
        return dict(loss=loss)
    upstream = s["upstream"] if case["reduction"] == "none" else None
    dx, dw = torch.autograd.grad(loss, (s["x"], s["w"]), upstream)
    return dict(loss=loss.detach(), dx=dx, dw=dw)


def _gemv_plain(s):
    n, groups = s["scales"].shape
    code = torch.stack((s["codes"] & 15, s["codes"] >> 4), 2).reshape(n, groups, -1).float()
    zero = 8.0 if s["zeros"] is None else s["zeros"].float()[:, :, None]
    w = ((code - zero) * s["scales"].float()[:, :, None]).reshape(n, -1)
    return (s["x"].float() @ w.T).to(s["x"].dtype)


def _loss_plain(s):
    case = s["case"]
    with torch.no_grad():
        x, w = s["x"].float(), s["w"].float()
        t = case.get("temperature", 1.0)
        z = (x @ w.T) / t
        top = z.max(1, keepdim=True).values
        lse = top + (z - top).exp().sum(1, keepdim=True).log()
        if case["op"] == "xent":
            ids = s["target"][:, None]
            there = ids != IGNORE
            p = there.float()
        else:
            ids = s["ids"]
            there = ids >= 0
            y = torch.where(there, s["logits"] / t, -math.inf)
            y = torch.exp(y - y.max(1, keepdim=True).values)
            y = torch.where(there, y, 0.0)
            p = y / y.sum(1, keepdim=True).clamp_min(1e-30)
        ids = torch.where(there, ids, 0)
        rows = there.any(1)
        logp = torch.where(p > 0, p, 1.0).log()
        loss = t * t * (p * (logp - z.gather(1, ids) + lse)).sum(1)
        if case["reduction"] == "none":
            total, up = loss, s["upstream"]
        elif case["reduction"] == "sum":
            total, up = loss.sum(), torch.ones_like(loss)
        else:
            count = rows.sum().clamp_min(1)
            total, up = loss.sum() / count, torch.ones_like(loss) / count
        if not case["grad"]:
            return dict(loss=total)
        dz = (z - lse).exp().scatter_add_(1, ids, -p)
        dz *= (up * rows * t)[:, None]
        return dict(loss=total, dx=(dz @ w).to(s["x"].dtype), dw=(dz.T @ x).to(s["w"].dtype))


def work(case):
    if case["op"] == "gemv":
        m, n, k, groups = case["rows"], case["out"], case["inp"], case["inp"] // case["group"]
        return {"bytes": n * k / 2 + n * groups * (3 if case["zeros"] else 2) + 2 * m * (k + n), "flops": 2 * m * n * k}
    n, d, v = case["tokens"], case["hidden"], case["vocab"]
    kept = n * (1 - case.get("masked", 0.0))  # tokens that have a loss
    directions = 2 if case["grad"] else 1
    lists = n * (8 if case["op"] == "xent" else 12 * case["topk"])
    # the logits, and with a gradient the two products with their derivative
    return {"bytes": directions * 2 * (n + v) * d + lists, "flops": (6 if case["grad"] else 2) * kept * d * v}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "gemv":
        out, groups = s["scales"].shape
        per = case["group"] // 2
        c = s["codes"].view(out, groups, per)
        zero = torch.full((out, groups, 1), 8.0, dtype=torch.float64, device="cuda")
        if s["zeros"] is not None:
            zero = s["zeros"].double().unsqueeze(-1)
        x = s["x"].double().view(-1, groups, per, 2)
        y = torch.zeros((x.shape[0], out), dtype=torch.float64, device="cuda")
        for g in range(groups):  # a group of columns at a time
            low, high = (c[:, g] % 16).double() - zero[:, g], (c[:, g] // 16).double() - zero[:, g]
            y += (x[:, g, :, 0] @ low.T + x[:, g, :, 1] @ high.T) * s["scales"][:, g].double()
        return y
    x = s["x"].detach().double().requires_grad_(case["grad"])
    w = s["w"].detach().double().requires_grad_(case["grad"])
    t = case.get("temperature", 1.0)
    logq = torch.log_softmax(x @ w.T / t, dim=1)
    if case["op"] == "xent":
        has = s["target"] != IGNORE
        loss = torch.where(has, -logq.gather(1, s["target"].clamp_min(0)[:, None])[:, 0], 0.0)
    else:
        listed_, ids = s["ids"] >= 0, s["ids"].clamp_min(0)
        has = listed_.any(1)
        scores = (s["logits"].double() / t).masked_fill(~listed_, -1e300)
        p = torch.softmax(scores, dim=1) * listed_
        loss = t ** 2 * (torch.special.xlogy(p, p) - p * logq.gather(1, ids)).sum(1)
    if case["reduction"] == "mean":
        out = loss.sum() / max(1, int(has.sum()))
    else:
        out = loss.sum() if case["reduction"] == "sum" else loss
    if not case["grad"]:
        return dict(loss=out)
    dx, dw = torch.autograd.grad(out, (x, w), s["upstream"].double() if case["reduction"] == "none" else None)
    return dict(loss=out.detach(), dx=dx, dw=dw)
