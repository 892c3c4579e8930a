"""How far the output head's losses may be from 64 bits at any size: bounds that follow how errors
add up, instead of the worst case of every addition.

A logit is a sum of D exact products in fp32.  A partial sum of k of them is a random walk, about
sqrt(k) |x||w| / D, on a line to k z / D; each addition is off by at most STEP of it.  The squares add
up to STEP^2 (|x|^2 |w|^2 / 2 + D z^2 / 3), of which ``far`` is 8 times the root.  The sum of
exponentials has positive terms: a tile's 256 entries and the tiles are joined in at most 80 + V/8192
additions in a row, and with 2^-20 for exp2 and log2 that is ``off``, common to a row's probabilities.

The derivative of a logit is rounded to 16 bits (u, half a step; in fp16 2^-25 of a span of 2^15 at
the least), where the logits are kept it has their rounding too.  These are independent from entry to
entry: an element of a gradient is off by at most 6 times their root mean square, a row by twice
it (rows of few elements, each error at its largest), all of it by 0.8 times it, where spread
roundings have 0.58; and by the rounding of the result, and by what ``off`` does to it as a whole.
"""

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
STEP = 2.0 ** -23


def exact(x, w, ids, p, t, g):
    """(losses, dx, dw, what their bounds need) of ``sum(g * loss)`` in 64 bits.  ``ids [N, K]`` of which those
    below 0 are none, ``p [N, K]`` their probabilities."""
    a, b, g = x.double(), w.double(), g.double()[:, None]
    z = a @ b.T / t
    lse = torch.logsumexp(z, 1, keepdim=True)
    used, at = torch.where(ids >= 0, p.double(), 0.0), ids.clamp_min(0)
    has = (ids >= 0).any(1, keepdim=True)
    terms = torch.special.xlogy(used, used)
    zk = z.gather(1, at)
    loss = t * t * (terms - used * (zk - lse)).sum(1) * has[:, 0]
    q = torch.exp(z - lse) * has
    dl = g * t * q.scatter_add(1, at, -used)
    size = (terms.abs() + used * (zk.abs() + lse.abs())).sum(1)
    return loss, dl @ b, dl.T @ a, dict(x=a, w=b, z=z, lse=lse[:, 0], q=q, dl=dl, g=g, at=at, listed=ids >= 0, size=size, t=t)


def wrong(dt, true, got, kept=False, precise=False):
    """The names of what is further from ``true`` (of :func:`exact`) than it may be.  ``precise``: the
    derivative is multiplied in two 16-bit parts, so that u^2 is what its rounding costs."""
    (loss, dx, dw, m), u = true, U[dt]
    (n, d), v, t = m["x"].shape, m["w"].shape[0], m["t"]
    far = 8 * STEP * (m["x"].norm(dim=1) * m["w"].norm(dim=1).max() / t + (d ** 0.5 + 2) * m["z"].abs().amax(1))
    off = far + (80 + v / 8192) * STEP + 2.0 ** -20 + 4 * STEP * m["lse"].abs()
    bad = []

    def over(name, error, bound):
        if not bool((error <= bound).all()):
            bad.append(name)

    over("loss", (got[0].double() - loss).abs(), t * t * (2 * off + (8 + m["at"].shape[1]) * STEP * m["size"]))
    span = m["g"].abs() * t * m["q"]
    each = ((u * u if precise else u) * m["dl"]).square() + (span * (far + 2.0 ** -20)[:, None]).square()
    if dt == torch.float16:
        each += (float(m["g"].abs().max()) * t * 2.0 ** -40) ** 2
    if kept:
        code = torch.where(m["q"] < 2.0 ** -24, 2.0 ** -8, torch.where(m["q"] < 2.0 ** -8, 2.0 ** -11, 2.0 ** -13))
        listed = torch.zeros_like(m["q"]).scatter_add_(1, m["at"], m["listed"].double()) > 0
        each += torch.where(listed, 0.0, span * code).square()

    def gradient(name, result, true, each, dl, shift, b, length):
        spread = (each @ b.square()).sqrt() + length ** 0.5 * STEP * (dl.square() @ b.square()).sqrt()
        common = (shift @ b).abs()
        error = (result.double() - true).abs()
        tiny = 2.0 ** -24  # of fp16
        over(name, error, 6 * spread + common + u * true.abs() + tiny)
        over(name + " row", error.norm(dim=1), 2 * spread.norm(dim=1) + common.norm(dim=1) + u * true.norm(dim=1)
             + tiny * true.shape[1] ** 0.5)
        over(name + " whole", error.norm(), 0.8 * (spread.norm().square() + (u * true.norm()).square()).sqrt() + common.norm()
             + tiny * true.numel() ** 0.5)

    shift = span * off[:, None]
    gradient("dx", got[1], dx, each, m["dl"], shift, m["w"], v)
    gradient("dw", got[2], dw, each.T, m["dl"].T, shift.T, m["x"], n)
    return bad


# (tokens, width, vocabulary, dtype): each at one of the largest sizes that are taken
LARGEST = [(3, 65536, 300, torch.bfloat16), (3, 65535, 300, torch.float16), (1 << 20, 8, 16, torch.bfloat16),
           (2, 8, 1 << 24, torch.float16), (17, 9, 1 << 22, torch.bfloat16)]


def largest(n, d, v, dt, dev):
    """Inputs that show every part of a long sum.  ``marks``: 64 places of the longest axis, its ends
    and the borders of tiles and pieces among them, that together carry half of the sum, so that each
    of them is worth far more than the roundings of all."""
    gen = torch.Generator(device=dev).manual_seed(n + d + v)

    def randn(*shape):
        return torch.randn(shape, device=dev, generator=gen)

    long = max(n, d, v)
    marks = torch.randint(0, long, (64,), device=dev, generator=gen)
    marks[:10] = torch.tensor([0, 255, 256, long // 2 - 1, long // 2, long - 257, long - 256, long - 255, long - 2, long - 1])
    marks = marks.unique()
    up = torch.full((n,), 1024.0 if dt == torch.float16 else 1.0, device=dev)
    w, x = randn(v, d) * d ** -0.5, randn(n, d)
    target = torch.randint(0, v, (n,), device=dev, generator=gen)
    if long == v:  # marked entries: logits ln(V / 64) above the others, in one direction each
        x = x.abs() + 1
        w = 0.25 * w
        axis = torch.arange(len(marks), device=dev) % d
        w[marks] = 0
        # the direction's mean logit over the tokens
        w[marks, axis] = torch.log(torch.tensor(v / 64.0, device=dev)) / x.mean(0)[axis]
        target[: len(marks)] = marks[-n:][: len(target)]
    elif long == n:  # marked tokens: as much upstream as the random sum of all others has
        up = torch.full((n,), 1.0, device=dev)
        up[marks] = (n / 64.0) ** 0.5
    return x.to(dt), w.to(dt), target, up, marks
