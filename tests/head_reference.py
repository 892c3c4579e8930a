"""The output head's operators in 64 bits, and how far a kernel may be from them.

Error model of the kernels.  u is half a step of the 16-bit type relative to a value (bf16
2^-8, fp16 2^-11).  A logit is a sum of D exact products in fp32: its error is at most
(D + 8) 2^-23 sum |x w| (each addition rounds or cuts off the last bit of a partial sum).  The
exponent's argument rounds once more, and exp2 and log2 are good to 2^-21 of their result.
Where the logits are kept in 16 bits for the backward pass, an entry that is no target is off by
half a step of 2^-12 in exp2's argument, ln 2 2^-13 = 8.5e-5 of its value, or of 2^-10, 3.4e-4,
where it is less than 2^-8 of its tile's largest, or of 2^-7, 2.71e-3, where less than 2^-24; the
number of steps, up to 65535, is itself rounded to fp32 on both ways, which adds 2^-6 of a step.
2^-13, 2^-11 and 2^-8 are above these."""

import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
STEP = 2.0 ** -23


def targets_of(target, ignore, n, v):
    """(ids, p) of a cross entropy: one target of probability 1, or none."""
    there = target != ignore
    return torch.where(there, target, -1)[:, None], there.double()[:, None]


def teacher_of(ids, logits, t):
    """(ids, p) of a teacher's lists: the softmax over the entries of each."""
    s = torch.where(ids >= 0, logits.double() / t, -math.inf)
    top = s.amax(1, keepdim=True)
    e = torch.where(s == -math.inf, 0.0, torch.exp(s - torch.where(top == -math.inf, 0.0, top)))
    total = e.sum(1, keepdim=True)
    return torch.where(total > 0, ids, -1), torch.where(total > 0, e / total, 0.0)


def head(x, w, ids, p, t, g, kept=True):
    """loss [n], dx, dw and their bounds for ``sum(g * loss)``, all in 64 bits; ``kept``: with the
    logits kept in 16 bits."""
    dt = x.dtype
    u = U[dt]
    has = (ids >= 0).any(1)
    x = torch.where(has[:, None], x.double(), 0.0)  # a row without a target reaches nothing
    w, g = w.double(), torch.where(has, g.double(), 0.0)
    z = x @ w.T / t
    dz = (x.abs() @ w.abs().T / t) * (x.shape[1] + 8) * STEP + z.abs() * 2 * STEP
    lse = torch.logsumexp(z, 1, keepdim=True)
    at = ids.clamp_min(0)
    used = torch.where(ids >= 0, p, 0.0)
    each = t * t * (torch.special.xlogy(used, used) - used * (z.gather(1, at) - lse)).sum(1)
    off = dz.amax(1) + lse.abs()[:, 0] * 4 * STEP + 2.0 ** -20 + w.shape[0] * STEP
    loss = dict(value=each * has, bound=(t * t * (2 * off + (each.abs() / (t * t) + 16) * 8 * STEP)) * has)
    q = torch.exp(z - lse)
    dl = q.clone().scatter_add_(1, at, -used) * (g * t)[:, None]
    # the stored derivative: q's error, one rounding, and what fp16 cannot hold under 2^-25 2^-15
    ddl = (q * (dz + off[:, None] + 2.0 ** -20)) * (g.abs() * t)[:, None] + u * dl.abs() + g.abs().max() * t * 2.0 ** -39
    if kept:
        code = torch.where(q < 2.0 ** -24, 2.0 ** -8, torch.where(q < 2.0 ** -8, 2.0 ** -11, 2.0 ** -13))
        code = q * code * (g.abs() * t)[:, None]
        listed = torch.zeros_like(q).scatter_add_(1, at, (ids >= 0).double()) > 0
        ddl = ddl + torch.where(listed, 0.0, code)
    ddl = torch.where(has[:, None], ddl, 0.0)
    size = dl.abs() + ddl

    def product(a, da, b):
        value = a @ b
        long = (a.shape[1] + 72) * STEP  # additions of a sum, over the pieces and splits too
        wrong = da @ b.abs() * (1 + 4 * STEP) + long * (size if a is dl else size.T) @ b.abs()
        return dict(value=value, bound=wrong + u * (value.abs() + wrong) + 2.0 ** -24)

    return loss, product(dl, ddl, w), product(dl.T, ddl.T, x)


def check(name, got, want):
    """Every element within its own bound."""
    got = got.double()
    assert got.shape == want["value"].shape, name
    off = (got - want["value"]).abs()
    bad = ~(off <= want["bound"])
    assert not bool(bad.any()), (name, int(bad.sum()), bad.nonzero()[0].tolist(), float(off[bad].max()),
                                 float(want["bound"][bad].max()))
