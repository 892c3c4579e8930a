"""Screens of a GPU with the output head's operators (``tk-gpu loss`` and ``tk-gpu gemv``).

The GEMM screen (``gemm.screen``) proves the matrix cores and the LDS.  These run what a
training step and a token server run on such a node, and check the answers: the exponential
and logarithm, sums across lanes, transposing LDS reads and the three products of a backward
pass, for a cross entropy and a distillation (:func:`loss_screen`), and 4-bit codes unpacked and scaled on the way from HBM
(:func:`gemv_screen`).  Every pass has to give the bits of the first one, and the first is
compared with 64-bit sums that torch forms.  Both need PyTorch-ROCm on the node.
"""

from contextlib import contextmanager
from dataclasses import asdict, dataclass
from typing import Any, Dict

from .native import NativeUnavailable

SAMPLE = 64  # tokens, and vocabulary entries, whose gradients are computed again in 64 bits


def _torch(dev: int):
    try:
        import torch
    except ImportError as exc:
        raise NativeUnavailable("this screen needs PyTorch-ROCm") from exc
    if not torch.cuda.is_available():
        raise NativeUnavailable("no GPU")
    if not 0 <= dev < torch.cuda.device_count():
        raise NativeUnavailable(f"no GPU {dev} (there are {torch.cuda.device_count()})")
    return torch


@contextmanager
def _on(torch, dev: int):
    """``dev`` as the current device; what it has no memory for is a refusal."""
    try:
        with torch.cuda.device(dev):
            yield
    except torch.OutOfMemoryError as exc:
        raise NativeUnavailable("the GPU's memory does not hold a screen of these sizes") from exc


@dataclass
class LossScreen:
    tokens: int
    vocab: int
    hidden: int
    dtype: str
    entries: int  # of a teacher's list, 0: no distillation
    ms: float  # a step of the cross entropy
    distill_ms: float
    tflops: float  # of the 6 N V D that a step of the cross entropy cannot do without
    differing: int  # values that were not the first pass' bits, over all passes
    bad_losses: int
    bad_dx: int
    bad_dw: int
    max_norm_error: float  # |error| / tolerance, the worst of all that was compared

    @property
    def ok(self) -> bool:
        return self.differing == self.bad_losses == self.bad_dx == self.bad_dw == 0

    def to_json(self) -> Dict[str, Any]:
        return dict(asdict(self), ok=self.ok)


@dataclass
class GemvScreen:
    rows: int
    out: int
    inp: int
    group: int
    dtype: str
    us: float
    gbps: float
    differing: int
    bad: int
    first_bad: int  # row * out + column, -1: none
    max_norm_error: float

    @property
    def ok(self) -> bool:
        return self.differing == self.bad == 0

    def to_json(self) -> Dict[str, Any]:
        return dict(asdict(self), ok=self.ok)


def _dtype(torch, name: str):
    types = {"bf16": torch.bfloat16, "fp16": torch.float16}
    if name not in types:
        raise ValueError(f"unknown dtype '{name}' ({' | '.join(types)})")
    return types[name]


def _timed(torch, call, reps: int) -> float:
    """The best of ``reps`` calls, in seconds, by events on the current stream."""
    best = float("inf")
    for _ in range(max(1, reps)):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        call()
        end.record()
        end.synchronize()
        best = min(best, start.elapsed_time(end) * 1e-3)
    return best


STEP = 2.0 ** -23  # of an fp32 sum, relative to it, at most


class _Verdict:
    """Counts of what was off by more than its tolerance, and the worst error / tolerance of all."""

    def __init__(self):
        self.worst = 0.0

    def over(self, got, want, tol) -> int:
        ratio = ((got.double() - want).abs() / tol).nan_to_num(nan=float("inf"))
        self.worst = max(self.worst, float(ratio.max()))
        return int((ratio > 1).sum())


def head_data(torch, tokens: int, vocab: int, hidden: int, dt, gen):
    """``(x, w, target)`` of a head whose logits have a standard deviation of 3, so that a token's
    probabilities are neither one entry nor all alike, and its softmax is a large part of its
    gradient (0.9 % of it at a deviation of 1 and 32768 entries)."""
    dev = gen.device
    w = (torch.randn((vocab, hidden), device=dev, generator=gen) * hidden ** -0.5).to(dt)
    target = torch.randint(0, vocab, (tokens,), device=dev, generator=gen)
    x = 3 * torch.randn((tokens, hidden), device=dev, generator=gen)
    return (x + 8 * torch.rand((tokens, 1), device=dev, generator=gen) * w[target].float()).to(dt), w, target


def judge_step(torch, x, w, ids, p, t, loss, dx, dw, rows, at):
    """``(bad losses, bad in dx, bad in dw, worst error / tolerance)`` of the sum over all tokens of
    ``t^2 sum_k p_k (log p_k - log q_{id_k})``, ``q`` the softmax of ``x @ w.T / t``: every token's
    loss, ``dx`` of the tokens ``rows`` and ``dw`` of the entries ``at``, against 64 bits.  On any device.

    Tolerances.  A logit is a sum of D products whose partial sums grow as a random walk to |x||w|
    / sqrt(D) and as a line to z: rounding each costs about STEP (|x||w| + sqrt(D) |z|) at most,
    here times 8 (``far``).  The sum of exponentials is of at most 80 + V/8192 additions in a row, all
    positive; with 2^-20 for the exponential and logarithm that is the row's ``off``, common to all of
    its probabilities.  The derivative of a logit is rounded to 16 bits, half a step u each; these
    roundings are independent, so a gradient's element is off by 6 standard deviations at most, 6 u
    sqrt(sum (dl b)^2), and half a step of its own.  A row of a gradient as a whole is off by u times
    its terms' root mean square and u times itself, more than twice what roundings that are spread
    evenly give; this finds what is wrong a little everywhere."""
    n, d = x.shape
    v, u, c = w.shape[0], torch.finfo(x.dtype).eps / 2, 2048
    verdict, inf = _Verdict(), float("inf")
    used = torch.where(ids >= 0, p.double(), 0.0)
    at_ids = ids.clamp_min(0)
    # 64-bit logits of all tokens, a block at a time: their logsumexp, the largest, and the targets'
    lse, top, zk = (torch.empty(s, dtype=torch.float64, device=x.device) for s in ((n,), (n,), tuple(ids.shape)))
    for n0 in range(0, n, 4096):
        part = slice(n0, n0 + 4096)
        xs = x[part].double()
        m, s, big = xs.new_full((len(xs),), -inf), xs.new_zeros(len(xs)), xs.new_zeros(len(xs))
        for v0 in range(0, v, c):
            z = xs @ w[v0:v0 + c].double().T / t
            m2 = torch.maximum(m, z.amax(1))
            s, m = s * torch.exp(m - m2) + torch.exp(z - m2[:, None]).sum(1), m2
            big = torch.maximum(big, z.abs().amax(1))
        lse[part], top[part] = m + torch.log(s), big
        for k in range(ids.shape[1]):
            zk[part, k] = (xs * w[at_ids[part, k]].double()).sum(1) / t
    far = 8 * STEP * (x.double().norm(dim=1) * float(w.float().norm(dim=1).max()) / t + (d ** 0.5 + 2) * top)
    off = far + (80 + v / 8192) * STEP + 2.0 ** -20 + 4 * STEP * lse.abs()
    terms = torch.special.xlogy(used, used)
    true = t * t * (terms - used * (zk - lse[:, None])).sum(1)
    size = (terms.abs() + used * (zk.abs() + lse.abs()[:, None])).sum(1)
    bad_losses = verdict.over(loss, true, t * t * (2 * off + (8 + ids.shape[1]) * STEP * size))

    delta = far + 2.0 ** -20 + v ** 0.5 * STEP
    xr, lse_r, off_r, delta_r = x[rows].double(), lse[rows, None], off[rows, None], delta[rows, None]
    true, square, drift = (torch.zeros((len(rows), d), dtype=torch.float64, device=x.device) for _ in range(3))
    for v0 in range(0, v, c):
        ws = w[v0:v0 + c].double()
        q = torch.exp(xr @ ws.T / t - lse_r)
        here = (ids[rows] >= v0) & (ids[rows] < v0 + c)
        dl = q.scatter_add(1, torch.where(here, ids[rows] - v0, 0).clamp(0, len(ws) - 1), -torch.where(here, used[rows], 0.0)) * t
        true += dl @ ws
        square += dl.square() @ ws.square()
        drift += t * (q @ ws)

    def compare(got, true, spread, common):
        tol = 6 * spread + common + u * true.abs() + 1e-7
        rowwise = spread.norm(dim=1) + common.norm(dim=1) + u * true.norm(dim=1) + 1e-7 * d ** 0.5
        return verdict.over(got, true, tol) + verdict.over((got.double() - true).norm(dim=1), 0 * rowwise, rowwise)

    bad_dx = compare(dx[rows], true, square.sqrt() * (u + delta_r), off_r * drift.abs())

    true, square, drift = (torch.zeros((len(at), d), dtype=torch.float64, device=x.device) for _ in range(3))
    wa = w[at].double()
    for n0 in range(0, n, 4096):
        part = slice(n0, n0 + 4096)
        xs = x[part].double()
        q = torch.exp(xs @ wa.T / t - lse[part, None])
        dl = q.clone()
        for k in range(ids.shape[1]):
            dl -= (ids[part, k, None] == at[None]) * used[part, k, None]
        true += t * (dl.T @ xs)
        each = (u * dl).square() + (q * (delta + off)[part, None]).square() + n * STEP ** 2 * dl.square()
        square += t * t * (each.T @ xs.square())
        drift += t * (q.T @ xs)
    bad_dw = compare(dw[at], true, square.sqrt(), float(off.max()) * drift.abs())
    return bad_losses, bad_dx, bad_dw, verdict.worst


def loss_screen(dev: int = 0, tokens: int = 4096, vocab: int = 32768, hidden: int = 4096, reps: int = 3,
                dtype: str = "bf16", inject: int = -1, entries: int = 64) -> LossScreen:
    """``reps`` training steps of the head (loss and both gradients) on random operands, and as
    many distillation steps from lists of ``entries`` logits (0: none).  ``inject`` changes one
    value of the last cross entropy's weight gradient, which has to show."""
    torch = _torch(dev)
    from .loss import linear_cross_entropy, linear_distill

    dt, temperature, entries = _dtype(torch, dtype), 2.0, min(entries, vocab)
    with _on(torch, dev):
        gen = torch.Generator(device="cuda").manual_seed(0x5eed)
        x, w, target = head_data(torch, tokens, vocab, hidden, dt, gen)
        x.requires_grad_()
        w.requires_grad_()
        ones = torch.ones(tokens, device="cuda")
        rows = torch.randperm(tokens, device="cuda", generator=gen)[:SAMPLE]
        at = torch.randperm(vocab, device="cuda", generator=gen)[:SAMPLE]
        hits = len(at) // 2  # half of them are some token's target
        at[:hits] = target[torch.randint(0, tokens, (hits,), device="cuda", generator=gen)]

        def passes(call, changed):
            """(seconds, values that differ from the first pass', the first pass)"""

            def step():
                loss = call()
                return (loss.detach(), *torch.autograd.grad(loss, (x, w), ones))

            bits = torch.int16
            first = step()
            seconds, differing = float("inf"), 0
            for turn in range(max(1, reps)):
                got = []
                seconds = min(seconds, _timed(torch, lambda: got.extend(step()), 1))
                if changed >= 0 and turn == max(1, reps) - 1:
                    got[2].view(-1)[changed] += 1
                # the bits, so that a NaN that repeats is no difference here (the comparison below finds it)
                differing += sum(int((a.view(bits) != b.view(bits)).sum()) for a, b in zip(got, first))
            return seconds, differing, first

        def judged(ids, p, t, first):
            return judge_step(torch, x.detach(), w.detach(), ids, p, t, *first, rows, at)

        seconds, differing, first = passes(lambda: linear_cross_entropy(x, w, target, reduction="none"), inject)
        found = [judged(target[:, None], torch.ones((tokens, 1), device="cuda"), 1.0, first)]
        distill = 0.0
        if entries:  # the target and entries that may occur twice, some of them none
            ids = torch.randint(-vocab // 8, vocab, (tokens, entries), device="cuda", generator=gen)
            ids[:, 0] = target
            logits = 2 * torch.randn((tokens, entries), device="cuda", generator=gen)
            distill, more, first = passes(lambda: linear_distill(x, w, ids, logits, temperature=temperature,
                                                                 reduction="none"), -1)
            differing += more
            p = torch.softmax(logits.double().masked_fill(ids < 0, -float("inf")) / temperature, 1)
            found.append(judged(ids, p, temperature, first))
        bad_losses, bad_dx, bad_dw = (sum(f[i] for f in found) for i in range(3))
    return LossScreen(tokens, vocab, hidden, dtype, entries, seconds * 1e3, distill * 1e3,
                      6e-12 * tokens * vocab * hidden / seconds, differing, bad_losses, bad_dx, bad_dw,
                      max(f[3] for f in found))


def gemv_screen(dev: int = 0, rows: int = 1, out: int = 16384, inp: int = 16384, group: int = 128, reps: int = 20,
                dtype: str = "bf16", inject: int = -1) -> GemvScreen:
    """``reps`` products of ``rows`` tokens with one 4-bit weight of random codes, each result
    compared with the 64-bit one.  ``inject`` changes one value of the last result."""
    torch = _torch(dev)
    from .gemv import dequantize_w4, gemv_w4

    dt = _dtype(torch, dtype)
    if group < 32 or group % 32 or inp < group or inp % group:
        raise ValueError(f"a group of {group} must be a multiple of 32 that divides {inp} columns")
    with _on(torch, dev), torch.no_grad():
        gen = torch.Generator(device="cuda").manual_seed(0x5eed)
        codes = torch.randint(0, 256, (out, inp // 2), device="cuda", generator=gen, dtype=torch.uint8)
        scales = (torch.rand((out, inp // group), device="cuda", generator=gen) + 0.5).to(dt)
        zeros = torch.randint(4, 12, (out, inp // group), device="cuda", generator=gen, dtype=torch.uint8)
        x = torch.randn((rows, inp), device="cuda", generator=gen).to(dt)
        first = gemv_w4(x, codes, scales, zeros)
        seconds, differing = float("inf"), 0
        for turn in range(max(1, reps)):
            got = torch.empty_like(first)
            seconds = min(seconds, _timed(torch, lambda: gemv_w4(x, codes, scales, zeros, out=got), 1))
            if inject >= 0 and turn == max(1, reps) - 1:
                got.view(-1)[inject] += 64
            differing += int((got.view(torch.int16) != first.view(torch.int16)).sum())
        u, step32, bad, first_bad, worst = torch.finfo(dt).eps / 2, 2.0 ** -23, 0, -1, 0.0
        per = x.double().abs().view(rows, -1, group).sum(2)
        for n0 in range(0, out, 2048):
            part = slice(n0, n0 + 2048)
            true = x.double() @ dequantize_w4(codes[part], scales[part], zeros[part]).double().T
            size = per @ scales[part].double().T
            # fp32 sums of up to 31 sum |x| a group, of codes and of zeros, then one addition a group
            tol = u * true.abs() + (62 * (group + 4) + 31 * (inp // group + 8)) * step32 * size
            ratio = ((first[:, part].double() - true).abs() / tol).nan_to_num(nan=float("inf"))
            worst = max(worst, float(ratio.max()))
            off = (ratio > 1).nonzero()
            bad += len(off)
            if len(off) and first_bad < 0:
                first_bad = int(off[0, 0]) * out + n0 + int(off[0, 1])
    nbytes = out * inp // 2 + 3 * out * (inp // group) + 2 * rows * (inp + out)
    return GemvScreen(rows, out, inp, group, dtype, seconds * 1e6, nbytes / seconds * 1e-9, differing, bad, first_bad,
                      worst)
