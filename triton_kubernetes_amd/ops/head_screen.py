"""Screens of a GPU with the output head's operators (``tk-gpu loss`` and ``tk-gpu gemv``).

The GEMM screen (``gemm.screen``) proves the matrix cores and the LDS.  These run what a
training step and a token server run on such a node, and check the answers: the exponential
and logarithm, sums across lanes, transposing LDS reads and the three products of a backward
pass (:func:`loss_screen`), and 4-bit codes unpacked and scaled on the way from HBM
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
    ms: float
    tflops: float  # of the 6 N V D that a step cannot do without
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


def _over(torch, got, want, tol):
    """(elements off by more than ``tol`` or not finite, the worst error / tolerance)."""
    ratio = ((got.double() - want).abs() / tol).nan_to_num(nan=float("inf"))
    return int((ratio > 1).sum()), float(ratio.max())


def loss_screen(dev: int = 0, tokens: int = 4096, vocab: int = 32768, hidden: int = 4096, reps: int = 3,
                dtype: str = "bf16", inject: int = -1) -> LossScreen:
    """``reps`` training steps of the head (loss and both gradients) on random operands.
    ``inject`` changes one value of the last pass' weight gradient, which has to show."""
    torch = _torch(dev)
    from .loss import linear_cross_entropy

    dt = _dtype(torch, dtype)
    with _on(torch, dev):
        gen = torch.Generator(device="cuda").manual_seed(0x5eed)
        w = (torch.randn((vocab, hidden), device="cuda", generator=gen) * hidden ** -0.5).to(dt).requires_grad_()
        target = torch.randint(0, vocab, (tokens,), device="cuda", generator=gen)
        x = torch.randn((tokens, hidden), device="cuda", generator=gen)
        x = (x + 8 * torch.rand((tokens, 1), device="cuda", generator=gen) * w.detach()[target].float()).to(dt)
        x.requires_grad_()
        ones = torch.ones(tokens, device="cuda")

        def step():
            loss = linear_cross_entropy(x, w, target, reduction="none")
            return (loss.detach(), *torch.autograd.grad(loss, (x, w), ones))

        bits = torch.int16
        first = step()
        seconds, differing = float("inf"), 0
        for turn in range(max(1, reps)):
            got = []
            seconds = min(seconds, _timed(torch, lambda: got.extend(step()), 1))
            if inject >= 0 and turn == max(1, reps) - 1:
                got[2].view(-1)[inject] += 1
            # the bits, so that a NaN that repeats is no difference here (the comparison below finds it)
            differing += sum(int((a.view(bits) != b.view(bits)).sum()) for a, b in zip(got, first))
        loss, dx, dw = first[0].double(), first[1], first[2]

        u, step32 = torch.finfo(dt).eps / 2, 2.0 ** -23
        xs, ws = x.detach().double(), w.detach()
        rows = torch.randperm(tokens, device="cuda", generator=gen)[:SAMPLE]
        z = xs[rows] @ ws.double().T
        lse = torch.logsumexp(z, 1)
        true = lse - z.gather(1, target[rows, None])[:, 0]
        # a logit is a sum of `hidden` fp32 products, the sum of exponentials one of `vocab`
        far = (hidden + 8) * step32 * (xs[rows].norm(dim=1) * float(ws.float().norm(dim=1).max())) + vocab * step32
        bad_losses, worst = _over(torch, loss[rows], true, 2 * far + 32 * step32 * (1 + true.abs() + lse.abs()))
        dl = torch.exp(z - lse[:, None]).scatter_add_(1, target[rows, None], -torch.ones_like(lse)[:, None])
        size = dl.abs() @ ws.double().abs()
        bad_dx, more = _over(torch, dx[rows], dl @ ws.double(),
                             (u + 4 * far[:, None] + vocab * step32) * size + u * (dl @ ws.double()).abs() + 1e-7)
        worst = max(worst, more)
        # entries of the weight's gradient: the softmax there follows from the tokens' losses
        at = torch.randperm(vocab, device="cuda", generator=gen)[:SAMPLE]
        at[: SAMPLE // 2] = target[torch.randint(0, tokens, (len(at[: SAMPLE // 2]),), device="cuda", generator=gen)]
        z_own = (xs * ws[target].double()).sum(1)
        hit = (target[:, None] == at[None]).double()
        q = torch.exp(xs @ ws[at].double().T - (loss + z_own)[:, None])
        err = 4 * ((hidden + 8) * step32 * xs.norm(dim=1) * float(ws.float().norm(dim=1).max()) + vocab * step32)
        dl = q - hit
        size = dl.abs().T @ xs.abs()
        true = dl.T @ xs
        bad_dw, more = _over(torch, dw[at], true, (u + tokens * step32) * size + (q * err[:, None]).T @ xs.abs()
                             + u * true.abs() + 1e-7)
        worst = max(worst, more)
    return LossScreen(tokens, vocab, hidden, dtype, seconds * 1e3, 6e-12 * tokens * vocab * hidden / seconds, differing,
                      bad_losses, bad_dx, bad_dw, worst)


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
