"""What the loss screen's comparison passes and what it finds, on the CPU: results that are as
exact as the kernels' pass, and results that are wrong in every pass alike do not."""

import pytest
import torch

from triton_kubernetes_amd.ops import head_screen

SIZES = [(300, 2000, 256), (256, 4096, 4096)]


def _step(tokens, vocab, hidden, dt):
    """Inputs, the softmax and targets of each token, and results that round as the kernels do."""
    gen = torch.Generator().manual_seed(tokens)
    x, w, target = head_screen.head_data(torch, tokens, vocab, hidden, dt, gen)
    z = x.double() @ w.double().T
    lse = torch.logsumexp(z, 1)
    q = torch.exp(z - lse[:, None])
    hit = torch.nn.functional.one_hot(target, vocab).double()
    loss = (lse - z.gather(1, target[:, None])[:, 0]).float()
    rows = torch.randperm(tokens, generator=gen)[:head_screen.SAMPLE]
    at = torch.cat((target[rows[:32]], torch.randperm(vocab, generator=gen)[:32]))
    return x, w, target, q, hit, loss, rows, at


def _gradients(x, w, dl):
    dl = dl.to(x.dtype).double() if x.dtype == torch.bfloat16 else (dl * 2.0 ** 15).to(x.dtype).double() * 2.0 ** -15
    return (dl @ w.double()).to(x.dtype), (dl.T @ x.double()).to(x.dtype)


def _judged(x, w, target, loss, dx, dw, rows, at):
    return head_screen.judge_step(torch, x, w, target[:, None], torch.ones((len(x), 1)), 1.0, loss, dx, dw, rows, at)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("size", SIZES)
def test_what_is_right_passes_and_what_is_wrong_does_not(size, dt):
    x, w, target, q, hit, loss, rows, at = _step(*size, dt)
    dx, dw = _gradients(x, w, q - hit)

    def judged(loss=loss, dx=dx, dw=dw):
        return _judged(x, w, target, loss, dx, dw, rows, at)

    assert judged()[:3] == (0, 0, 0) and judged()[3] <= 1
    v, n = size[1], size[0]
    half = q.clone()
    half[:, : v // 2] = 0
    piece = q.clone()
    piece[:, v // 2: v // 2 + 256] = 0  # a tile of the vocabulary
    few = q.clone()
    few[n // 2: n // 2 + 64] = 0  # a step's tokens
    for name, wrong in (("half the vocabulary", _gradients(x, w, half - hit)[0]), ("a tile", _gradients(x, w, piece - hit)[0]),
                        ("no softmax", _gradients(x, w, -hit)[0]), ("no targets", _gradients(x, w, q)[0]),
                        ("5 % too large", (dx.double() * 1.05).to(dt)), ("zeros", 0 * dx), ("NaN", dx * float("nan")),
                        ("the next token's", dx.roll(1, 0)), ("columns shifted", dx.roll(1, 1))):
        assert judged(dx=wrong)[1] > 0, name
    for name, wrong in (("64 tokens", _gradients(x, w, few - hit)[1]), ("no softmax", _gradients(x, w, -hit)[1]),
                        ("no targets", _gradients(x, w, q)[1]), ("5 % too large", (dw.double() * 1.05).to(dt)),
                        ("zeros", 0 * dw), ("NaN", dw * float("nan")), ("the next entry's", dw.roll(1, 0))):
        assert judged(dw=wrong)[2] > 0, name
    for name, wrong in (("0.01 off", loss + 0.01), ("a tile's sum lost", loss + torch.log1p(-q[:, :256].sum(1)).float()),
                        ("NaN", loss * float("nan"))):
        assert judged(loss=wrong)[0] > 0, name


def test_one_wrong_value_of_each_is_found():
    x, w, target, q, hit, loss, rows, at = _step(*SIZES[0], torch.bfloat16)
    dx, dw = _gradients(x, w, q - hit)
    for place in range(3):
        got = [loss.clone(), dx.clone(), dw.clone()]
        where = (rows[3],) if place == 0 else (rows[3], 5) if place == 1 else (at[3], 5)
        got[place][where] += 0.02 if place == 0 else 0.25
        assert [bool(b) for b in _judged(x, w, target, *got, rows, at)[:3]] == [place == i for i in range(3)]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_a_teachers_lists_are_judged(dt):
    """Lists with an entry twice, with none, and with probabilities of 0, at a temperature of 2."""
    t, (x, w, target, _, _, _, rows, at) = 2.0, _step(*SIZES[0], dt)
    n, v = SIZES[0][:2]
    gen = torch.Generator().manual_seed(9)
    ids = torch.randint(-300, v, (n, 20), generator=gen)
    ids[:, 0] = ids[:, 5] = target
    p = torch.softmax(torch.randn((n, 20), generator=gen).double().masked_fill(ids < 0, -float("inf")), 1)
    z = x.double() @ w.double().T / t
    lse = torch.logsumexp(z, 1, keepdim=True)
    loss = t * t * (torch.special.xlogy(p, p) - p * (z.gather(1, ids.clamp_min(0)) - lse)).sum(1)
    dl = t * torch.exp(z - lse).scatter_add(1, ids.clamp_min(0), -p)
    once = t * torch.exp(z - lse).scatter(1, ids.clamp_min(0), 0)
    dx, dw = _gradients(x, w, dl)

    def judged(loss, dx, dw):
        return head_screen.judge_step(torch, x, w, ids, p, t, loss.float(), dx, dw, rows, at)

    assert judged(loss, dx, dw)[:3] == (0, 0, 0)
    wrong = _gradients(x, w, once)
    assert judged(loss, wrong[0], dw)[1] and judged(loss, dx, wrong[1])[2] and judged(loss / t, dx, dw)[0]
