"""Losses that are small because the model is sure: differences of large logits, which have to come
from the same sums."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]
NAMES = {torch.bfloat16: "bf16", torch.float16: "fp16"}


def _sure(n, d, v, dt, logit):
    """Each token's target has a logit near ``logit``, the others have a deviation of about 2."""
    gen = torch.Generator(device="cuda").manual_seed(n + d)
    w = (torch.randn((v, d), device="cuda", generator=gen) * d ** -0.5).to(dt)
    target = torch.randint(0, v, (n,), device="cuda", generator=gen)
    x = 2 * torch.randn((n, d), device="cuda", generator=gen) + logit * w[target].float()
    return x.to(dt), w, target, gen


def _additions(v):
    """Of one row's sum of exponentials, in a row: a lane's, a tile's and the tiles'."""
    return 80 + v / 8192


@pytest.mark.parametrize("keep", [False, True], ids=["again", "kept"])
@pytest.mark.parametrize("tiles", [0, 7], ids=["large", "small"])
@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("n,d,v,logit", [(33, 4096, 3000, 60.0), (5, 1000, 50021, 40.0), (300, 77, 1030, 80.0), (70, 512, 9000, 25.0)])
def test_cross_entropy(n, d, v, logit, dt, tiles, keep, monkeypatch):
    """loss = log(sum of exp(z_v - z_t)): the largest term is 1 and exact, the others are off by the error of
    a logit, about 8 STEP (|x||w| + sqrt(D) |z|) of themselves, each addition by half a step of the sum, and
    the exponentials and the logarithm by 2^-21 of what they give beside 1."""
    from triton_kubernetes_amd.ops import loss

    monkeypatch.setattr(loss, "small_products", lambda *a: tiles)
    x, w, target, _ = _sure(n, d, v, dt, logit)
    w.requires_grad_()
    got = loss.linear_cross_entropy(x, w, target, reduction="none", keep_logits=keep).detach().double()
    with torch.no_grad():
        z = x.double() @ w.double().T
        far = z - z.gather(1, target[:, None])
        rest = torch.exp(far.scatter(1, target[:, None], -float("inf"))).sum(1)  # the terms beside the target's
        want = torch.log1p(rest)
        step = 2.0 ** -23
        err = 8 * step * (x.double().norm(dim=1) * w.double().norm(dim=1).max() + d ** 0.5 * z.abs().amax(1))
        # (a sum of s rounds by s / 2 steps; d log(s) = ds / s)
        bound = _additions(v) * step / 2 + rest / (1 + rest) * (2 * err + 2.0 ** -20) + want * 2.0 ** -20
    assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() / bound).max())


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("n,d,v,k", [(33, 4096, 3000, 20), (5, 1000, 50021, 3), (300, 72, 1030, 70), (3, 5008, 36401, 4), (9, 77, 500, 16)])
@pytest.mark.parametrize("tiles", [0, 7], ids=["large", "small"])
def test_distillation(n, d, v, k, dt, tiles, monkeypatch):
    """The student agrees with its teacher, whose lists are the student's own logits of 16 bits or less:
    sum p (log p - log q) is a difference of nearly equal numbers, each good to a few steps."""
    from triton_kubernetes_amd.ops import loss

    monkeypatch.setattr(loss, "small_products", lambda *a: tiles)
    x, w, target, gen = _sure(n, d, v, dt, 50.0)
    ids = torch.randint(0, v, (n, k), device="cuda", generator=gen)
    ids[:, 0] = target
    with torch.no_grad():
        z = x.double() @ w.double().T
        logits = z.gather(1, ids).float()
    got = loss.linear_distill(x, w, ids, logits, reduction="none").double()
    logp, logq = torch.log_softmax(logits.double(), 1), torch.log_softmax(z, 1).gather(1, ids)
    p = logp.exp()
    want = (p * (logp - logq)).sum(1)
    step = 2.0 ** -23
    err = 8 * step * (x.double().norm(dim=1) * w.double().norm(dim=1).max() + d ** 0.5 * z.abs().amax(1))
    # by entry: p's rounding (the softmax of k numbers), the logarithm's, the distances'; and the sums
    each = (p * ((logp.abs() + logq.abs()) * 8 * step + k * step + 2.0 ** -20 * (logp.abs() + 2.0 ** -3))).sum(1)
    other = 1 - p.amax(1)  # what a logit's error changes is not the largest's share
    bound = _additions(v) * step / 2 + k * step + each + 4 * err * other + want.abs() * 2.0 ** -20
    assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() / bound).max())


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
def test_a_vocabulary_of_one_has_no_loss(dt):
    """The target is all there is: its logit, however large, is the logarithm of the sum, to the bit."""
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy, linear_distill

    gen = torch.Generator(device="cuda").manual_seed(1)
    for d in (8, 77, 4096):
        x = (9 * torch.randn((40, d), device="cuda", generator=gen)).to(dt)
        w = torch.randn((1, d), device="cuda", generator=gen).to(dt)
        t = torch.zeros(40, device="cuda", dtype=torch.int64)
        # (one term: exp2 of how far the rounded maximum is from it, whose logarithm is that again)
        assert float(linear_cross_entropy(x, w, t, reduction="none").abs().max()) <= 2.0 ** -23
        lists = linear_distill(x, w, t[:, None].expand(40, 5), torch.zeros((40, 1), device="cuda").expand(40, 5), reduction="none")
        assert float((lists + torch.log(torch.tensor(5.0))).abs().max()) <= 2.0 ** -21
