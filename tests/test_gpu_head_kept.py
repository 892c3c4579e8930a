"""What the output head's losses hold between their passes, and the form that keeps the logits
in 16 bits because the caller asks for it (tests/head_reference.py derives the tolerances)."""

import pytest
import torch

import head_reference as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]
NAMES = {torch.bfloat16: "bf16", torch.float16: "fp16"}


def _inputs(n, d, v, dt, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    w = (torch.randn((v, d), device="cuda", generator=gen) * d ** -0.5).to(dt)
    t = torch.randint(0, v, (n,), device="cuda", generator=gen)
    x = torch.randn((n, d), device="cuda", generator=gen)
    x += 4 * torch.rand((n, 1), device="cuda", generator=gen) * w[t].float()
    return x.to(dt), w, t


def test_losses_alive_at_once_hold_no_logits():
    """Four losses of 600 x 40000 logits between their passes: each holds its packed x and less
    than a byte for every eighth logit."""
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy, linear_distill

    n, d, v = 600, 512, 40_000
    x, w, t = _inputs(n, d, v, torch.bfloat16, 1)
    x.requires_grad_()
    w.requires_grad_()
    linear_cross_entropy(x, w, t)  # the library is loaded
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    alive = [linear_cross_entropy(x, w, t), linear_distill(x, w, t[:, None], torch.zeros((n, 1), device="cuda")),
             linear_cross_entropy(x[:300], w, t[:300]), linear_cross_entropy(x, w, t, reduction="sum")]
    held = torch.cuda.memory_allocated() - before
    assert held < 4 * (2 * n * d + n * v // 8), held
    torch.autograd.grad(sum(alive), (x, w))


@pytest.mark.parametrize("tiles", [0, 7], ids=["large", "small"])
@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("n,d,v,k", [(1, 8, 1, 0), (5, 72, 257, 0), (257, 1000, 5003, 0), (300, 77, 1030, 0), (513, 128, 513, 0),
                                     (7, 72, 257, 5), (130, 264, 1111, 64), (300, 512, 999, 33)])
def test_kept_logits(n, d, v, k, dt, tiles, monkeypatch):
    from triton_kubernetes_amd.ops import loss

    monkeypatch.setattr(loss, "small_products", lambda *a: tiles)
    x, w, t = _inputs(n, d, v, dt, 2)
    gen = torch.Generator(device="cuda").manual_seed(3)
    up = torch.rand(n, device="cuda", generator=gen) - 0.3
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    if k:
        ids = torch.randint(0, v, (n, k), device="cuda", generator=gen)
        ids[torch.rand((n, k), device="cuda", generator=gen) < 0.2] = -1
        logits = torch.randn((n, k), device="cuda", generator=gen) * 3
        got = loss.linear_distill(a, b, ids, logits, temperature=2.0, reduction="none", keep_logits=True)
        lists, temp = ref.teacher_of(ids, logits, 2.0), 2.0
    else:
        got = loss.linear_cross_entropy(a, b, t, reduction="none", keep_logits=True)
        lists, temp = ref.targets_of(t, -100, n, v), 1.0
    want = ref.head(x, w, *lists, temp, up.double(), kept=True)
    for name, value, bound in zip(("loss", "dx", "dw"), (got.detach(), *torch.autograd.grad(got, (a, b), up)), want):
        ref.check(name, value, bound)
