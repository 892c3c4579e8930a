"""The output head's losses at the largest sizes that they take, and at ordinary ones, within
bounds that follow how errors add up: a part of a sum that is left out is outside them
(tests/test_head_norms.py shows that at these sizes and with these inputs)."""

import pytest
import torch

import head_norms

pytestmark = pytest.mark.gpu


def _check(x, w, ids, p, t, up, call, kept):
    true = head_norms.exact(x, w, ids, p, t, up)
    a, b = x.requires_grad_(), w.requires_grad_()
    loss = call(a, b)
    got = (loss.detach(), *torch.autograd.grad(loss, (a, b), up))
    assert head_norms.wrong(x.dtype, true, got, kept) == []


@pytest.mark.parametrize("keep", [False, True], ids=["again", "kept"])
@pytest.mark.parametrize("n,d,v,dt", head_norms.LARGEST)
def test_largest_sizes(n, d, v, dt, keep):
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy

    x, w, target, up, _ = head_norms.largest(n, d, v, dt, "cuda")
    _check(x, w, target[:, None], torch.ones((n, 1), device="cuda"), 1.0, up,
           lambda x, w: linear_cross_entropy(x, w, target, reduction="none", keep_logits=keep), keep)
    torch.cuda.empty_cache()


@pytest.mark.parametrize("n,d,v,dt", [(2, 8, 1 << 24, torch.float16), (1 << 18, 8, 16, torch.bfloat16),
                                      (17, 9, 1 << 22, torch.bfloat16), (3, 65536, 300, torch.bfloat16)])
def test_largest_distillations(n, d, v, dt):
    from triton_kubernetes_amd.ops.loss import linear_distill

    x, w, target, up, marks = head_norms.largest(n, d, v, dt, "cuda")
    gen = torch.Generator(device="cuda").manual_seed(n)
    ids = torch.randint(-v // 8, v, (n, 24), device="cuda", generator=gen)
    ids[:, 0], ids[0, 1:11] = target, marks[-10:] % v
    logits = torch.randn((n, 24), device="cuda", generator=gen)
    p = torch.softmax(logits.double().masked_fill(ids < 0, -float("inf")) / 2.0, 1)
    _check(x, w, ids, p, 2.0, up, lambda x, w: linear_distill(x, w, ids, logits, temperature=2.0, reduction="none"), False)
    torch.cuda.empty_cache()


@pytest.mark.parametrize("keep", [False, True], ids=["again", "kept"])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("n,d,v", [(1, 512, 50021), (48, 512, 1000), (257, 1000, 5003), (600, 256, 50021), (1500, 1288, 8000)])
@pytest.mark.parametrize("tiles", [None, 0, 7], ids=["rule", "large", "small"])
def test_ordinary_sizes(n, d, v, dt, keep, tiles, monkeypatch):
    from triton_kubernetes_amd.ops import loss

    if tiles is not None:
        monkeypatch.setattr(loss, "small_products", lambda *a: tiles)
    gen = torch.Generator(device="cuda").manual_seed(n)
    w = (torch.randn((v, d), device="cuda", generator=gen) * d ** -0.5).to(dt)
    target = torch.randint(0, v, (n,), device="cuda", generator=gen)
    x = 3 * torch.randn((n, d), device="cuda", generator=gen) + 6 * torch.rand((n, 1), device="cuda", generator=gen) * w[target].float()
    up = torch.rand(n, device="cuda", generator=gen) + 0.1
    ids = torch.where(torch.rand(n, device="cuda", generator=gen) < 0.2, -1, target) if n > 1 else target
    _check(x.to(dt), w, ids[:, None], torch.ones((n, 1), device="cuda"), 1.0, up,
           lambda x, w: loss.linear_cross_entropy(x, w, ids, ignore_index=-1, reduction="none", keep_logits=keep), keep)
