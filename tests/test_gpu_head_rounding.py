"""How much more than their own rounding the gradients have: a derivative that is rounded to 16 bits
costs at most as much again, but one number that is most of a token's derivative is not left to
chance."""

import pytest
import torch

import head_norms

pytestmark = pytest.mark.gpu


def _ratio(got, true):
    """Its error over that of rounding the exact result once."""
    return float((got.double() - true).norm() / (true.to(got.dtype).double() - true).norm())


@pytest.mark.parametrize("keep", [False, True], ids=["again", "kept"])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("n,d,v", [(600, 64, 19044), (2400, 104, 13164), (3000, 488, 4924), (5000, 1000, 3000)])
def test_gradients_of_x_that_are_mostly_their_targets(n, d, v, dt, keep):
    """Upstream gradients of 1 to 1.25, of which a 16-bit type holds the fewest steps (bf16: 128 of 2^-7), and
    targets with little probability: the derivative is nearly all at the target.  Its rounding is made good,
    and of the rest's, at most 1/8 of the norm, sqrt(1 + 1/64) = 1.01 is left; 1.05 with what is less even."""
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy

    gen = torch.Generator(device="cuda").manual_seed(n)
    w = (torch.randn((v, d), device="cuda", generator=gen) * d ** -0.5).to(dt)
    x = torch.randn((n, d), device="cuda", generator=gen).to(dt)
    target = torch.randint(0, v, (n,), device="cuda", generator=gen)
    up = 1 + torch.rand(n, device="cuda", generator=gen) / 4
    a = x.clone().requires_grad_()
    dx, = torch.autograd.grad(linear_cross_entropy(a, w, target, reduction="none", keep_logits=keep), a, up)
    _, true, _, m = head_norms.exact(x, w, target[:, None], torch.ones((n, 1), device="cuda"), 1.0, up)
    rest = m["dl"].scatter(1, target[:, None], 0.0)
    assert float(rest.norm() / m["dl"].norm()) <= 1 / 8
    assert _ratio(dx, true) <= 1.05


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("n", [200, 1300])
def test_gradients_of_x_that_are_mostly_a_few_entries_of_a_list(n, dt):
    """Two entries of probability 1/4 and 3/4 a token, both above 1/8: as for a single target."""
    from triton_kubernetes_amd.ops.loss import linear_distill

    d, v = 136, 9000
    gen = torch.Generator(device="cuda").manual_seed(n)
    w = (torch.randn((v, d), device="cuda", generator=gen) * d ** -0.5).to(dt)
    x = torch.randn((n, d), device="cuda", generator=gen).to(dt)
    ids = torch.randint(0, v, (n, 2), device="cuda", generator=gen)
    logits = torch.tensor([0.0, 3.0], device="cuda").log1p().expand(n, 2)
    up = 1 + torch.rand(n, device="cuda", generator=gen) / 4
    a = x.clone().requires_grad_()
    dx, = torch.autograd.grad(linear_distill(a, w, ids, logits, reduction="none"), a, up)
    p = torch.softmax(logits.double(), 1)
    true = head_norms.exact(x, w, ids, p, 1.0, up)[1]
    assert _ratio(dx, true) <= 1.05
