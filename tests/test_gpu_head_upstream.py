"""Upstream gradients that are not finite: they reach their own tokens' gradient of x, and w's,
as the formula has it, and no other token's."""

import pytest
import torch

import head_reference as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


def _inputs(dt):
    gen = torch.Generator(device="cuda").manual_seed(3)
    w = (torch.randn((700, 64), device="cuda", generator=gen) / 8).to(dt)
    return torch.randn((40, 64), device="cuda", generator=gen).to(dt), w, torch.randint(0, 700, (40,), device="cuda", generator=gen)


@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("dt", DTYPES, ids=["bf16", "fp16"])
def test_one_token_of_many(dt, bad):
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy

    x, w, t = _inputs(dt)
    up = torch.rand(40, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4)) + 0.5
    up[7] = 0.0
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss = linear_cross_entropy(a, b, t, reduction="none")
    want = torch.autograd.grad(loss, a, up, retain_graph=True)[0]
    broken = up.clone()
    broken[3] = bad
    dx, dw = torch.autograd.grad(loss, (a, b), broken)
    others = torch.arange(40, device="cuda") != 3
    # the span of fp16 goes by the largest finite number, which may be another one without token 3
    exact = ref.head(x, w, *ref.targets_of(t, -100, 40, 700), 1.0, up.double(), kept=False)[1]
    off = (dx.double() - exact["value"]).abs()[others]
    assert bool((off <= exact["bound"][others]).all())
    assert not bool(torch.isfinite(dx[3]).any()) and not bool(torch.isfinite(dw).any())
    assert torch.equal(want[7], torch.zeros_like(want[7])) and torch.equal(dx[7], want[7])


@pytest.mark.parametrize("dt", DTYPES, ids=["bf16", "fp16"])
@pytest.mark.parametrize("rest", [0.0, 2.0 ** -140])
def test_all_others_are_nothing(dt, rest):
    """The largest finite number is 0, or no normal fp32 number."""
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy

    x, w, t = _inputs(dt)
    for one in (rest, float("inf")):
        up = torch.full((40,), rest, device="cuda")
        up[3] = one
        a = x.clone().requires_grad_()
        dx = torch.autograd.grad(linear_cross_entropy(a, w, t, reduction="none"), a, up)[0]
        others = torch.arange(40, device="cuda") != 3
        assert not bool(dx[others].any())
        assert bool(torch.isfinite(dx[3]).all()) == (one == rest)
