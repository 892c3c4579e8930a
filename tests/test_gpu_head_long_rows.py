"""Large tiles over few tokens with very long rows of the logits' derivative, whose places past the
last token come near 32 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,v", [(65, 6_100_000), (70, 5_500_000)])
def test_rows_of_millions_of_entries(n, v):
    from triton_kubernetes_amd.ops import loss

    d = 64
    assert n * d * v > 3 << 32 and not loss.small_products(n, d, v) & 2
    assert loss.pieces(n, v) >= v  # one piece: a row is 2 v bytes, 192 of them past 2^31
    gen = torch.Generator(device="cuda").manual_seed(n)
    w = (torch.randn((v, d), device="cuda", generator=gen) / 4).bfloat16()
    x = torch.randn((n, d), device="cuda", generator=gen).bfloat16().requires_grad_()
    t = torch.randint(0, v, (n,), device="cuda", generator=gen)
    up = torch.rand(n, device="cuda", generator=gen) + 0.5
    got, = torch.autograd.grad(loss.linear_cross_entropy(x, w, t, reduction="none"), x, up)
    parts = [w[a:a + 500_000].double() for a in range(0, v, 500_000)]
    z = [x.detach().double() @ part.T for part in parts]
    lse = torch.logsumexp(torch.stack([torch.logsumexp(b, 1) for b in z]), 0)
    dx = sum(torch.exp(b - lse[:, None]) @ part for b, part in zip(z, parts)) - w[t].double()
    dx *= up.double()[:, None]
    off = (got.double() - dx).norm(dim=1) / dx.norm(dim=1)
    assert float(off.max()) <= 2 * 2.0 ** -8
    torch.cuda.empty_cache()


def test_few_tokens_in_large_tiles_are_refused(monkeypatch):
    """What the rules for tiles never ask for."""
    from triton_kubernetes_amd.ops import loss

    monkeypatch.setattr(loss, "small_products", lambda *a: 0)
    w = torch.zeros((10_000_000, 8), device="cuda", dtype=torch.bfloat16)
    x = torch.zeros((2, 8), device="cuda", dtype=torch.bfloat16, requires_grad=True)
    got = loss.linear_cross_entropy(x, w, torch.zeros(2, device="cuda", dtype=torch.int64))
    with pytest.raises(loss.LossError, match="too long"):
        got.backward()
