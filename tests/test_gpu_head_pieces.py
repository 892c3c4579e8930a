"""Pieces of the vocabulary that are cut to a whole tile less, so that they stay within their memory."""

import pytest
import torch

import head_norms

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("small", [0, 7])
def test_many_tokens_in_pieces_of_one_tile(small, monkeypatch):
    from triton_kubernetes_amd.ops import loss

    n, d, v = 6000, 72, 700
    monkeypatch.setattr(loss, "DL_BYTES", 2 * n * loss.TILE)
    monkeypatch.setattr(loss, "small_products", lambda *a: small)
    assert loss.pieces(n, v) == loss.TILE
    gen = torch.Generator(device="cuda").manual_seed(5)
    w = (torch.randn((v, d), device="cuda", generator=gen) / 8).bfloat16().requires_grad_()
    x = (3 * torch.randn((n, d), device="cuda", generator=gen)).bfloat16().requires_grad_()
    t = torch.randint(0, v, (n,), device="cuda", generator=gen)
    up = torch.rand(n, device="cuda", generator=gen) + 0.1
    got = loss.linear_cross_entropy(x, w, t, reduction="none")
    true = head_norms.exact(x.detach(), w.detach(), t[:, None], torch.ones((n, 1), device="cuda"), 1.0, up)
    assert head_norms.wrong(x.dtype, true, (got.detach(), *torch.autograd.grad(got, (x, w), up))) == []
