"""The sums of x's gradient by packed rows: only the device knows how many there are, and so into
how many splits of the vocabulary they fall."""

import pytest
import torch

import head_reference as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tiles", [0, 7], ids=["large", "small"])
@pytest.mark.parametrize("rows", [0, 1, 63, 64, 65, 129, 255, 257, 640, 1301])
def test_any_number_of_packed_rows(rows, tiles, monkeypatch):
    from triton_kubernetes_amd.ops import loss

    monkeypatch.setattr(loss, "small_products", lambda *a: tiles)
    n, d, v = 1301, 328, 9001
    gen = torch.Generator(device="cuda").manual_seed(rows)
    w = (torch.randn((v, d), device="cuda", generator=gen) * d ** -0.5).bfloat16()
    x = torch.randn((n, d), device="cuda", generator=gen).bfloat16()
    t = torch.randint(0, v, (n,), device="cuda", generator=gen)
    t[torch.randperm(n, device="cuda", generator=gen)[rows:]] = -100
    a = x.clone().requires_grad_()
    up = torch.rand(n, device="cuda", generator=gen)
    got = loss.linear_cross_entropy(a, w, t, reduction="none")
    dx, = torch.autograd.grad(got, a, up)
    want = ref.head(x, w, *ref.targets_of(t, -100, n, v), 1.0, up.double(), kept=False)
    ref.check("loss", got.detach(), want[0])
    ref.check("dx", dx, want[1])
    # and as a whole: a split too few or too many is far more than two roundings
    off = (dx.double() - want[1]["value"]).norm()
    assert float(off) <= 2 * 2.0 ** -8 * float(want[1]["value"].norm())
