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


def _dw(n, d, v, dt, target, keep=False, lists=0):
    """(its ratio, dw, the exact one) of w's gradient, upstream gradients of 1 to 1.25."""
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy, linear_distill

    gen = torch.Generator(device="cuda").manual_seed(n)
    w = (torch.randn((v, d), device="cuda", generator=gen) * d ** -0.5).to(dt)
    x = torch.randn((n, d), device="cuda", generator=gen).to(dt)
    up = 1 + torch.rand(n, device="cuda", generator=gen) / 4
    b = w.clone().requires_grad_()
    if lists:
        logits = torch.tensor([0.0, 3.0], device="cuda").log1p().expand(n, 2)
        dw, = torch.autograd.grad(linear_distill(x, b, target, logits, reduction="none", keep_logits=keep), b, up)
        true = head_norms.exact(x, w, target, torch.softmax(logits.double(), 1), 1.0, up)
    else:
        dw, = torch.autograd.grad(linear_cross_entropy(x, b, target, reduction="none", keep_logits=keep), b, up)
        true = head_norms.exact(x, w, target[:, None], torch.ones((n, 1), device="cuda"), 1.0, up)
    return _ratio(dw, true[2]), dw, true


@pytest.mark.parametrize("tiles", [0, 7], ids=["large", "small"])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("n,d,v", [(300, 128, 5000), (513, 64, 19044), (2400, 104, 13164), (3000, 488, 4924), (4000, 264, 50021)])
def test_gradients_of_w_that_are_mostly_their_targets(n, d, v, dt, tiles, monkeypatch):
    from triton_kubernetes_amd.ops import loss

    monkeypatch.setattr(loss, "small_products", lambda *a: tiles)
    gen = torch.Generator(device="cuda").manual_seed(v)
    target = torch.randint(0, v, (n,), device="cuda", generator=gen)
    assert _dw(n, d, v, dt, target)[0] <= 1.05
    pairs = torch.randint(0, v, (n, 2), device="cuda", generator=gen)
    assert _dw(n, d, v, dt, pairs, lists=2)[0] <= 1.05


@pytest.mark.parametrize("tiles", [0, 7], ids=["large", "small"])
@pytest.mark.parametrize("n", [500, 1500, 5000])
def test_many_tokens_of_the_same_targets(n, tiles, monkeypatch):
    """Every token's target is one of four neighbours, in one tile, or one at a tile's border: hundreds of
    hits of one tile, and of one row."""
    from triton_kubernetes_amd.ops import loss

    monkeypatch.setattr(loss, "small_products", lambda *a: tiles)
    gen = torch.Generator(device="cuda").manual_seed(n)
    for among in ([700, 701, 702, 703], [255, 256, 511, 512], [0, 2999]):
        target = torch.tensor(among, device="cuda")[torch.randint(0, len(among), (n,), device="cuda", generator=gen)]
        _, dw, (_, _, true, m) = _dw(n, 264, 3000, torch.bfloat16, target)
        rows = torch.tensor(among, device="cuda")
        assert _ratio(dw[rows], true[rows]) <= 1.05


def test_lists_by_pieces_parts_and_masked_tokens(monkeypatch):
    from triton_kubernetes_amd.ops import loss

    n, d, v = 3000, 136, 5003
    gen = torch.Generator(device="cuda").manual_seed(5)
    target = torch.randint(0, v, (n,), device="cuda", generator=gen)
    want = {}
    for tiles in (0, 7):
        monkeypatch.setattr(loss, "small_products", lambda *a, tiles=tiles: tiles)
        for memory, parts in ((2 * n * 1024, 1), (2 * n * 256, 1), (512 << 20, 1), (512 << 20, 7), (512 << 20, 64)):
            monkeypatch.setattr(loss, "DL_BYTES", memory)
            monkeypatch.setattr(loss, "weight_parts", lambda *a, parts=parts: parts)
            for masked in (0.0, 0.7, 0.9):  # 3000, 900 and 300 packed rows: lists, lists, none
                some = torch.where(torch.rand(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(6)) < masked,
                                   -100, target)
                w = (torch.randn((v, d), device="cuda", generator=torch.Generator(device="cuda").manual_seed(7)) * d ** -0.5).bfloat16()
                x = torch.randn((n, d), device="cuda", generator=torch.Generator(device="cuda").manual_seed(8)).bfloat16()
                up = 1 + torch.rand(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(9)) / 4
                b = w.clone().requires_grad_()
                dw, = torch.autograd.grad(loss.linear_cross_entropy(x, b, some, reduction="none"), b, up)
                if masked not in want:
                    keep = some >= 0
                    want[masked] = head_norms.exact(x[keep], w, some[keep][:, None],
                                                    torch.ones((int(keep.sum()), 1), device="cuda"), 1.0, up[keep])[2]
                assert _ratio(dw, want[masked]) <= 1.05, (tiles, memory, parts, masked)
