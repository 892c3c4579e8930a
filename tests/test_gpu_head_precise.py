"""Gradients of the output head's losses whose derivative is multiplied in two 16-bit parts."""

import pytest
import torch

import head_norms

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]
NAMES = {torch.bfloat16: "bf16", torch.float16: "fp16"}


def _inputs(n, d, v, dt, spread=1.0):
    gen = torch.Generator(device="cuda").manual_seed(n + v)
    w = (torch.randn((v, d), device="cuda", generator=gen) * d ** -0.5).to(dt)
    target = torch.randint(0, v, (n,), device="cuda", generator=gen)
    x = spread * torch.randn((n, d), device="cuda", generator=gen)
    x += 6 * torch.rand((n, 1), device="cuda", generator=gen) * w[target].float()
    return x.to(dt), w, target, torch.rand(n, device="cuda", generator=gen) + 0.1, gen


def _run(call, x, w, up):
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss = call(a, b)
    return (loss.detach(), *torch.autograd.grad(loss, (a, b), up))


def _ratio(got, true):
    """Its error over that of rounding the exact result once."""
    return float((got.double() - true).norm() / (true.to(got.dtype).double() - true).norm())


SIZES = [(1, 8, 300), (1, 512, 50021), (48, 512, 1000), (257, 1000, 5003), (300, 77, 1030), (600, 256, 50021), (1500, 1288, 8000)]


@pytest.mark.parametrize("tiles", [None, 0, 7], ids=["rule", "large", "small"])
@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("n,d,v", SIZES)
def test_cross_entropy(n, d, v, dt, tiles, monkeypatch):
    from triton_kubernetes_amd.ops import loss

    if tiles is not None:
        monkeypatch.setattr(loss, "small_products", lambda *a: tiles)
    x, w, target, up, gen = _inputs(n, d, v, dt, 3.0)
    ids = torch.where(torch.rand(n, device="cuda", generator=gen) < 0.2, -1, target) if n > 1 else target
    true = head_norms.exact(x, w, ids[:, None], torch.ones((n, 1), device="cuda"), 1.0, up)
    got = _run(lambda x, w: loss.linear_cross_entropy(x, w, ids, ignore_index=-1, reduction="none", precise_grad=True), x, w, up)
    assert head_norms.wrong(dt, true, got, precise=True) == []
    if d * n > 20_000:  # many roundings; fp32 sums leave 2^-17 of a result where bf16 rounds 2^-9.5
        assert _ratio(got[1], true[1]) <= 1.02 and _ratio(got[2], true[2]) <= 1.02


@pytest.mark.parametrize("tiles", [None, 0, 7], ids=["rule", "large", "small"])
@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("n,d,v,k", [(7, 72, 257, 5), (300, 512, 9999, 33), (333, 1288, 50021, 100), (900, 256, 8000, 64)])
def test_distillation(n, d, v, k, dt, tiles, monkeypatch):
    from triton_kubernetes_amd.ops import loss

    if tiles is not None:
        monkeypatch.setattr(loss, "small_products", lambda *a: tiles)
    x, w, target, up, gen = _inputs(n, d, v, dt)
    ids = torch.randint(-v // 8, v, (n, k), device="cuda", generator=gen)
    ids[:, 0] = ids[:, -1] = target
    logits = 3 * torch.randn((n, k), device="cuda", generator=gen)
    p = torch.softmax(logits.double().masked_fill(ids < 0, -float("inf")) / 2.0, 1)
    true = head_norms.exact(x, w, ids, p, 2.0, up)
    got = _run(lambda x, w: loss.linear_distill(x, w, ids, logits, temperature=2.0, reduction="none", precise_grad=True), x, w, up)
    assert head_norms.wrong(dt, true, got, precise=True) == []
    if d * n > 20_000:
        assert _ratio(got[1], true[1]) <= 1.02 and _ratio(got[2], true[2]) <= 1.02


@pytest.mark.parametrize("tiles", [0, 7], ids=["large", "small"])
def test_pieces_splits_and_parts(tiles, monkeypatch):
    from triton_kubernetes_amd.ops import loss

    n, d, v = 1500, 264, 5003
    monkeypatch.setattr(loss, "small_products", lambda *a: tiles)
    x, w, target, up, _ = _inputs(n, d, v, torch.float16, 3.0)
    true = head_norms.exact(x, w, target[:, None], torch.ones((n, 1), device="cuda"), 1.0, up)
    for memory, groups, parts in ((4 * n * 1024, 30, 1), (4 * n * 256, 1, 1), (loss.DL_BYTES, 4096, 5)):
        monkeypatch.setattr(loss, "DL_BYTES", memory)
        monkeypatch.setattr(loss, "fill", lambda small, groups=groups: groups)
        monkeypatch.setattr(loss, "weight_parts", lambda *a, parts=parts: parts)
        got = _run(lambda x, w: loss.linear_cross_entropy(x, w, target, reduction="none", precise_grad=True), x, w, up)
        assert head_norms.wrong(x.dtype, true, got, precise=True) == []


def test_the_loss_is_the_same_and_each_gradient_alone_too():
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy

    x, w, target, _, _ = _inputs(200, 136, 3000, torch.bfloat16)
    both = _run(lambda x, w: linear_cross_entropy(x, w, target, precise_grad=True), x, w, None)
    assert torch.equal(both[0], linear_cross_entropy(x, w, target))
    for place, (a, b) in enumerate(((x.clone().requires_grad_(), w), (x, w.clone().requires_grad_()))):
        one, = torch.autograd.grad(linear_cross_entropy(a, b, target, precise_grad=True), (a, b)[place])
        assert torch.equal(one, both[1 + place])
    for _ in range(3):
        again = _run(lambda x, w: linear_cross_entropy(x, w, target, precise_grad=True), x, w, None)
        assert all(torch.equal(p, q) for p, q in zip(again, both))


def test_captured_and_replayed():
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy

    x, w, target, _, _ = _inputs(300, 136, 3000, torch.bfloat16)

    def step():
        a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
        loss = linear_cross_entropy(a, b, target, precise_grad=True)
        return (loss.detach(), *torch.autograd.grad(loss, (a, b)))

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(4):
        x.mul_(0.75)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step())), turn


def test_kept_logits_are_refused():
    from triton_kubernetes_amd.ops.loss import LossError, linear_cross_entropy

    x, w, target, _, _ = _inputs(20, 64, 300, torch.bfloat16)
    w.requires_grad_()
    with pytest.raises(LossError, match="kept logits"):
        linear_cross_entropy(x, w, target, keep_logits=True, precise_grad=True)
    linear_cross_entropy(x, w, target, keep_logits=None, precise_grad=True).backward()
