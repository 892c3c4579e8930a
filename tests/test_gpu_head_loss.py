"""The output head's losses (csrc/tk_loss.hip) on the MI355X against their definition in 64
bits (tests/head_reference.py derives the tolerances)."""

import pytest
import torch

import head_reference as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]
NAMES = {torch.bfloat16: "bf16", torch.float16: "fp16"}


def _gen(*key):
    return torch.Generator(device="cuda").manual_seed(hash(key) % (1 << 31))


def _inputs(n, d, v, dt, gen, sure=4.0):
    w = (torch.randn((v, d), device="cuda", generator=gen) * d ** -0.5).to(dt)
    t = torch.randint(0, v, (n,), device="cuda", generator=gen)
    x = torch.randn((n, d), device="cuda", generator=gen)
    x += sure * torch.rand((n, 1), device="cuda", generator=gen) * w[t].float()
    return x.to(dt), w, t


def _run(call, x, w, g):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = call(x, w)
    return (loss.detach(), *torch.autograd.grad(loss, (x, w), g))


def _against(call, x, w, ids, p, t=1.0, reduction="none", gen=None, kept=True):
    n = x.shape[0]
    count = max(1, int((ids >= 0).any(1).sum()))
    up = torch.rand(n, device="cuda", generator=gen) - 0.3 if reduction == "none" else torch.tensor(0.75, device="cuda")
    loss, dx, dw = _run(call, x, w, up)
    g = up.double() if reduction == "none" else torch.full((n,), 0.75, device="cuda", dtype=torch.float64)
    if reduction == "mean":
        g = g / count
    want, wdx, wdw = ref.head(x, w, ids, p, t, g, kept)
    if reduction != "none":
        over = 1 if reduction == "sum" else count
        want = dict(value=want["value"].sum() / over, bound=(want["bound"].sum() + want["value"].abs().sum() * 1e-6) / over)
    ref.check("loss", loss, want)
    ref.check("dx", dx, wdx)
    ref.check("dw", dw, wdw)
    return loss, dx, dw


SIZES = [(1, 8, 1), (1, 64, 300), (2, 72, 256), (5, 72, 257), (48, 512, 1000), (255, 264, 511), (257, 1000, 5003),
         (300, 77, 1030), (64, 8, 70001), (513, 128, 513), (1, 4096, 2000)]


@pytest.mark.parametrize("tiles", [0, 7], ids=["large", "small"])
@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("kept", [True, False], ids=["kept", "again"])
@pytest.mark.parametrize("n,d,v", SIZES)
def test_cross_entropy(n, d, v, dt, kept, tiles, monkeypatch):
    from triton_kubernetes_amd.ops import loss
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy

    monkeypatch.setattr(loss, "small_products", lambda *a: tiles)
    monkeypatch.setattr(loss, "keeps", lambda *a: kept)
    gen = _gen(n, d, v)
    x, w, t = _inputs(n, d, v, dt, gen)
    for reduction in ("none", "mean"):
        _against(lambda x, w: linear_cross_entropy(x, w, t, reduction=reduction), x, w, *ref.targets_of(t, -100, n, v),
                 reduction=reduction, gen=gen, kept=kept)


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("kept", [True, False], ids=["kept", "again"])
@pytest.mark.parametrize("n,d,v,k,temp", [(1, 64, 300, 1, 1.0), (7, 72, 257, 5, 2.0), (130, 264, 1111, 64, 0.7),
                                          (40, 77, 5003, 130, 2.0), (300, 512, 999, 33, 1.0)])
@pytest.mark.parametrize("tiles", [0, 7], ids=["large", "small"])
def test_distill(n, d, v, k, temp, dt, kept, tiles, monkeypatch):
    from triton_kubernetes_amd.ops import loss
    from triton_kubernetes_amd.ops.loss import linear_distill

    monkeypatch.setattr(loss, "small_products", lambda *a: tiles)
    monkeypatch.setattr(loss, "keeps", lambda *a: kept)
    gen = _gen(n, d, v, k)
    x, w, _ = _inputs(n, d, v, dt, gen)
    ids = torch.randint(0, v, (n, k), device="cuda", generator=gen)  # the same id twice among them
    ids[torch.rand((n, k), device="cuda", generator=gen) < 0.2] = -1
    ids[-1] = -5  # no entry at all
    logits = torch.randn((n, k), device="cuda", generator=gen) * 3
    logits[torch.rand((n, k), device="cuda", generator=gen) < 0.1] = -float("inf")
    if n > 2:
        logits[1] = -float("inf")
    for reduction in ("none", "sum"):
        _against(lambda x, w: linear_distill(x, w, ids, logits, temperature=temp, reduction=reduction), x, w,
                 *ref.teacher_of(ids, logits, temp), t=temp, reduction=reduction, gen=gen, kept=kept)


def test_one_id_listed_many_times():
    from triton_kubernetes_amd.ops.loss import linear_distill

    gen = _gen(3)
    x, w, t = _inputs(9, 64, 400, torch.bfloat16, gen)
    ids = t[:, None].expand(9, 70)
    logits = torch.randn((9, 70), device="cuda", generator=gen)
    _against(lambda x, w: linear_distill(x, w, ids, logits, reduction="none"), x, w, *ref.teacher_of(ids, logits, 1.0),
             gen=gen)


@pytest.mark.parametrize("kept", [0.0, 0.02, 0.5])
def test_masked_rows_hold_anything(kept):
    """Infinities and NaN in a masked row reach no loss and no gradient, and its gradient is 0."""
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy

    n, d, v = 700, 128, 900
    gen = _gen(5, int(kept * 100))
    x, w, t = _inputs(n, d, v, torch.bfloat16, gen)
    mask = torch.rand(n, device="cuda", generator=gen) >= kept
    t[mask] = 7  # the number that is ignored may be a vocabulary entry
    t[~mask & (t == 7)] = 8
    x[mask] = torch.tensor([float("nan"), float("inf"), -float("inf"), 3e38], device="cuda").repeat(d // 4).to(x.dtype)
    loss, dx, dw = _against(lambda x, w: linear_cross_entropy(x, w, t, ignore_index=7, reduction="none"), x, w,
                            *ref.targets_of(t, 7, n, v), gen=gen)
    assert bool((loss[mask] == 0).all()) and bool((dx[mask] == 0).all())
    mean = linear_cross_entropy(x, w, t, ignore_index=7)
    assert bool(torch.isfinite(mean))
    if kept == 0.0:
        assert float(mean) == 0 and not bool(dw.any())


def test_target_outside_the_vocabulary_is_nan():
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy, linear_distill

    x, w, t = _inputs(6, 64, 300, torch.bfloat16, _gen(6))
    t[2], t[4] = 300, -1
    loss, dx, _ = _run(lambda x, w: linear_cross_entropy(x, w, t, reduction="none"), x, w, torch.ones(6, device="cuda"))
    bad = torch.tensor([0, 0, 1, 0, 1, 0], device="cuda", dtype=torch.bool)
    assert torch.equal(loss.isnan(), bad) and torch.equal(dx.isnan().any(1), bad)
    ids = torch.tensor([[1, 2], [300, -1], [-1, -1], [3, 1 << 40], [4, 4], [0, -9]], device="cuda")
    loss = linear_distill(x, w, ids, torch.zeros((6, 2), device="cuda"), reduction="none")
    assert loss.isnan().tolist() == [False, True, False, True, False, False] and float(loss[2]) == 0


def test_logits_far_apart():
    """Logits of +-hundreds: the sums keep a running maximum."""
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy

    gen = _gen(8)
    x, w, t = _inputs(33, 64, 3000, torch.bfloat16, gen)
    x = x * 100
    _against(lambda x, w: linear_cross_entropy(x, w, t, reduction="none"), x, w, *ref.targets_of(t, -100, 33, 3000),
             gen=gen)


def test_rows_of_very_different_weight_fp16():
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy

    gen = _gen(9)
    x, w, t = _inputs(40, 64, 500, torch.float16, gen)
    up = torch.logspace(-4, 3, 40, device="cuda")
    got = _run(lambda x, w: linear_cross_entropy(x, w, t, reduction="none"), x, w, up)
    want = ref.head(x, w, *ref.targets_of(t, -100, 40, 500), 1.0, up)
    for name, g, r in zip(("loss", "dx", "dw"), got, want):
        ref.check(name, g, r)


def _layouts():
    def sliced(a):
        return torch.cat((a, a), 1)[:, :a.shape[1]]

    def offset(a):
        b = torch.empty(a.numel() + 1, device="cuda", dtype=a.dtype)[1:].view(a.shape)
        return b.copy_(a)

    def turned(a):
        return a.t().contiguous().t()

    def spread(a):
        b = torch.zeros((*a.shape, 2), device="cuda", dtype=a.dtype)
        b[..., 0] = a
        return b[..., 0]

    return [sliced, offset, turned, spread]


@pytest.mark.parametrize("layout", _layouts(), ids=lambda f: f.__name__)
def test_strides_and_alignment(layout):
    """Any layout of x and w gives the contiguous result to the bit."""
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy

    x, w, t = _inputs(60, 136, 777, torch.bfloat16, _gen(10))
    call = lambda x, w: linear_cross_entropy(x, w, t)  # noqa: E731
    want = _run(call, x, w, None)
    for a, b in ((layout(x), w), (x, layout(w)), (layout(x), layout(w))):
        for got, ex in zip(_run(call, a, b, None), want):
            assert torch.equal(got, ex)


def test_leading_dimensions_and_expanded_gradients():
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy, linear_distill

    x, w, t = _inputs(24, 64, 300, torch.float16, _gen(11))
    up = torch.rand(24, device="cuda")
    for flat, shaped in ((up, up.view(2, 3, 4)), (up[:1].expand(24), up[:1].expand(24).view(2, 3, 4)),
                         (up.bfloat16().float(), up.bfloat16().float().view(4, 3, 2).transpose(0, 2))):
        if shaped.shape == (2, 3, 4) and not shaped.is_contiguous():
            flat = shaped.reshape(-1)
        a = _run(lambda x, w: linear_cross_entropy(x, w, t, reduction="none"), x, w, flat)
        b = _run(lambda x, w: linear_cross_entropy(x.view(2, 3, 4, 64), w, t.view(2, 3, 4).int(), reduction="none"), x, w,
                 shaped)
        assert b[0].shape == (2, 3, 4) and torch.equal(a[0], b[0].reshape(-1))
        assert torch.equal(a[1], b[1]) and torch.equal(a[2], b[2])
    ids = torch.randint(0, 300, (24, 3), device="cuda")
    loss = linear_distill(x.view(6, 4, 64), w, ids.view(6, 4, 3), torch.zeros((6, 4, 3), device="cuda").half(),
                          reduction="none")
    assert torch.equal(loss.reshape(-1), linear_distill(x, w, ids, torch.zeros((24, 3), device="cuda"), reduction="none"))
    one = linear_cross_entropy(x[0], w, t[0])  # a single token without a batch
    assert one.shape == () and torch.equal(one, linear_cross_entropy(x[:1], w, t[:1]))


def test_nothing_to_learn_from():
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy, linear_distill

    x, w, t = _inputs(4, 64, 300, torch.bfloat16, _gen(12))
    for call, rows in ((lambda x, w: linear_cross_entropy(x, w, t[:0]), 0),
                       (lambda x, w: linear_distill(x, w, t[:, None][:, :0], x[:, :0].detach()), 4)):
        loss, dx, dw = _run(call, x[:rows], w, None)
        assert float(loss) == 0 and not bool(dx.any()) and not bool(dw.any()) and dx.shape == x[:rows].shape


def test_pieces_and_splits(monkeypatch):
    """A vocabulary in many pieces, its last one ragged, and split sums of x's gradient."""
    from triton_kubernetes_amd.ops import loss

    n, d, v = 300, 264, 5003
    monkeypatch.setattr(loss, "DL_BYTES", 2 * n * 1024)
    assert loss.pieces(n, v) == 1024
    gen = _gen(13)
    x, w, t = _inputs(n, d, v, torch.float16, gen)
    call = lambda x, w: loss.linear_cross_entropy(x, w, t, reduction="none")  # noqa: E731
    for groups, tiles in ((1, 0), (30, 7), (14, 0), (4096, 2), (4096, 5)):
        monkeypatch.setattr(loss, "fill", lambda small, groups=groups: groups)
        monkeypatch.setattr(loss, "small_products", lambda *a, tiles=tiles: tiles)
        _against(call, x, w, *ref.targets_of(t, -100, n, v), gen=gen)


def test_only_the_gradients_asked_for():
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy

    x, w, t = _inputs(70, 64, 600, torch.bfloat16, _gen(14))
    loss, dx, dw = _run(lambda x, w: linear_cross_entropy(x, w, t), x, w, None)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    linear_cross_entropy(a, w, t).backward()
    linear_cross_entropy(x, b, t).backward()
    assert torch.equal(a.grad, dx) and torch.equal(b.grad, dw)
    assert not linear_cross_entropy(x, w, t).requires_grad
    again = linear_cross_entropy(a, b, t)
    again.backward()
    assert torch.equal(b.grad, dw + dw)  # accumulated by autograd
    with pytest.raises(RuntimeError):
        again.backward()


def test_weight_changed_between_the_passes_is_refused():
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy

    x, w, t = _inputs(8, 64, 300, torch.bfloat16, _gen(15))
    w.requires_grad_()
    loss = linear_cross_entropy(x, w, t)
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_gradient_is_the_losss_slope():
    """Central differences of the kernel's own loss: steps of 2^-6 that bf16 holds exactly."""
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy

    n, d, v, h = 12, 64, 300, 2.0 ** -6
    gen = _gen(16)
    x = torch.randint(-32, 33, (n, d), device="cuda", generator=gen).float() / 32
    w = torch.randint(-32, 33, (v, d), device="cuda", generator=gen).float() / 64
    t = torch.randint(0, v, (n,), device="cuda", generator=gen)
    step = torch.randint(-1, 2, (n, d), device="cuda", generator=gen).float()
    turn = torch.randint(-1, 2, (v, d), device="cuda", generator=gen).float()

    def loss(x, w):
        assert torch.equal(x.bfloat16().float(), x) and torch.equal(w.bfloat16().float(), w)
        return linear_cross_entropy(x.bfloat16(), w.bfloat16(), t, reduction="sum")

    def true(x, w):
        return -(torch.log_softmax(x.double() @ w.double().T, 1).gather(1, t[:, None])).sum()

    _, dx, dw = _run(lambda x, w: linear_cross_entropy(x, w, t, reduction="sum"), x.bfloat16(), w.bfloat16(), None)
    a, b = x.double().requires_grad_(), w.double().requires_grad_()
    ex, ew = torch.autograd.grad(true(a, b), (a, b))
    for grad, exact, move in ((dx, ex, (step, None)), (dw, ew, (None, turn))):
        at = lambda s: (x + s * move[0] if move[0] is not None else x, w + s * move[1] if move[1] is not None else w)  # noqa: E731
        along = move[0] if move[0] is not None else move[1]
        slope = (loss(*at(h)) - loss(*at(-h))).double() / (2 * h)
        formula = (true(*at(h)) - true(*at(-h))) / (2 * h)
        # each loss of ~6 a token is good to 2^-18 of itself; the difference divides by 2h
        tol = 2 * n * 12 * 2.0 ** -18 / (2 * h)
        assert abs(float(slope - formula)) <= tol, (float(slope), float(formula), tol)
        # the gradient: 2 roundings an element (dl's and the result's)
        got, want = (grad.double() * along).sum(), (exact * along).sum()
        curve = abs(float(formula - want))  # what the step of h costs
        assert abs(float(slope - got)) <= tol + curve + 2 * 2.0 ** -8 * float((exact.abs() * along.abs()).sum()) + 0.05


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
def test_same_bits_every_time(dt):
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy

    x, w, t = _inputs(600, 256, 5000, dt, _gen(17))
    call = lambda x, w: linear_cross_entropy(x, w, t)  # noqa: E731
    first = _run(call, x, w, None)
    for _ in range(3):
        for got, want in zip(_run(call, x, w, None), first):
            assert torch.equal(got, want)


def test_runs_on_torchs_current_stream():
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy

    x, w, t = _inputs(300, 128, 2000, torch.bfloat16, _gen(18))
    want = _run(lambda x, w: linear_cross_entropy(x, w, t), x * 2, w, None)
    s, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(other):  # two calls at once, each with its own workspaces
        late = _run(lambda x, w: linear_cross_entropy(x, w, t), x * 2, w, None)
    with torch.cuda.stream(s):
        got = _run(lambda x, w: linear_cross_entropy(x, w, t), x * 2, w, None)
    torch.cuda.synchronize()
    for a, b, c in zip(got, late, want):
        assert torch.equal(a, c) and torch.equal(b, c)


def test_captured_and_replayed():
    """Both directions in a graph: each replay follows what its inputs then hold."""
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy, linear_distill

    gen = _gen(19)
    sets = [_inputs(200, 128, 1500, torch.bfloat16, gen) for _ in range(3)]
    for s in sets[1:]:
        s[2][torch.rand(200, device="cuda", generator=gen) < 0.5] = -100
    ids = torch.randint(0, 1500, (200, 9), device="cuda", generator=gen)
    logits = torch.randn((200, 9), device="cuda", generator=gen)
    x, w, t = (a.clone() for a in sets[0])

    def both(x, w, t):
        x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
        loss = linear_cross_entropy(x, w, t)
        one = torch.autograd.grad(loss, (x, w))
        soft = linear_distill(x, w, ids, logits, temperature=2.0)
        return (loss.detach(), *one, soft.detach(), *torch.autograd.grad(soft, (x, w)))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        both(x, w, t)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(x, w, t)
    for turn in range(6):
        s = sets[turn % 3]
        for a, b in zip((x, w, t), s):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, both(*s)):
            assert torch.equal(got, want), turn


def test_gradient_of_a_shared_weight():
    """A weight used twice, and an x that is the sum of two: autograd adds what each use gives."""
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy

    x, w, t = _inputs(50, 64, 400, torch.bfloat16, _gen(20))
    _, dx, dw = _run(lambda x, w: linear_cross_entropy(x, w, t), x, w, None)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    (linear_cross_entropy(a, b, t) + linear_cross_entropy(a, b, t)).backward()
    assert torch.equal(a.grad, dx + dx) and torch.equal(b.grad, dw + dw)
    row = x[:1].clone().requires_grad_()
    linear_cross_entropy(row.expand(50, 64), w, t, reduction="sum").backward()
    each = _run(lambda x, w: linear_cross_entropy(x, w, t, reduction="sum"), x[:1].expand(50, 64).contiguous(), w, None)
    assert torch.allclose(row.grad.float()[0], each[1].float().sum(0), rtol=2.0 ** -7, atol=1e-2)


def test_long_offsets():
    """A weight of more than 2^32 bytes: entries past the 32-bit offsets count, forward and back."""
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy

    d, v, n = 16384, 140_000, 3
    w = torch.zeros((v, d), device="cuda", dtype=torch.bfloat16)
    x = torch.zeros((n, d), device="cuda", dtype=torch.bfloat16)
    x[:, 0] = 4.0
    w[v - 2, 0] = 3.0  # logit 12
    t = torch.tensor([v - 2, v - 1, 0], device="cuda")
    loss, dx, dw = _run(lambda x, w: linear_cross_entropy(x, w, t, reduction="none"), x, w, torch.ones(n, device="cuda"))
    import math

    lse = math.log(v - 1 + math.exp(12.0))
    assert torch.allclose(loss.double().cpu(), torch.tensor([lse - 12, lse, lse], dtype=torch.float64), rtol=0, atol=1e-4)
    q, rest = math.exp(12 - lse), math.exp(-lse)
    assert abs(float(dx[1, 0]) / (3 * q) - 1) < 2.0 ** -7
    got = dw[:, 0].double().cpu()
    for at, value in ((v - 2, 4 * (3 * q - 1)), (v - 1, 4 * (3 * rest - 1)), (0, 4 * (3 * rest - 1)), (7, 12 * rest)):
        assert abs(float(got[at]) - value) <= 3 * 2.0 ** -8 * 4, (at, float(got[at]), value)
    assert not bool(dw[:, 1:].any())


@pytest.mark.parametrize("distill", [False, True], ids=["target", "teacher"])
@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
def test_the_targets_derivative_is_not_rounded_for_few_tokens(dt, distill):
    """One token: w's gradient at its target is (q - 1) x.  With q <= 2^-5 from a logit off by at most
    2^-12, q - 1 is good to 2^-16, so that little but the result's own rounding is left of it
    (a 16-bit q - 1 alone would be off by up to half a step more)."""
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy, linear_distill

    d, v = 2048, 300
    gen = _gen(21, int(distill))
    x, w, t = _inputs(1, d, v, dt, gen, sure=0.0)
    if distill:
        call = lambda x, w: linear_distill(x, w, t[:, None], torch.zeros((1, 1), device="cuda"))  # noqa: E731
    else:
        call = lambda x, w: linear_cross_entropy(x, w, t)  # noqa: E731
    _, _, dw = _run(call, x, w, None)
    q = torch.softmax(x.double() @ w.double().T, 1)[0, t[0]]
    assert float(q) <= 2.0 ** -5
    true = (q - 1) * x.double()[0]
    # (fp16 results under 2^-14 have absolute steps of 2^-24)
    off = (dw[t[0]].double() - true).abs() - true.abs() * (ref.U[dt] + 2.0 ** -15) - 2.0 ** -25
    assert float(off.max()) <= 0


def test_a_teachers_list_of_the_lowest_value_is_uniform():
    """A mask of fp32's lowest value, which a division by the temperature would turn into -inf."""
    from triton_kubernetes_amd.ops.loss import linear_distill

    gen = _gen(22)
    x, w, t = _inputs(3, 64, 400, torch.bfloat16, gen)
    ids = torch.stack((t, (t + 1) % 400), 1)
    low = torch.finfo(torch.float32).min
    logits = torch.tensor([[low, low], [0.0, low], [-float("inf"), low]], device="cuda")
    for temp in (0.5, 1.0):
        got = _run(lambda x, w: linear_distill(x, w, ids, logits, temperature=temp, reduction="none"), x, w,
                   torch.ones(3, device="cuda"))
        same = torch.tensor([[0.0, 0.0], [0.0, -1e4], [-float("inf"), 0.0]], device="cuda")
        want = _run(lambda x, w: linear_distill(x, w, ids, same, temperature=temp, reduction="none"), x, w,
                    torch.ones(3, device="cuda"))
        for a, b in zip(got, want):
            assert torch.equal(a, b) and bool(torch.isfinite(a).all())


def test_many_tokens_with_gaps(monkeypatch):
    """More tokens than two rows a wave pack, most of them masked; those that are left are the last
    ones of a run, the first and the last token among them."""
    from triton_kubernetes_amd.ops import loss
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy

    # (the tiles go by all tokens, and small ones add the same numbers in another order)
    monkeypatch.setattr(loss, "small_products", lambda *a: 0)
    n, d, v = 100_003, 16, 40
    gen = _gen(23)
    x, w, t = _inputs(n, d, v, torch.bfloat16, gen)
    keep = torch.rand(n, device="cuda", generator=gen) < 0.01
    keep[[0, n - 1]] = True
    t[~keep] = -100
    loss, dx, dw = _run(lambda x, w: linear_cross_entropy(x, w, t, reduction="none"), x, w, torch.ones(n, device="cuda"))
    few = _run(lambda x, w: linear_cross_entropy(x, w, t[keep], reduction="none"), x[keep], w,
               torch.ones(int(keep.sum()), device="cuda"))
    assert torch.equal(loss[keep], few[0]) and not bool(loss[~keep].any())
    assert torch.equal(dx[keep], few[1]) and not bool(dx[~keep].any())
    assert torch.equal(dw, few[2])


def test_more_listed_entries_than_a_launch_has_waves():
    from triton_kubernetes_amd.ops.loss import linear_distill

    n, d, v, k = 65536, 8, 1024, 1024
    gen = _gen(24)
    x, w, _ = _inputs(n, d, v, torch.bfloat16, gen)
    ids = torch.arange(k, device="cuda").expand(n, k)
    logits = torch.randn((n, k), device="cuda", generator=gen)
    loss = linear_distill(x, w, ids, logits, reduction="none")
    at = torch.cat((torch.arange(300), torch.arange(n - 300, n))).to("cuda")
    want = ref.head(x[at], w, ids[at], *[ref.teacher_of(ids[at], logits[at], 1.0)[1]], 1.0, torch.ones(600, device="cuda"))
    ref.check("loss", loss[at], want[0])


def test_a_weight_of_one_row_with_any_stride():
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy

    gen = _gen(25)
    x, w, t = _inputs(4, 64, 1, torch.bfloat16, gen)
    lone = torch.empty((1, 128), device="cuda", dtype=w.dtype)
    lone[:, ::2] = w
    for other in (w[0].expand(1, 64), lone[:, ::2], lone[0, ::2].expand(1, 64)):
        # the only entry there is: 0, but for the logit, which the kernels add up in two orders
        _against(lambda x, w: linear_cross_entropy(x, w, t, reduction="none"), x, other, *ref.targets_of(t, -100, 4, 1),
                 gen=gen)


def test_capture_is_refused_while_an_eager_graph_of_the_same_leaves_lives():
    """torch would leave the eager stream unjoined in the capture, which ends the process."""
    from triton_kubernetes_amd.ops.loss import LossError, linear_cross_entropy

    x, w, t = _inputs(40, 64, 300, torch.bfloat16, _gen(26))
    x.requires_grad_()
    w.requires_grad_()
    alive = linear_cross_entropy(x, w, t)
    for leaves in ((x, w), (x.detach(), w), (x, w.detach())):
        with pytest.raises(LossError, match="eager graph"), torch.cuda.graph(torch.cuda.CUDAGraph()):
            linear_cross_entropy(*leaves, t)
    with torch.cuda.stream(torch.cuda.Stream()):  # another stream alone is no trouble
        torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
        linear_cross_entropy(x, w, t)
        torch.cuda.current_stream().synchronize()
    want = torch.autograd.grad(alive, (x, w))
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = torch.autograd.grad(linear_cross_entropy(x, w, t), (x, w))
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_first_call_of_a_process_may_be_a_captured_one():
    import subprocess
    import sys

    code = """
import torch
from triton_kubernetes_amd.ops.gemv import gemv_w4, pack_w4
from triton_kubernetes_amd.ops.loss import linear_cross_entropy
gen = torch.Generator(device="cuda").manual_seed(1)
w = torch.randn((500, 128), device="cuda", generator=gen).bfloat16().requires_grad_()
x = torch.randn((70, 128), device="cuda", generator=gen).bfloat16().requires_grad_()
t = torch.randint(0, 500, (70,), device="cuda", generator=gen)
codes = pack_w4(torch.randint(0, 16, (500, 128), device="cuda", generator=gen, dtype=torch.uint8))
scales = torch.ones((500, 1), device="cuda", dtype=torch.bfloat16)
def run():
    loss = linear_cross_entropy(x, w, t)
    return (loss.detach(), *torch.autograd.grad(loss, (x, w)), gemv_w4(x.detach()[:3], codes, scales),
            gemv_w4(x.detach()[:40], codes, scales))
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = run()
for _ in range(3):
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, run()))
print("same")
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100)
    assert done.returncode == 0 and done.stdout.strip().endswith("same"), done.stderr[-2000:]


def test_keep_logits_decides_what_stays_between_the_passes():
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy, linear_distill

    n, d, v = 300, 64, 20_000
    gen = _gen(27)
    x, w, t = _inputs(n, d, v, torch.bfloat16, gen)
    x.requires_grad_()
    logits = torch.zeros((n, 1), device="cuda")
    for call in (lambda **k: linear_cross_entropy(x, w, t, **k), lambda **k: linear_distill(x, w, t[:, None], logits, **k)):
        held, losses, grads = [], [], []
        for keep in (False, True, None):
            torch.cuda.synchronize()
            before = torch.cuda.memory_allocated()
            loss = call(keep_logits=keep)
            held.append(torch.cuda.memory_allocated() - before)
            first = torch.autograd.grad(loss, x, retain_graph=True)[0]
            assert torch.equal(first, torch.autograd.grad(loss, x)[0])  # the kept logits stay as they are
            losses.append(loss.detach())
            grads.append(first.float())
            del loss
        assert held[0] < 2 * n * v <= held[1] == held[2]
        assert torch.equal(losses[0], losses[1]) and torch.equal(grads[1], grads[2])
        # both round the derivative to 16 bits; one half step 2^-8 of each, and the result's
        size = (torch.softmax(x.detach().float() @ w.float().T, 1).abs() @ w.float().abs() + w[t].float().abs()) / n
        assert bool(((grads[0] - grads[1]).abs() <= 4 * 2.0 ** -8 * size).all())
        with torch.no_grad():
            before = torch.cuda.memory_allocated()
            loss = call(keep_logits=True)  # without a backward pass nothing is kept
            assert torch.cuda.memory_allocated() - before < 2 * n * v


@pytest.mark.parametrize("n,d,v,masked", [(300, 136, 70, 0.0), (2049, 72, 300, 0.0), (1500, 77, 130, 0.7),
                                          (1500, 77, 130, 1.0), (4096, 256, 64, 0.98)])
@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
def test_weight_gradient_in_parts(n, d, v, masked, dt, monkeypatch):
    """Tokens split for w's gradient, parts without any token among them."""
    from triton_kubernetes_amd.ops import loss

    gen = _gen(28, n, d)
    x, w, t = _inputs(n, d, v, dt, gen)
    t[torch.rand(n, device="cuda", generator=gen) < masked] = -100
    call = lambda x, w: loss.linear_cross_entropy(x, w, t, reduction="none")  # noqa: E731
    monkeypatch.setattr(loss, "small_products", lambda *a: 7)
    assert n < 512 or loss.weight_parts(n, d, v) > 1
    for parts in (loss.weight_parts(n, d, v), 2, 64):
        monkeypatch.setattr(loss, "weight_parts", lambda *a, parts=parts: parts)
        _against(call, x, w, *ref.targets_of(t, -100, n, v), gen=gen)


@pytest.mark.parametrize("n,d,v,dt", [(3, 65536, 300, torch.bfloat16), (3, 65535, 300, torch.float16),
                                      (1 << 20, 8, 16, torch.bfloat16), (2, 8, 1 << 24, torch.float16),
                                      (17, 9, 1 << 22, torch.bfloat16)])
def test_largest_sizes(n, d, v, dt):
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy

    gen = _gen(29, n, d)
    x, w, t = _inputs(n, d, v, dt, gen)
    for keep in (True, False):
        _against(lambda x, w: linear_cross_entropy(x, w, t, reduction="none", keep_logits=keep), x, w,
                 *ref.targets_of(t, -100, n, v), gen=gen, kept=keep)
        torch.cuda.empty_cache()


def test_sizes_past_a_launch_are_refused():
    from triton_kubernetes_amd.ops.loss import LossError, linear_cross_entropy

    x = torch.zeros((1, 16), device="cuda", dtype=torch.bfloat16).expand(1 << 20, 16)
    t = torch.zeros(1, device="cuda", dtype=torch.int64).expand(1 << 20)
    w = torch.zeros((1 << 19, 16), device="cuda", dtype=torch.bfloat16)
    with pytest.raises(LossError, match="tokens x vocabulary"):
        linear_cross_entropy(x, w, t)
    wide = torch.zeros((1, 16384), device="cuda", dtype=torch.bfloat16)
    with pytest.raises(LossError, match="tokens x width"):
        linear_cross_entropy(wide.expand(1 << 20, 16384), wide, t)


def test_a_second_derivative_is_refused():
    from triton_kubernetes_amd.ops.loss import LossError, linear_cross_entropy

    x, w, t = _inputs(20, 64, 300, torch.bfloat16, _gen(30))
    x.requires_grad_()
    want = torch.autograd.grad(linear_cross_entropy(x, w, t), x)[0]
    dx = torch.autograd.grad(linear_cross_entropy(x, w, t), x, create_graph=True)[0]
    assert torch.equal(dx, want)
    with pytest.raises(RuntimeError):  # torch's own: x is nothing that dx was made from
        torch.autograd.grad(dx.float().sum(), x)
    w.requires_grad_()
    dw = torch.autograd.grad(linear_cross_entropy(x, w, t), w, create_graph=True)[0]
    with pytest.raises(LossError, match="second derivative"):
        torch.autograd.grad(dw.float().sum(), w)
    loss = linear_cross_entropy(x, w, t)  # a penalty of the gradient would have none otherwise, silently
    dx = torch.autograd.grad(loss, x, create_graph=True)[0]
    with pytest.raises(LossError, match="second derivative"):
        (loss + dx.float().norm()).backward()
