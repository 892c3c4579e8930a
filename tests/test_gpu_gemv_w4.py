"""4-bit matrix-vector products (csrc/tk_gemv_w4.hip) on the MI355X against their definition
in 64 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]
NAMES = {torch.bfloat16: "bf16", torch.float16: "fp16"}
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _gen(*key):
    return torch.Generator(device="cuda").manual_seed(hash(key) % (1 << 31))


def _weight(n, k, group, dt, zeros, gen, exact=False):
    codes = torch.randint(0, 16, (n, k), device="cuda", generator=gen, dtype=torch.uint8)
    zero = torch.randint(0, 16, (n, k // group), device="cuda", generator=gen, dtype=torch.uint8) if zeros else None
    if exact:  # powers of two
        scales = 2.0 ** torch.randint(-1, 2, (n, k // group), device="cuda", generator=gen)
    else:
        scales = torch.rand((n, k // group), device="cuda", generator=gen) + 0.1
    return codes, scales.to(dt), zero


def _true(codes, scales, zero):
    n, groups = scales.shape
    z = 8.0 if zero is None else zero.double()[:, :, None]
    return ((codes.double().view(n, groups, -1) - z) * scales.double()[:, :, None]).reshape(n, -1)


EXACT = [(1, 1, 32, 32, False), (1, 16, 64, 32, True), (2, 15, 96, 96, True), (1, 100, 128, 128, False),
         (3, 1000, 160, 32, True), (16, 33, 1024, 64, False), (17, 4096, 256, 128, True), (5, 129, 4128, 32, False),
         (33, 48, 2048, 2048, True), (64, 130, 1056, 96, True), (64, 257, 512, 128, False), (1, 4097, 1024, 128, True),
         (8, 640, 8192, 64, False), (40, 17, 64, 64, True)]


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("m,n,k,group,zeros", EXACT)
def test_exact_on_small_integers(m, n, k, group, zeros, dt):
    """x of small integers and scales of powers of two: every sum is exact in fp32, so the
    result is the true one rounded once, to the bit."""
    from triton_kubernetes_amd.ops import gemv

    gen = _gen(m, n, k, group)
    codes, scales, zero = _weight(n, k, group, dt, zeros, gen, exact=True)
    x = torch.randint(-2, 3, (m, k), device="cuda", generator=gen).to(dt)
    # (16 + 15) |x| K and 31 |x| K / 2 steps of 1/2: under 2^24 for K <= 8192 and |x| <= 2 on average 1.2
    got = gemv.gemv_w4(x, gemv.pack_w4(codes), scales, zero)
    assert torch.equal(got, (x.double() @ _true(codes, scales, zero).T).to(dt))


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("m,n,k,group,zeros", EXACT)
def test_random_numbers(m, n, k, group, zeros, dt):
    """Per group at most group additions of partial sums up to 31 sum |x|, twice (the codes' and
    the zero's part), then one addition a group; each off by at most 2^-23; one rounding."""
    from triton_kubernetes_amd.ops import gemv

    gen = _gen(m, n, k, group, 1)
    codes, scales, zero = _weight(n, k, group, dt, zeros, gen)
    x = torch.randn((m, k), device="cuda", generator=gen).to(dt)
    got = gemv.gemv_w4(x, gemv.pack_w4(codes), scales, zero).double()
    w = _true(codes, scales, zero)
    true = x.double() @ w.T
    size = x.double().abs().view(m, -1, group).sum(2) @ scales.double().T  # sum over groups of s sum |x|
    bound = U[dt] * true.abs() + (2 * 31 * (group + 4) + 31 * (k // group + 8)) * 2.0 ** -23 * size
    off = (got - true).abs()
    assert bool((off <= bound * 1.01 + 1e-30).all()), float((off / bound).max())
    # the bound above is a worst case; fp32 sums of K random terms are good to sqrt(K) steps
    rel = float(off.norm() / true.norm())
    assert rel <= U[dt] / 2 + 2.0 ** -23 * 64 * k ** 0.5, rel


def test_layouts_batches_and_out():
    from triton_kubernetes_amd.ops import gemv

    gen = _gen(2)
    codes, scales, zero = _weight(200, 256, 64, torch.bfloat16, True, gen)
    packed = gemv.pack_w4(codes)
    x = torch.randn((12, 256), device="cuda", generator=gen).bfloat16()
    want = gemv.gemv_w4(x, packed, scales, zero)
    wide = torch.cat((x, x), 1)
    odd = torch.empty(12 * 256 + 1, device="cuda", dtype=x.dtype)[1:].view(12, 256).copy_(x)
    for other in (wide[:, :256], wide[:, 256:], odd, x.t().contiguous().t(), x.view(3, 4, 256), x.view(2, 3, 2, 256)):
        got = gemv.gemv_w4(other, packed, scales, zero)
        assert got.shape == (*other.shape[:-1], 200) and torch.equal(got.reshape(12, 200), want)
    # a single row and a batch add in another order: both round fp32 sums that are 2^-17 apart
    assert torch.allclose(gemv.gemv_w4(x[3], packed, scales, zero).float(), want[3].float(), rtol=2.0 ** -7, atol=1e-3)
    one = x[:1].expand(5, 256)  # stride 0
    assert torch.equal(gemv.gemv_w4(one, packed, scales, zero), want[:1].expand(5, 200))
    room = torch.full((14, 200), 77.0, device="cuda", dtype=x.dtype)
    assert gemv.gemv_w4(x, packed, scales, zero, out=room[1:13]).data_ptr() == room[1].data_ptr()
    assert torch.equal(room[1:13], want) and bool((room[[0, 13]] == 77).all())
    assert gemv.gemv_w4(x[:0], packed, scales, zero).shape == (0, 200)
    assert gemv.gemv_w4(x, packed[:0], scales[:0], zero[:0]).shape == (12, 0)


def test_a_rows_result_does_not_depend_on_the_others():
    """Serving: a token's result is its own, whatever the batch holds (NaN in another row)."""
    from triton_kubernetes_amd.ops import gemv

    gen = _gen(3)
    codes, scales, _ = _weight(300, 512, 128, torch.float16, False, gen)
    packed = gemv.pack_w4(codes)
    x = torch.randn((16, 512), device="cuda", generator=gen).half()
    want = gemv.gemv_w4(x, packed, scales)
    x[5] = float("nan")
    got = gemv.gemv_w4(x, packed, scales)
    keep = torch.arange(16, device="cuda") != 5
    assert torch.equal(got[keep], want[keep]) and bool(got[5].isnan().all())


def test_quantized_weight_round_trip_on_the_gpu():
    from triton_kubernetes_amd.ops import gemv

    gen = _gen(4)
    w = (torch.randn((500, 384), device="cuda", generator=gen) * 0.05).bfloat16()
    x = torch.randn((2, 384), device="cuda", generator=gen).bfloat16()
    for symmetric in (True, False):
        q = gemv.quantize_w4(w, 128, symmetric)
        true = x.double() @ gemv.dequantize_w4(*q).double().T
        got = gemv.gemv_w4(x, *q).double()
        assert float((got - true).norm() / true.norm()) <= 2.0 ** -8


def test_streams_and_graphs():
    from triton_kubernetes_amd.ops import gemv

    gen = _gen(5)
    codes, scales, zero = _weight(1000, 1024, 128, torch.bfloat16, True, gen)
    packed = gemv.pack_w4(codes)
    xs = [torch.randn((3, 1024), device="cuda", generator=gen).bfloat16() for _ in range(3)]
    want = [gemv.gemv_w4(x, packed, scales, zero) for x in xs]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        x = xs[0] * 2
        got = gemv.gemv_w4(x.mul_(0.5), packed, scales, zero)
    s.synchronize()
    assert torch.equal(got, want[0])
    x = xs[0].clone()
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for g in graphs:  # two graphs of the same call
        with torch.cuda.graph(g):
            outs.append(gemv.gemv_w4(x, packed, scales, zero))
    for turn in range(6):
        x.copy_(xs[turn % 3])
        graphs[turn % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[turn % 2], want[turn % 3])


def test_long_offsets():
    """Codes past 2^32 bytes."""
    from triton_kubernetes_amd.ops import gemv

    n, k = 140_000, 65536
    packed = torch.full((n, k // 2), 0x88, device="cuda", dtype=torch.uint8)
    packed[n - 3, k // 2 - 1] = 0x98  # the last code is 9
    scales = torch.ones((n, 1), device="cuda", dtype=torch.bfloat16)
    x = torch.zeros((1, k), device="cuda", dtype=torch.bfloat16)
    x[0, k - 1] = 5.0
    got = gemv.gemv_w4(x, packed, scales)
    want = torch.zeros((1, n), device="cuda", dtype=torch.bfloat16)
    want[0, n - 3] = 5.0
    assert torch.equal(got, want)


def test_refusals_on_the_gpu():
    from triton_kubernetes_amd.ops import gemv

    gen = _gen(6)
    codes, scales, zero = _weight(64, 128, 64, torch.bfloat16, True, gen)
    packed = gemv.pack_w4(codes)
    x = torch.zeros((2, 128), device="cuda", dtype=torch.bfloat16)
    ok = (x, packed, scales, zero)
    gemv.gemv_w4(*ok)
    for bad in ((x.new_zeros((65, 128)), packed, scales, zero), (x, packed.cpu(), scales, zero),
                (x, packed, scales.cpu(), zero), (x, packed, scales, zero.cpu()),
                (x, packed.t().contiguous().t(), scales, zero), (x.clone().requires_grad_(), packed, scales, zero),
                (x, torch.empty(64 * 64 + 1, device="cuda", dtype=torch.uint8)[1:].view(64, 64), scales, zero)):
        with pytest.raises(gemv.GemvError):
            gemv.gemv_w4(*bad)
    for out in (x.new_zeros((2, 65)), x.new_zeros((2, 64)).half(), x.new_zeros((2, 128))[:, :64]):
        with pytest.raises(gemv.GemvError):
            gemv.gemv_w4(*ok, out=out)
    with torch.no_grad():
        gemv.gemv_w4(x.clone().requires_grad_(), packed, scales, zero)


def test_out_may_not_share_memory_with_what_is_read():
    from triton_kubernetes_amd.ops import gemv

    codes, scales, zero = _weight(128, 128, 64, torch.bfloat16, True, _gen(7))
    packed = gemv.pack_w4(codes)
    room = torch.zeros((5, 128), device="cuda", dtype=torch.bfloat16)
    for x, out in ((room[:2], room[:2]), (room[:2], room[1:3]), (room[1:4:2], room[2:4])):
        with pytest.raises(gemv.GemvError, match="share"):
            gemv.gemv_w4(x, packed, scales, zero, out=out)
    with pytest.raises(gemv.GemvError, match="share"):
        gemv.gemv_w4(room[:2], packed, scales, zero, out=scales.view(-1)[:256].view(2, 128))
    with pytest.raises(gemv.GemvError, match="no gradient"):
        gemv.gemv_w4(room[:2], packed, scales, zero, out=torch.zeros_like(room[:2]).requires_grad_())
    gemv.gemv_w4(room[:2], packed, scales, zero, out=room[2:4])


@pytest.mark.parametrize("m", [1, 3, 16, 17, 64])
@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
def test_both_forms_of_few_rows_and_calls_at_once(m, dt, monkeypatch):
    """Each row by itself and all together, split and whole, on small integers: the same bits; on
    three streams at once."""
    from triton_kubernetes_amd.ops import gemv

    n, k, group = 530, 3200, 32
    gen = _gen(8, m)
    codes, scales, zero = _weight(n, k, group, dt, True, gen, exact=True)
    packed = gemv.pack_w4(codes)
    x = torch.randint(-2, 3, (m, k), device="cuda", generator=gen).to(dt)
    want = (x.double() @ _true(codes, scales, zero).T).to(dt)
    torch.cuda.synchronize()
    got = []
    for parts in (0, 1, 5):
        monkeypatch.setattr(gemv, "splits", lambda *a, parts=parts: parts)
        with torch.cuda.stream(torch.cuda.Stream()):
            got.append(gemv.gemv_w4(x, packed, scales, zero))
    torch.cuda.synchronize()
    for one in got:
        assert torch.equal(one, want)


def test_an_infinite_x_shows_in_its_row_alone(monkeypatch):
    from triton_kubernetes_amd.ops import gemv

    codes, scales, zero = _weight(100, 256, 64, torch.bfloat16, True, _gen(9))
    packed = gemv.pack_w4(codes)
    x = torch.ones((20, 256), device="cuda", dtype=torch.bfloat16)
    bad = x.clone()
    bad[7, 100] = float("inf")
    keep = torch.arange(20, device="cuda") != 7
    for parts in (0, 1):
        monkeypatch.setattr(gemv, "splits", lambda *a, parts=parts: parts)
        want, got = (gemv.gemv_w4(a, packed, scales, zero) for a in (x, bad))
        assert torch.equal(got[keep], want[keep]) and bool(got[7].isnan().all())


@pytest.mark.parametrize("m,n,k,group", [(1, 5, 1 << 20, 32), (3, 5, 1 << 20, 1 << 20), (33, 3, 1 << 19, 64),
                                         (1, 1 << 24, 32, 32), (2, 1 << 22, 64, 64), (20, 1 << 22, 32, 32)])
def test_largest_sizes(m, n, k, group):
    """x of one column that counts, per row another: the products are exact."""
    from triton_kubernetes_amd.ops import gemv

    gen = _gen(10, m, k)
    codes, scales, zero = _weight(n, k, group, torch.bfloat16, True, gen, exact=True)
    packed = gemv.pack_w4(codes)
    at = torch.randint(0, k, (m,), device="cuda", generator=gen)
    at[0] = k - 1
    x = torch.zeros((m, k), device="cuda", dtype=torch.bfloat16)
    x[torch.arange(m, device="cuda"), at] = 3.0
    want = (codes[:, at].float() - zero[:, at // group].float()) * scales[:, at // group].float() * 3
    assert torch.equal(gemv.gemv_w4(x, packed, scales, zero), want.t().bfloat16())
