"""The output head's operators without a GPU: what they refuse, the rules that size their
workspaces, the C entries' own checks, and the 4-bit weight format."""

import pytest
import torch

from triton_kubernetes_amd.ops import gemv, loss


def _x(*shape, dt=torch.bfloat16):
    return torch.zeros(shape, dtype=dt)


@pytest.mark.parametrize("x,w,message", [
    (_x(4, 8, dt=torch.float32), _x(9, 8, dt=torch.float32), "both bf16 or both fp16"),
    (_x(4, 8), _x(9, 8, dt=torch.float16), "both bf16 or both fp16"),
    (_x(4, 8), _x(9, 16), r"x \[..., D\] and w \[V, D\]"),
    (_x(4, 8), _x(8), r"x \[..., D\] and w \[V, D\]"),
    (_x(4, 8), _x(9, 8), "CUDA tensors on one device"),
])
def test_losses_refuse_inputs(x, w, message):
    ids = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(loss.LossError, match=message):
        loss.linear_cross_entropy(x, w, ids)
    with pytest.raises(loss.LossError, match=message):
        loss.linear_distill(x, w, ids[:, None], torch.zeros(4, 1))


@pytest.mark.parametrize("n", [1, 47, 48, 4096, 8192, 1 << 20])
@pytest.mark.parametrize("v", [1, 256, 257, 1000, 50021, 262144, 1 << 24])
def test_pieces_cover_the_vocabulary_within_the_workspace(n, v):
    piece = loss.pieces(n, v)
    assert piece % loss.TILE == 0 and piece >= loss.TILE
    assert piece == loss.TILE or (piece - loss.TILE) * n * 2 <= 1.5 * loss.DL_BYTES
    assert min(n, loss.TILE) * piece < 1 << 29  # what the C entry takes
    count = -(-v // piece)
    assert (count - 1) * piece < v  # no empty piece


FIELDS = ("n", "d", "v", "k", "ldx", "ldw", "ldg", "ignore", "piece", "fill", "dev", "f16", "distill", "reduction",
          "temperature", "want", "small", "parts", "x", "w", "ids", "teacher", "grad", "loss", "kept", "room", "codes", "wc", "dx", "dw",
          "stream")


def _args(**fields):
    base = dict(n=4, d=8, v=16, k=1, ldx=8, ldw=8, reduction=2, temperature=1.0, piece=256, fill=256, w=4096)
    return loss._ARGS.pack(*({**dict.fromkeys(FIELDS, 0), **base, **fields}[f] for f in FIELDS))


@pytest.mark.parametrize("n,d,k", [(1, 1, 1), (7, 72, 1), (333, 1288, 100), (8192, 4096, 64)])
def test_buffers_have_the_sizes_that_the_kernels_take(n, d, k):
    lib = loss._lib()
    for distill in (0, 1):
        assert lib.tkl_kept_bytes(_args(n=n, d=d, k=k, distill=distill)) == loss.kept_bytes(n, d, n * k * distill)
        for want, groups, small, piece, parts in ((3, 256, 0, 512, 1), (1, 512, 2, 4096, 0), (2, 256, 0, 256, 3),
                                                  (1, 1, 0, 32768, 1), (3, 4096, 7, 256, 64)):
            args = _args(n=n, d=d, v=200, k=k, want=want, piece=piece, fill=groups, small=small, distill=distill,
                         parts=parts)
            assert lib.tkl_room_bytes(args) == loss.room_bytes(n, d, piece, groups, small, want, distill,
                                                               parts * 200 if parts > 1 else 0)


@pytest.mark.parametrize("fields,message", [
    (dict(n=0), "tokens"), (dict(n=(1 << 20) + 1), "tokens"), (dict(d=0), "width"), (dict(d=65537), "width"),
    (dict(v=0), "vocabulary"), (dict(v=(1 << 24) + 1), "vocabulary"), (dict(k=0), "targets"), (dict(k=1025), "targets"),
    (dict(d=7), "aligned"), (dict(ldw=9), "aligned"), (dict(w=4098), "aligned"), (dict(ldw=0), "row stride"),
    (dict(ldw=1 << 22), "row stride"), (dict(reduction=3), "reduction"), (dict(temperature=0.0), "temperature"),
    (dict(temperature=float("nan")), "temperature"), (dict(n=1 << 20, v=1 << 19), "tokens x vocabulary"),
    (dict(n=1 << 20, d=1 << 14, ldw=1 << 14), "tokens x width"),
])
def test_the_c_entries_check_before_the_gpu(fields, message):
    lib = loss._lib()
    for call in (lib.tkl_forward, lib.tkl_backward):
        assert call(_args(**fields)) == -1
        assert message in lib.tkl_last_error().decode()


@pytest.mark.parametrize("fields", [dict(piece=0), dict(piece=255), dict(piece=1 << 25), dict(fill=0), dict(fill=4097),
                                    dict(n=300, piece=1 << 21), dict(parts=65), dict(parts=-1),
                                    dict(parts=2, v=300)])
def test_the_c_backward_checks_its_pieces(fields):
    assert loss._lib().tkl_backward(_args(**fields)) == -1


def test_gemv_refuses_inputs():
    codes, scales = torch.zeros((4, 32), dtype=torch.uint8), _x(4, 2)
    for x, c, s, z, message in (
            (_x(1, 64, dt=torch.float32), codes, scales, None, "both bf16 or both fp16"),
            (_x(1, 64, dt=torch.float16), codes, scales, None, "both bf16 or both fp16"),
            (_x(1, 64), codes.int(), scales, None, "codes uint8"),
            (_x(1, 64), codes[0], scales, None, "codes uint8"),
            (_x(1, 64), codes, scales[:3], None, "codes uint8"),
            (_x(1, 64), codes, _x(4, 3), None, "groups do not divide"),
            (_x(1, 64), codes, _x(4, 4), None, "groups do not divide"),
            (_x(1, 64), codes, _x(4, 0), None, "groups do not divide"),
            (_x(1, 64), codes, scales, torch.zeros((4, 2)), "zeros uint8"),
            (_x(1, 64), codes, scales, torch.zeros((4, 1), dtype=torch.uint8), "zeros uint8"),
            (_x(1, 32), codes, scales, None, "does not go with"),
            (_x(1, 64), codes, scales, None, "CUDA tensors on one device")):
        with pytest.raises(gemv.GemvError, match=message):
            gemv.gemv_w4(x, c, s, z)


@pytest.mark.parametrize("m,n,k,group,ldx,ldy,x,codes", [
    (0, 4, 64, 64, 64, 4, 4096, 4096), (65, 4, 64, 64, 64, 4, 4096, 4096), (1, 0, 64, 64, 64, 4, 4096, 4096),
    (1, 4, 64, 48, 64, 4, 4096, 4096), (1, 4, 64, 0, 64, 4, 4096, 4096), (1, 4, 96, 64, 96, 4, 4096, 4096),
    (1, 4, 64, 64, 32, 4, 4096, 4096), (1, 4, 64, 64, 68, 4, 4096, 4096), (1, 4, 64, 64, 64, 4, 4098, 4096),
    (1, 4, 64, 64, 64, 4, 4096, 4104), (1, 4, 64, 64, 64, 3, 4096, 4096)])
def test_the_gemv_c_entry_checks_before_the_gpu(m, n, k, group, ldx, ldy, x, codes):
    lib = gemv._lib()
    assert lib.tkv_gemv_w4(gemv._ARGS.pack(0, 0, m, n, k, group, 1, ldx, ldy, x, codes, 4096, 0, 4096, 0, 0)) == -1
    assert lib.tkv_last_error()


def test_the_gemv_c_entry_checks_its_splits():
    for splits in (-1, 2, 65):  # 2 without room for the sums
        assert gemv._lib().tkv_gemv_w4(gemv._ARGS.pack(0, 0, 1, 4, 64, 64, splits, 64, 4, 4096, 4096, 4096, 0, 4096, 0, 0)) == -1
        assert b"splits" in gemv._lib().tkv_last_error()


def test_pack_and_quantize_refuse():
    for bad in (torch.zeros((2, 3), dtype=torch.uint8), torch.zeros((2, 4)), torch.full((2, 4), 16, dtype=torch.uint8)):
        with pytest.raises(gemv.GemvError):
            gemv.pack_w4(bad)
    for w, group in ((torch.zeros((2, 64)), 64), (_x(2, 64), 48), (_x(2, 64), 128), (_x(2, 96), 64), (_x(2, 64), 0),
                     (torch.full((2, 64), float("inf"), dtype=torch.bfloat16), 64)):
        with pytest.raises(gemv.GemvError):
            gemv.quantize_w4(w, group)


def test_packing_order():
    codes = torch.arange(32, dtype=torch.uint8).remainder(16).view(1, 32)
    packed = gemv.pack_w4(codes)
    assert packed[0, 0] == 0x10 and packed[0, 7] == 0xfe
    scales, zeros = torch.ones((1, 1), dtype=torch.float16), torch.tensor([[3]], dtype=torch.uint8)
    assert torch.equal(gemv.dequantize_w4(packed, scales, zeros), codes.float() - 3)
    assert torch.equal(gemv.dequantize_w4(packed, scales), codes.float() - 8)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("symmetric", [True, False])
def test_quantized_values_are_the_nearest(dt, symmetric):
    """Half a step of the group's scale, plus what the rounding of the scale moves the ends by."""
    g = torch.Generator().manual_seed(3)
    w = (torch.randn((9, 192), generator=g) * torch.logspace(-2, 1, 9)[:, None]).to(dt)
    w[4] = 0
    w[5] = w[5].abs()
    codes, scales, zeros = gemv.quantize_w4(w, 64, symmetric)
    back = gemv.dequantize_w4(codes, scales, zeros)
    step = scales.float().repeat_interleave(64, 1)
    # the scale may round down by u: the farthest value is then 15 u steps past the last code;
    # a zero rounds to a whole code, which moves an end by half a step more
    most = 0.5 + 16 * torch.finfo(dt).eps + (0.0 if symmetric else 0.5)
    assert bool(((back - w.float()).abs() <= most * step + 1e-30).all())
    assert bool((back[4] == 0).all())


@pytest.mark.parametrize("argv", [["loss", "--tokens", "0"], ["loss", "--dtype", "fp8"], ["gemv", "--rows", "0"],
                                  ["gemv", "--group", "x"]])
def test_screen_commands_check_their_counts(argv, capsys):
    from triton_kubernetes_amd.ops import cli

    with pytest.raises(SystemExit) as exc:
        cli.main(argv)
    assert exc.value.code == 2


@pytest.mark.parametrize("argv", [["loss"], ["gemv"]])
def test_screen_commands_without_a_gpu(argv, capsys, monkeypatch):
    from triton_kubernetes_amd.ops import cli

    monkeypatch.setattr(torch.cuda, "is_available", lambda: False)
    assert cli.main(argv) == 2
    assert "tk-gpu: no GPU" in capsys.readouterr().err


@pytest.mark.parametrize("m", [1, 2, 16, 17, 64])
@pytest.mark.parametrize("n,k", [(1, 32), (100, 4096), (4096, 4128), (131072, 4096), (16, 1 << 20)])
def test_gemv_splits_leave_no_part_empty(m, n, k):
    parts = gemv.splits(m, n, k)
    if parts == 0:  # each row by itself
        return
    chunks = -(-k // 128)
    per = -(-(-(-chunks // parts)) // 2) * 2  # as the launch divides them
    assert 1 <= parts <= 64 and (parts - 1) * per < chunks <= parts * per
    assert m > 1


def test_tile_rules_at_their_corners():
    assert loss.small_products(1, 512, 1000) == 7 and loss.small_products(1024, 512, 1000) == 7
    assert loss.small_products(64, 4096, 131072) == 3 and loss.small_products(65, 4096, 131072) == 0
    assert loss.small_products(8192, 4096, 131072) == 0


def test_a_group_whose_scale_is_as_small_as_the_type_has():
    w = torch.zeros((2, 64), dtype=torch.bfloat16)
    w[0, 3] = 2.0 ** -130  # the scale is subnormal in bf16, and 1 / scale no fp32 number
    w[1] = 2.0 ** -130
    for symmetric in (True, False):
        codes, scales, zeros = gemv.quantize_w4(w, 32, symmetric)
        back = gemv.dequantize_w4(codes, scales, zeros)
        assert bool(torch.isfinite(back).all())
        assert float((back - w.float()).abs().max()) <= 2.0 ** -133  # 8 steps of 2^-133, 7 of them reached
