"""What a call of the output head's operators plans before the GPU has anything to do: what is
kept between the passes, how the vocabulary is cut, which settings are refused."""

import inspect

import pytest
import torch

from triton_kubernetes_amd.ops import loss

CUDA = torch.device("cuda", 0)


def plan(n, d, v, *, k=0, keep="default", temperature=1.0, dt=torch.bfloat16):
    """The plan of a training step of these sizes; ``k`` entries of a teacher's lists."""
    call = loss.linear_distill if k else loss.linear_cross_entropy
    if keep == "default":
        keep = inspect.signature(call).parameters["keep_logits"].default

    def meta(*shape, dtype=dt):
        return torch.Size(shape), dtype, CUDA

    rules = (loss.small_products, loss.keeps, loss.pieces, loss.fill, loss.weight_parts, loss.DL_BYTES, loss.KEEP_BYTES)
    return loss._plan(call.__name__, meta(n, d), meta(v, d), meta(*([n, k] if k else [n]), dtype=torch.int64),
                      meta(n, k, dtype=torch.float32) if k else None, "mean", temperature, -100, keep, True, rules)


@pytest.mark.parametrize("k", [0, 64])
@pytest.mark.parametrize("n,d,v", [(48, 512, 1000), (512, 256, 32000), (4096, 4096, 32768), (8192, 4096, 131072)])
def test_no_logits_are_kept_unless_the_caller_says_so(n, d, v, k):
    usual = plan(n, d, v, k=k)
    assert not usual.keep and usual.codes == 0
    # x's packed rows, and a few numbers a token and listed entry
    assert usual.kept <= 2 * n * (d + 63) + n * (40 + 8 * k) + 512
    assert plan(n, d, v, k=k, keep=False).kept == usual.kept
    kept = plan(n, d, v, k=k, keep=True)
    assert kept.keep and kept.kept >= usual.kept + 2 * n * v
    where_faster = plan(n, d, v, k=k, keep=None)
    assert where_faster.keep == loss.keeps(n, d, v)


def test_the_backward_workspace_has_a_place_for_the_number_of_splits():
    """What k_dx found and k_dx_out has to go by: 4 bytes between the factors and the residuals."""
    from test_head_ops import _args

    sizes = dict(n=3, d=64, piece=256, fill=1, small=0, want=1, distill=1)
    want = 2 * 3 * 256 + 4 * 3 * 64 + 4 * (3 + 1) + 4 + 16 * 3  # dl, sums, factors, splits, residuals
    want = -(-want // 16) * 16
    assert loss._lib().tkl_room_bytes(_args(**sizes)) == want
    assert loss.room_bytes(3, 64, 256, 1, 0, 1, 1) == want


@pytest.mark.parametrize("n", [1, 300, 48_211, 524_288, 700_001, 1_040_000, 1 << 20])
@pytest.mark.parametrize("v", [1, 257, 51_400, 262_144, 1 << 24])
def test_a_piece_of_the_vocabulary_stays_within_its_memory(n, v):
    if -(-v // loss.TILE) * -(-n // loss.TILE) >= 1 << 23:
        return  # refused
    piece = loss.pieces(n, v)
    assert piece % loss.TILE == 0 and 2 * n * piece <= 1.5 * loss.DL_BYTES
    assert (-(-v // piece) - 1) * piece < v  # none is empty


@pytest.mark.parametrize("temperature", [0.0, -1.0, float("nan"), float("inf"), 1e300, 1e20, 2.0 ** 33, 2.0 ** -33, 1e-20, 5e-324])
def test_temperatures_whose_square_or_quotient_fp32_does_not_hold_are_refused(temperature):
    from test_head_ops import _args

    with pytest.raises(loss.LossError, match="temperature"):
        plan(4, 64, 300, k=3, temperature=temperature)
    if temperature < 1e38 or temperature != temperature:
        for call in (loss._lib().tkl_forward, loss._lib().tkl_backward):
            assert call(_args(temperature=temperature)) == -1
            assert b"temperature" in loss._lib().tkl_last_error()


@pytest.mark.parametrize("temperature", [2.0 ** -32, 0.7, 1, 2.0 ** 32])
def test_temperatures_that_are_taken(temperature):
    assert plan(4, 64, 300, k=3, temperature=float(temperature)).temperature == temperature


def test_a_precise_gradient_has_two_parts_in_the_memory_of_one():
    from test_head_ops import _args

    def precise(n, d, v, keep=False):
        def meta(*shape, dtype=torch.bfloat16):
            return torch.Size(shape), dtype, CUDA

        return loss._plan("linear_cross_entropy", meta(n, d), meta(v, d), meta(n, dtype=torch.int64), None, "mean", 1.0, -100,
                          keep, True, (), True)

    for n, d, v in ((1, 8, 1), (48, 512, 1000), (4096, 4096, 32768), (8192, 4096, 131072), (1 << 20, 8, 40)):
        p, usual = precise(n, d, v), plan(n, d, v)
        assert p.small == usual.small | 8 and not p.keep and p.kept == usual.kept
        assert 4 * n * p.piece <= max(1.5 * loss.DL_BYTES, 4 * n * loss.TILE) and p.piece <= usual.piece
        args = _args(n=n, d=d, v=v, want=3, piece=p.piece, fill=p.groups, small=p.small, parts=p.parts[3])
        assert loss._lib().tkl_room_bytes(args) == p.room[3]
    assert not precise(48, 512, 1000, None).keep
    with pytest.raises(loss.LossError, match="kept logits"):
        precise(48, 512, 1000, True)
    assert loss._lib().tkl_backward(_args(small=8, codes=4096)) == -1
    assert b"kept logits" in loss._lib().tkl_last_error()


@pytest.mark.parametrize("n,piece", [(1, 1 << 24), (2, 10_000_128), (30, 8_000_000 // 256 * 256), (64, 8_388_352)])
def test_rows_too_long_for_large_tiles_are_refused_by_the_c_entry(n, piece):
    """193 - n rows behind the last one, of 2 ``piece`` bytes each, against 2^31: past that a copy of rows
    that are not there would read them."""
    from test_head_ops import _args

    assert (193 - n) * 2 * piece >= 1 << 31 and n * piece < 1 << 29
    for small in (0, 5, 8):
        assert loss._lib().tkl_backward(_args(n=n, v=piece, piece=piece, want=1, small=small)) == -1
        assert b"too long" in loss._lib().tkl_last_error()


@pytest.mark.parametrize("v", [4_000_000, 5_000_000, 6_190_000, 6_200_000, 8_000_000, 1 << 24])
def test_no_rule_asks_for_rows_that_long(v):
    for n in [*range(1, 130), 192, 193, 256, 300]:
        for d in (8, 64, 4096):
            if not loss.small_products(n, d, v) & 2:
                for piece in (loss.pieces(n, v), min(loss.pieces(n, v), loss.pieces(2 * n, v))):
                    assert (193 - min(n, 193)) * 2 * piece < 1 << 31
