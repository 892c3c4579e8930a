"""Weights at the ends of their type's range, quantized to 4 bits."""

import pytest
import torch

from triton_kubernetes_amd.ops import gemv


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("symmetric", [True, False])
def test_the_largest_weights_keep_their_values(dt, symmetric):
    """A group from the type's lowest value to its highest: 15 steps of 2 / 15 of it each.  (Of
    bf16's half range: a span past fp32 is refused.)"""
    top = torch.finfo(dt).max / (2 if dt == torch.bfloat16 and not symmetric else 1)
    w = torch.linspace(-1, 1, 64).double().mul(top).to(dt).view(1, 64)
    w = torch.cat((w, w.abs(), -w.abs(), w.new_full((1, 64), top)))
    codes, scales, zeros = gemv.quantize_w4(w, 64, symmetric)
    assert bool(torch.isfinite(scales).all())
    back = gemv.dequantize_w4(codes, scales, zeros).double()
    step = scales.double()
    # half a step, and a half more for a zero rounded to a whole code; the scale's own rounding, 15 steps
    most = (0.5 + 16 * torch.finfo(dt).eps + (0.0 if symmetric else 0.5)) * step
    assert bool(((back - w.double()).abs() <= most).all())


def test_a_span_past_fp32_is_refused():
    w = torch.full((2, 64), 2.0 ** 127).bfloat16()
    w[1, 5] = -2.0 ** 127
    with pytest.raises(gemv.GemvError, match="span"):
        gemv.quantize_w4(w, 32, symmetric=False)
    gemv.quantize_w4(w[:1], 32, symmetric=False)


def test_ordinary_weights_are_quantized_as_before():
    """The scale is the span over 15, rounded once; subnormal and ordinary spans."""
    gen = torch.Generator().manual_seed(1)
    for dt in (torch.bfloat16, torch.float16):
        for size in (1.0, 2.0 ** -13, 1e3):
            w = (torch.randn((40, 128), generator=gen) * size).to(dt)
            v = w.float().view(40, 2, 64)
            lo, hi = v.amin(2).clamp_max(0), v.amax(2).clamp_min(0)
            scales = ((hi - lo) / 15).to(dt)
            step = torch.where(scales.float() > 0, scales.float(), float("inf"))
            zeros = (-lo / step).round().clamp(0, 15)
            codes = (v / step[:, :, None] + zeros[:, :, None]).round().clamp(0, 15).to(torch.uint8)
            got = gemv.quantize_w4(w, 64, symmetric=False)
            assert torch.equal(got[1], scales) and torch.equal(got[2], zeros.to(torch.uint8))
            assert torch.equal(got[0], gemv.pack_w4(codes.view(40, 128)))
