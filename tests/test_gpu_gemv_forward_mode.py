"""The 4-bit products under torch's forward-mode differentiation: a tensor with a tangent is
refused, as one that wants a gradient is."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

pytestmark = pytest.mark.gpu


def test_a_tangent_is_refused():
    from triton_kubernetes_amd.ops.gemv import GemvError, gemv_w4, pack_w4

    gen = torch.Generator(device="cuda").manual_seed(4)
    packed = pack_w4(torch.randint(0, 16, (96, 128), device="cuda", generator=gen, dtype=torch.uint8))
    scales = torch.rand((96, 2), device="cuda", generator=gen).bfloat16() + 0.5
    x = torch.ones((2, 128), device="cuda", dtype=torch.bfloat16)
    out = torch.empty((2, 96), device="cuda", dtype=torch.bfloat16)
    want = gemv_w4(x, packed, scales)

    def dual(t):
        return forward_ad.make_dual(t, torch.ones_like(t))

    with forward_ad.dual_level():
        for bad in (dict(x=dual(x)), dict(scales=dual(scales)), dict(out=dual(out))):
            call = dict(dict(x=x, codes=packed, scales=scales), **bad)
            with pytest.raises(GemvError, match="no gradient"):
                gemv_w4(**call)
            with torch.no_grad(), pytest.raises(GemvError, match="no gradient"):  # which says nothing of tangents
                gemv_w4(**call)
        # tensors without a tangent pass, and what of a dual tensor is none
        assert torch.equal(gemv_w4(x, packed, scales, out=out), want)
        assert torch.equal(gemv_w4(forward_ad.unpack_dual(dual(x)).primal, packed, scales), want)
