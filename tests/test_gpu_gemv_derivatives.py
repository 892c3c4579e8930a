"""The 4-bit products have no derivative; what autograd must be told of that."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _weight(n=96, k=128):
    from triton_kubernetes_amd.ops.gemv import pack_w4

    gen = torch.Generator(device="cuda").manual_seed(4)
    codes = torch.randint(0, 16, (n, k), device="cuda", generator=gen, dtype=torch.uint8)
    return pack_w4(codes), torch.rand((n, k // 64), device="cuda", generator=gen).bfloat16() + 0.5


@pytest.mark.parametrize("m", [1, 3])
def test_out_is_a_change_that_autograd_sees(m):
    """A buffer that another operation has saved for its backward pass and that is then written."""
    from triton_kubernetes_amd.ops.gemv import gemv_w4

    packed, scales = _weight()
    x = torch.ones((m, 128), device="cuda", dtype=torch.bfloat16)
    room = torch.zeros((5, 96), device="cuda", dtype=torch.bfloat16)
    leaf = torch.ones((m, 96), device="cuda", dtype=torch.bfloat16, requires_grad=True)
    loss = (room[:m] * leaf).sum()  # keeps room[:m]
    version = room._version
    assert gemv_w4(x, packed, scales, out=room[:m]).data_ptr() == room.data_ptr()
    assert room._version == version + 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_out_of_an_inference_is_written():
    from triton_kubernetes_amd.ops.gemv import gemv_w4

    packed, scales = _weight()
    x = torch.ones((2, 128), device="cuda", dtype=torch.bfloat16)
    want = gemv_w4(x, packed, scales)
    with torch.inference_mode():
        out = torch.empty_like(want)
        gemv_w4(x, packed, scales, out=out)
    assert torch.equal(out, want)
    with torch.inference_mode():
        gemv_w4(x, packed, scales, out=want.zero_())
    assert torch.equal(out, want)
