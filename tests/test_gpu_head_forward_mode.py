"""The head's losses under forward-mode differentiation, which they do not have: no tangent is dropped."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["x", "w", "logits"])
@pytest.mark.parametrize("grads", [False, True])
def test_a_tangent_is_refused(which, grads):
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy, linear_distill

    gen = torch.Generator(device="cuda").manual_seed(1)
    tensors = dict(x=torch.randn((5, 64), device="cuda", generator=gen).bfloat16(),
                   w=torch.randn((90, 64), device="cuda", generator=gen).bfloat16(),
                   logits=torch.randn((5, 3), device="cuda", generator=gen))
    ids = torch.randint(0, 90, (5, 3), device="cuda", generator=gen)
    with forward_ad.dual_level():
        tensors[which] = forward_ad.make_dual(tensors[which], torch.ones_like(tensors[which]))
        with torch.set_grad_enabled(grads):
            with pytest.raises(RuntimeError, match="no gradient|forward mode|jvp|forward AD"):
                linear_distill(tensors["x"], tensors["w"], ids, tensors["logits"])
            if which != "logits":
                with pytest.raises(RuntimeError, match="no gradient|forward mode|jvp|forward AD"):
                    linear_cross_entropy(tensors["x"], tensors["w"], ids[:, 0])


def test_what_a_teacher_computes_without_gradients_is_taken():
    from triton_kubernetes_amd.ops.loss import linear_distill

    gen = torch.Generator(device="cuda").manual_seed(2)
    x, w = torch.randn((5, 64), device="cuda", generator=gen).bfloat16(), torch.randn((90, 64), device="cuda", generator=gen).bfloat16()
    ids = torch.randint(0, 90, (5, 3), device="cuda", generator=gen)
    logits = torch.randn((5, 3), device="cuda", generator=gen)
    want = linear_distill(x, w, ids, logits)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(logits, torch.ones_like(logits))
        assert torch.equal(linear_distill(x, w, ids, dual.detach()), want)
