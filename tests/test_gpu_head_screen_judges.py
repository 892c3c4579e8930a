"""The loss screen on a GPU that gives the same wrong answer every time: the comparison with 64
bits has to find it, the one between passes cannot."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_a_wrong_answer_that_repeats_is_found(dtype, monkeypatch):
    from triton_kubernetes_amd.ops import head_screen, loss

    right = loss.linear_cross_entropy

    def part(x, w, target, **settings):  # without the second half of the vocabulary, for targets in the first
        return right(x, w[: w.shape[0] // 2], target % (w.shape[0] // 2), **settings)

    good = head_screen.loss_screen(0, 1024, 8192, 4096, reps=2, dtype=dtype)
    assert good.ok
    monkeypatch.setattr(loss, "linear_cross_entropy", part)
    bad = head_screen.loss_screen(0, 1024, 8192, 4096, reps=2, dtype=dtype)
    assert bad.differing == 0 and bad.bad_losses and bad.bad_dx and bad.bad_dw and not bad.ok
    monkeypatch.setattr(loss, "linear_cross_entropy", lambda x, w, t, **settings: right(x * 1.0625, w, t, **settings))
    bad = head_screen.loss_screen(0, 1024, 8192, 4096, reps=2, dtype=dtype)
    assert bad.differing == 0 and bad.bad_losses and bad.bad_dx and bad.bad_dw and not bad.ok
