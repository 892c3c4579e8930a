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


def test_the_screen_runs_the_distillation_and_judges_it(monkeypatch):
    from triton_kubernetes_amd.ops import head_screen, loss

    for sizes in ((512, 3000, 512), (3, 40, 72), (1, 1, 8)):
        good = head_screen.loss_screen(0, *sizes, reps=2)
        assert good.ok and good.entries == min(64, sizes[1]) and good.distill_ms > 0, good
    alone = head_screen.loss_screen(0, 512, 3000, 512, reps=2, entries=0)
    assert alone.ok and alone.distill_ms == 0
    right = loss.linear_distill
    monkeypatch.setattr(loss, "linear_distill", lambda x, w, ids, logits, **settings: right(x, w, ids, logits * 1.125, **settings))
    bad = head_screen.loss_screen(0, 512, 3000, 512, reps=2)
    assert bad.differing == 0 and bad.bad_losses and bad.bad_dx and bad.bad_dw and not bad.ok


def test_the_command_takes_a_teachers_lists():
    import json
    import subprocess
    import sys

    for entries, code in (("5", 0), ("0", 0), ("1025", 2)):
        proc = subprocess.run([sys.executable, "-m", "triton_kubernetes_amd.ops.cli", "loss", "--tokens", "200", "--vocab", "2000",
                               "--hidden", "64", "--reps", "1", "--entries", entries], capture_output=True, text=True, timeout=110)
        assert proc.returncode == code, proc.stderr
        if not code:
            got = json.loads(proc.stdout)
            assert got["ok"] and got["entries"] == int(entries) and (got["distill_ms"] > 0) == (entries != "0")
