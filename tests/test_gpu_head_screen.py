"""The output head's operators together, as they are used: a head trained, distilled into,
quantized and answered with; and the screens that run them on a node."""

import json
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_head_from_training_to_answering():
    """A training step, a distillation step from its own top logits, then 4-bit answers: each
    stage against 64 bits, on the weights that the stage before left."""
    import head_reference as ref

    from triton_kubernetes_amd.ops.gemv import dequantize_w4, gemv_w4, quantize_w4
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy, linear_distill

    n, d, v = 96, 256, 1200
    gen = torch.Generator(device="cuda").manual_seed(21)
    w = (torch.randn((v, d), device="cuda", generator=gen) * d ** -0.5).bfloat16()
    x = torch.randn((n, d), device="cuda", generator=gen).bfloat16()
    target = torch.randint(0, v, (n,), device="cuda", generator=gen)
    target[::5] = -100
    teacher = (x.float() @ w.float().T).topk(32, dim=1)
    for step in range(3):
        leaf = w.clone().requires_grad_()
        up = torch.full((n,), 1.0 / n, device="cuda", dtype=torch.float64)
        hard = linear_cross_entropy(x, leaf, target, reduction="none")
        soft = linear_distill(x, leaf, teacher.indices, teacher.values, temperature=2.0, reduction="none")
        dh, = torch.autograd.grad(hard, leaf, up.float())
        ds, = torch.autograd.grad(soft, leaf, up.float())
        for grad, loss, (ids, p), t in ((dh, hard, ref.targets_of(target, -100, n, v), 1.0),
                                        (ds, soft, ref.teacher_of(teacher.indices, teacher.values, 2.0), 2.0)):
            want, _, wdw = ref.head(x, w, ids, p, t, up)
            ref.check("loss", loss.detach(), want)
            ref.check("dw", grad, wdw)
        w = (w.float() - 4.0 * (dh.float() + ds.float())).bfloat16()
    for rows in (1, 7):
        q = quantize_w4(w, 64, symmetric=False)
        got = gemv_w4(x[:rows], *q).double()
        true = x[:rows].double() @ dequantize_w4(*q).double().T
        assert float((got - true).norm() / true.norm()) <= 2.0 ** -8


def test_loss_screen_passes_and_sees_a_changed_value():
    from triton_kubernetes_amd.ops import head_screen

    for dtype in ("bf16", "fp16"):
        r = head_screen.loss_screen(0, 1024, 8000, 1024, reps=2, dtype=dtype)
        print(json.dumps(r.to_json()))
        assert r.ok and r.max_norm_error <= 1, r
    bad = head_screen.loss_screen(0, 512, 3000, 512, reps=2, inject=12345)
    assert not bad.ok and bad.differing == 1


def test_gemv_screen_passes_and_sees_a_changed_value():
    from triton_kubernetes_amd.ops import head_screen

    for rows, dtype in ((1, "bf16"), (20, "fp16")):
        r = head_screen.gemv_screen(0, rows, 5000, 4096, 64, reps=3, dtype=dtype)
        print(json.dumps(r.to_json()))
        assert r.ok and r.max_norm_error <= 1, r
    bad = head_screen.gemv_screen(0, 2, 4096, 4096, 128, reps=2, inject=777)
    assert not bad.ok and bad.differing == 1


@pytest.mark.parametrize("argv", [["loss", "--tokens", "300", "--vocab", "1111", "--hidden", "77", "--dtype", "fp16"],
                                  ["gemv", "--rows", "3", "--out", "500", "--inp", "4096", "--group", "32"]])
def test_commands(argv):
    proc = subprocess.run([sys.executable, "-m", "triton_kubernetes_amd.ops.cli", *argv], capture_output=True, text=True,
                          timeout=110)
    assert proc.returncode == 0, proc.stderr
    assert json.loads(proc.stdout)["ok"] is True


@pytest.mark.parametrize("argv", [["gemv", "--rows", "65"], ["gemv", "--inp", "100"], ["loss", "--hidden", "65537"]])
def test_commands_refuse_with_one_line(argv):
    proc = subprocess.run([sys.executable, "-m", "triton_kubernetes_amd.ops.cli", *argv, "--reps", "1"],
                          capture_output=True, text=True, timeout=110)
    assert proc.returncode == 2 and proc.stderr.strip().splitlines()[-1].startswith("tk-gpu: "), proc.stderr
