"""What tests/head_norms.py finds, at every size that the GPU tests use it for: results rounded as
the kernels round them are within its bounds; zeros, a missing part of a sum and a shifted result
are not."""

import pytest
import torch

import head_norms


def _round(dl, x, w):
    dt = x.dtype
    s = 1.0 if dt == torch.bfloat16 else 32768.0 / float(dl.abs().max().clamp_min(1e-30))
    r = (dl * s).to(dt).double() / s
    return (r @ w.double()).to(dt), (r.T @ x.double()).to(dt)


def _inputs(n, d, v, dt):
    x, w, target, up, marks = head_norms.largest(n, d, v, dt, "cpu")
    ids = target[:, None]
    true = head_norms.exact(x, w, ids, torch.ones((n, 1), dtype=torch.float64), 1.0, up)
    return x, w, ids, marks, true, (true[0].float(), *_round(true[3]["dl"], x, w))


def _kinds(dt, true, got):
    return {name.split()[0] for name in head_norms.wrong(dt, true, got)}


def _without(mark, x, w, ids, true):
    """The results of a pass that leaves out a marked entry, token or step of 64 columns."""
    (loss, _, _), m, long = true[:3], true[3], max(*x.shape, len(w))
    missing, loss = m["dl"].clone(), loss.float()
    if long == len(w):
        missing[:, mark] = 0
    elif long == len(x):
        missing[mark] = 0
    else:
        cut, c = x.double().clone(), int(mark) // 64 * 64
        cut[:, c:c + 64] = 0
        z = cut @ w.double().T
        loss = (torch.logsumexp(z, 1) - z.gather(1, ids)[:, 0]).float()
    got = [loss, *_round(missing, x, w)]
    if long == x.shape[1]:
        for result in got[1:]:
            result[:, c:c + 8] = 0
    return got


@pytest.mark.parametrize("n,d,v,dt", head_norms.LARGEST)
def test_at_the_largest_sizes(n, d, v, dt):
    x, w, ids, marks, true, right = _inputs(n, d, v, dt)
    assert not _kinds(dt, true, right)
    m = true[3]
    missing = _without(marks[-1], x, w, ids, true)
    if v < 1 << 24:
        assert _kinds(dt, true, (right[0], *_round(m["dl"] - m["g"] * m["q"], x, w))) == {"dx", "dw"}  # no softmax
    assert _kinds(dt, true, missing) >= {"dx", "dw"}


SMALLER = [(3, 8192, 300, torch.bfloat16), (1 << 15, 8, 16, torch.bfloat16), (2, 8, 1 << 18, torch.float16),
           (17, 9, 1 << 16, torch.bfloat16), (300, 256, 2000, torch.bfloat16), (700, 136, 901, torch.float16)]


@pytest.mark.parametrize("n,d,v,dt", SMALLER)
def test_wrong_results_are_found(n, d, v, dt):
    x, w, ids, marks, true, (loss, dx, dw) = _inputs(n, d, v, dt)
    assert not _kinds(dt, true, (loss, dx, dw))
    m = true[3]
    for dl in (0 * m["dl"], m["dl"] - m["g"] * m["q"], m["g"] * m["q"], 2 * m["dl"], 1.05 * m["dl"]):
        bad = _round(dl, x, w)
        assert _kinds(dt, true, (loss, bad[0], dw)) == {"dx"} and _kinds(dt, true, (loss, dx, bad[1])) == {"dw"}
    for part in ((loss + 0.02, dx, dw), (loss * float("nan"), dx, dw)):
        assert _kinds(dt, true, part) == {"loss"}
    assert _kinds(dt, true, (loss, dx.roll(1, 0), dw)) == {"dx"} and _kinds(dt, true, (loss, dx, dw.roll(1, 0))) == {"dw"}
    for mark in marks[[0, len(marks) // 2, -1]]:
        assert _kinds(dt, true, _without(mark, x, w, ids, true)) >= {"dx", "dw"}
