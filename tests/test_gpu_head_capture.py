"""Backward passes of the head's losses in a captured graph, by ``backward`` and by ``grad``, and
what holds a leaf's gradient node meanwhile."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _inputs(seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    w = (torch.randn((900, 128), device="cuda", generator=gen) / 8).bfloat16()
    return (torch.randn((90, 128), device="cuda", generator=gen).bfloat16(), w,
            torch.randint(0, 900, (90,), device="cuda", generator=gen))


@pytest.mark.parametrize("keep", [False, True], ids=["again", "kept"])
def test_backward_into_the_leaves_is_captured(keep):
    """``loss.backward()`` of leaves whose nodes are made in the capture: each replay writes the
    gradients of what the inputs then hold."""
    from triton_kubernetes_amd.ops.loss import linear_cross_entropy

    sets = [_inputs(s) for s in (1, 2, 3)]
    x, w, t = (a.clone() for a in sets[0])
    x.requires_grad_()
    w.requires_grad_()
    linear_cross_entropy(x, w, t, keep_logits=keep).backward()  # its graph is gone with this line
    x.grad = w.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = linear_cross_entropy(x, w, t, keep_logits=keep)
        loss.backward()
    for turn in range(6):
        data = sets[turn % 3]
        with torch.no_grad():
            for a, b in zip((x, w, t), data):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        a, b = (v.clone().requires_grad_() for v in data[:2])
        eager = linear_cross_entropy(a, b, data[2], keep_logits=keep)
        eager.backward()
        assert torch.equal(loss.detach(), eager.detach()) and torch.equal(x.grad, a.grad) and torch.equal(w.grad, b.grad), turn


def test_what_else_holds_a_node_is_named():
    """No loss is alive, but the weight's gradient node is, as a reducer holds it: the refusal says
    so, the way out that it names works, and so does the call once the node is free."""
    from triton_kubernetes_amd.ops.loss import LossError, linear_cross_entropy

    x, w, t = _inputs(4)
    x.requires_grad_()
    w.requires_grad_()
    edge = torch.autograd.graph.get_gradient_edge(w)
    want = torch.autograd.grad(linear_cross_entropy(x, w, t), (x, w))
    with pytest.raises(LossError, match="reducer"), torch.cuda.graph(torch.cuda.CUDAGraph()):
        linear_cross_entropy(x, w, t)

    def captured(*leaves):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            a, b = leaves or (x.detach().requires_grad_(), w.detach().requires_grad_())
            out = torch.autograd.grad(linear_cross_entropy(a, b, t), (a, b))
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))

    captured()
    del edge
    captured(x, w)
