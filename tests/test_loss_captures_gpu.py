"""Backward passes of the linear cross entropy that run in another capture than its loss, or in none."""

import pytest
import torch

from test_linear_cross_entropy_gpu import inputs, run


@pytest.mark.gpu
def test_a_backward_pass_in_a_graph_of_its_own_can_be_replayed_again():
    """The gradients that came with the loss are multiplied by the backward pass's factor: by that of each replay, not by all so far."""
    from flashfusedmoe_b200 import linear_cross_entropy
    h, w, t = inputs(300, 128, 1000)
    _, dh, dw = run(h, w, t)
    h, w = h.requires_grad_(), w.requires_grad_()
    factor = torch.tensor(2.0, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    forward, backward = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(forward, stream=side):
        loss = linear_cross_entropy(h, w, t)
    with torch.cuda.graph(backward, pool=forward.pool(), stream=side):
        grads = torch.autograd.grad(loss, (h, w), factor, retain_graph=True)
    forward.replay()
    for f in (2.0, 4.0, 0.5):
        factor.fill_(f)
        backward.replay()
        torch.cuda.synchronize()
        assert torch.equal(grads[0], dh * f) and torch.equal(grads[1], dw * f)
    # and by a backward pass outside of any graph, which again may follow a replay
    for f in (2.0, 4.0):
        forward.replay()
        again = torch.autograd.grad(loss, (h, w), torch.tensor(f, device="cuda"), retain_graph=True)
        torch.cuda.synchronize()
        assert torch.equal(again[0], dh * f) and torch.equal(again[1], dw * f)


@pytest.mark.gpu
def test_a_captured_backward_pass_of_a_loss_that_was_not():
    from flashfusedmoe_b200 import linear_cross_entropy
    h, w, t = inputs(300, 128, 1000)
    _, dh, dw = run(h, w, t)
    h, w = h.requires_grad_(), w.requires_grad_()
    factor = torch.tensor(2.0, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        loss = linear_cross_entropy(h, w, t)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        grads = torch.autograd.grad(loss, (h, w), factor, retain_graph=True)
    for f in (2.0, 4.0, 0.5):
        factor.fill_(f)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(grads[0], dh * f) and torch.equal(grads[1], dw * f)
