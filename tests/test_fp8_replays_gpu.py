"""GPU: the e4m3 copies of expert weights beside captured optimizer steps."""

import gc
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

import flashfusedmoe_b200 as ffm  # noqa: E402

DEV = "cuda"
layer_module = sys.modules["flashfusedmoe_b200.fused_moe"]   # the package has the function under this name


def test_fp8_copies_of_weights_that_replays_update():
    """A replayed step changes weights without raising their version: the e4m3 copy of an earlier call is not theirs."""
    torch.manual_seed(2)
    layer = ffm.MoELayer(256, 512, 4, top_k=2).to(DEV).bfloat16()
    opt = ffm.AdamW([layer.w_up, layer.w_down], lr=0.05)
    x = torch.randn(2048, 256, device=DEV).bfloat16()
    for p in (layer.w_up, layer.w_down):
        p.grad = torch.randn_like(p)
    opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    old = ffm.set_expert_gemm_precision("fp8")
    try:
        with torch.no_grad():
            for _ in range(3):
                out, _ = layer(x)
                fresh = ffm.MoELayer(256, 512, 4, top_k=2).to(DEV).bfloat16()
                fresh.load_state_dict(layer.state_dict())
                assert torch.equal(out, fresh(x)[0])
                graph.replay()
    finally:
        ffm.set_expert_gemm_precision(old)
    # once the weights are gone their address may be another tensor's
    assert layer_module._is_written_by_replays(layer.w_up)
    at = layer.w_up.untyped_storage().data_ptr()
    opt.state.clear()
    del layer, opt, graph, p
    gc.collect()
    ref = layer_module._replayed.get(at)
    assert ref is None or ref.expired()


def test_fp8_copies_made_in_a_capture_are_not_kept():
    """They are not filled before a replay."""
    torch.manual_seed(4)
    layer = ffm.MoELayer(256, 512, 4, top_k=2).to(DEV).bfloat16()
    x = torch.randn(2048, 256, device=DEV).bfloat16()
    with torch.no_grad():
        layer(x)
        torch.cuda.synchronize()
        old = ffm.set_expert_gemm_precision("fp8")
        try:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                captured, _ = layer(x)
            eager, _ = layer(x)
            twin = ffm.MoELayer(256, 512, 4, top_k=2).to(DEV).bfloat16()
            twin.load_state_dict(layer.state_dict())
            want, _ = twin(x)
            assert torch.equal(eager, want)
            graph.replay()
            assert torch.equal(captured, want)
        finally:
            ffm.set_expert_gemm_precision(old)


def test_fp8_training_steps_that_are_replayed_see_new_weights():
    """The weights of a captured forward and backward pass are updated between replays; the e4m3 copies kept from before the capture
    are not its."""
    torch.manual_seed(6)
    layer = ffm.MoELayer(256, 512, 4, top_k=2).to(DEV).bfloat16()
    x = torch.randn(2048, 256, device=DEV).bfloat16().requires_grad_()
    go = torch.randn_like(x)
    leaves = [x, *layer.parameters()]
    old = ffm.set_expert_gemm_precision("fp8")
    try:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                torch.autograd.grad(layer(x)[0], leaves, go)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out, _ = layer(x)
            grads = torch.autograd.grad(out, leaves, go)
        for _ in range(2):
            with torch.no_grad():
                layer.w_up.mul_(0.5)
                layer.w_down.add_(0.01)
            graph.replay()
            torch.cuda.synchronize()
            want, _ = layer(x)
            assert torch.equal(out, want)
            assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(want, leaves, go)))
    finally:
        ffm.set_expert_gemm_precision(old)
