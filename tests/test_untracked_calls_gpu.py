"""Calls whose result torch would take for something else than it is are refused: forward-mode tangents, which would be dropped, and
traces, which would hold outputs that nothing fills."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from flashfusedmoe_b200 import _lib, adamw_step, layer_norm, linear_cross_entropy


def refuse(call, match):
    with pytest.raises(RuntimeError, match=match):
        call()


def calls(device, dual):
    """Every operator with every operand `dual` once."""
    x, v = torch.randn(4, 64, device=device), torch.randn(64, device=device)
    h, w = x.bfloat16(), torch.randn(30, 64, device=device).bfloat16()
    t = torch.zeros(4, dtype=torch.int64, device=device)
    native = (t, -100, 1, 0.0, 0, 0, 0)   # the checks in Python come first on the host
    yield lambda: layer_norm(dual(x))
    yield lambda: layer_norm(x, dual(v))
    yield lambda: layer_norm(x, v, dual(v))
    yield lambda: layer_norm(x.detach().requires_grad_(), dual(v))
    if device == "cuda":
        yield lambda: linear_cross_entropy(dual(h), w, t)
        yield lambda: linear_cross_entropy(h.detach().requires_grad_(), dual(w), t)
    else:
        yield lambda: _lib.native().linear_cross_entropy(dual(h), w, *native)
        yield lambda: _lib.native().linear_cross_entropy(h, dual(w), *native)
    for k in range(4):
        operands = [torch.zeros(8, device=device) for _ in range(4)]
        operands[k] = dual(operands[k])
        step = torch.zeros((), dtype=torch.int32, device=device)
        yield lambda: adamw_step(*[[o] for o in operands], [step], lr=1e-3)


def check_tangents(device):
    with forward_ad.dual_level():
        for call in calls(device, lambda a: forward_ad.make_dual(a, torch.ones_like(a))):
            refuse(call, "forward-mode" if device == "cuda" else "forward-mode|no CPU path")


def test_tangents_on_the_host():
    check_tangents("cpu")
    with forward_ad.dual_level():
        x = torch.randn(4, 64)
        refuse(lambda: layer_norm(forward_ad.make_dual(x, x)), "forward-mode")


def test_traces_on_the_host():
    from torch.fx.experimental.proxy_tensor import make_fx
    x = torch.randn(4, 64)
    refuse(lambda: torch.jit.trace(layer_norm, x), "cannot be traced")
    refuse(lambda: make_fx(lambda a: layer_norm(a))(x), "cannot be traced")
    refuse(lambda: layer_norm(x), "no CPU path")   # and nothing is left behind


@pytest.mark.gpu
def test_tangents():
    check_tangents("cuda")
    x, w = torch.randn(4, 64, device="cuda").bfloat16().requires_grad_(), torch.randn(30, 64, device="cuda").bfloat16()
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    with forward_ad.dual_level():
        for y in (layer_norm(x), linear_cross_entropy(x, w, t), linear_cross_entropy(x, w, t, reduction="none")):
            one = torch.ones_like(y)
            refuse(lambda: torch.autograd.grad(y, x, forward_ad.make_dual(one, one)), "forward-mode")
        torch.autograd.grad(layer_norm(x).sum(), x)   # none of the operands has one


@pytest.mark.gpu
def test_traces():
    from torch.fx.experimental.proxy_tensor import make_fx
    x, w = torch.randn(4, 64, device="cuda").bfloat16(), torch.randn(30, 64, device="cuda").bfloat16()
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    linear_cross_entropy(x, w, t)
    for call in (lambda a: layer_norm(a), lambda a: linear_cross_entropy(a, w, t), lambda a: linear_cross_entropy(a, w, t, reduction="none")):
        for leaf in (x, x.detach().requires_grad_()):
            refuse(lambda: torch.jit.trace(call, leaf), "cannot be traced")
            refuse(lambda: make_fx(call)(leaf), "cannot be traced")


@pytest.mark.gpu
def test_function_transforms_are_refused():
    x, w = torch.randn(4, 64, device="cuda").bfloat16(), torch.randn(30, 64, device="cuda").bfloat16()
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    for call in (lambda a: layer_norm(a).float().sum(), lambda a: linear_cross_entropy(a, w, t)):
        refuse(lambda: torch.func.grad(call)(x), "functorch")
        refuse(lambda: torch.func.jvp(call, (x,), (x,)), "storage|forward-mode")
        refuse(lambda: torch.func.vmap(call)(x[None]), "storage")
