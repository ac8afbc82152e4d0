"""AdamW goes on from state dicts that it did not make itself with all that its options say."""

import pytest
import torch


def _torchs(dtype, device, size=5000, steps=3):
    """A parameter and the state dict of torch.optim.AdamW after some steps with it. (In fp16 a few values become NaN there: their second
    moment and eps are zero.)"""
    torch.manual_seed(0)
    p = torch.nn.Parameter((torch.rand(size, device=device) + 1.0).to(dtype))
    opt = torch.optim.AdamW([p], lr=1e-3)
    for _ in range(steps):
        p.grad = torch.randn_like(p)
        opt.step()
    return p, opt.state_dict()


def test_a_master_is_made_where_a_loaded_state_has_none():
    from flashfusedmoe_b200 import AdamW
    for options, dtype, expected in (({}, torch.bfloat16, True), ({}, torch.float16, True), ({}, torch.float32, False),
                                     ({"master_weights": False}, torch.bfloat16, False)):
        p, state = _torchs(dtype, "cpu")
        opt = AdamW([p], **options)
        opt.load_state_dict(state)
        with torch.no_grad():
            p.mul_(0.5)   # weights that are loaded after the optimizer's state
        s = opt._state_of(p, opt.param_groups[0])
        assert ("master" in s) == expected and s["step"].item() == 3
        if expected:
            assert s["master"].dtype == torch.float32 and torch.equal(s["master"].to(dtype).view(torch.int16), p.detach().view(torch.int16))
            again = AdamW([p])
            again.load_state_dict(opt.state_dict())
            with torch.no_grad():
                p.mul_(0.5)
            kept = again._state_of(p, again.param_groups[0])["master"]   # a loaded one stays
            assert torch.equal(kept.view(torch.int32), s["master"].view(torch.int32))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_small_updates_add_up_after_a_torch_state_was_loaded(dtype):
    """Steps of about 2^-14 at parameters from 1 to 2, whose half units are 2^-8 and 2^-11: each alone is lost, 256 are 2^-6 (the ratio of the moments
    is within a tenth of 1 after the first of these equal gradients have outweighed the old ones)."""
    from flashfusedmoe_b200 import AdamW
    p, state = _torchs(dtype, "cuda", steps=1)
    opt = AdamW([p], betas=(0.5, 0.5), weight_decay=0.0)
    opt.load_state_dict(state)
    for g in opt.param_groups:
        g.update(lr=2.0 ** -14, betas=(0.5, 0.5), weight_decay=0.0)
    old = p.detach().clone()
    p.grad = torch.ones_like(p)
    for _ in range(256):
        opt.step()
    finite = old.isfinite()
    moved = (old.double() - p.detach().double())[finite]
    assert finite.sum() > 4500
    assert (moved >= 2.0 ** -6 * 0.9 - 2.0 ** -8).all() and (moved <= 2.0 ** -6 * 1.1 + 2.0 ** -8).all()


@pytest.mark.gpu
def test_a_step_that_makes_a_master_is_not_captured():
    from flashfusedmoe_b200 import AdamW
    p, state = _torchs(torch.bfloat16, "cuda")
    opt = AdamW([p])
    opt.load_state_dict(state)
    p.grad = torch.ones_like(p)
    torch.cuda.synchronize()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(RuntimeError, match="cannot be captured"):
            opt.step()
    opt.step()
    assert "master" in opt.state[p]
