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


def _decoded(codes, scale, root=False):
    x = codes.reshape(-1).double() * torch.pow(2.0, scale.double() - 127).repeat_interleave(128)[:codes.numel()]
    return (x * x if root else x).view(codes.shape)


@pytest.mark.parametrize("shape", [(5000,), (33, 129), (4096,)])
def test_loaded_moments_are_held_in_8_bits_where_the_group_says_so(shape):
    """To nearest: half a step, 2^-4 of a value or 2^-10 of its block's scale, of the root for the second moment (twice that of the
    moment itself, and its square); the root itself is off by 2^-24."""
    from flashfusedmoe_b200 import AdamW
    n = torch.Size(shape).numel()
    p, state = _torchs(torch.float32, "cpu", size=n)
    with torch.no_grad():
        s = state["state"][0]
        s["exp_avg"].mul_(torch.logspace(-12, 3, n))
        s["exp_avg_sq"].mul_(torch.logspace(-40, 3, n))
        s["exp_avg"][:300] = s["exp_avg_sq"][:300] = 0.0
        s["exp_avg"][200], s["exp_avg_sq"][201], s["exp_avg"][202] = float("nan"), float("inf"), 3.0
    p = torch.nn.Parameter(p.detach().view(shape))
    s["exp_avg"], s["exp_avg_sq"] = s["exp_avg"].view(shape), s["exp_avg_sq"].view(shape)
    opt = AdamW([p], state_bits=8)
    opt.load_state_dict(state)
    mine = opt.state[p]
    for name, root in (("exp_avg", False), ("exp_avg_sq", True)):
        codes, scale = mine[name], mine[name + "_scale"]
        assert codes.dtype == torch.float8_e4m3fn and codes.shape == torch.Size(shape) and codes.is_contiguous()
        assert scale.dtype == torch.uint8 and scale.numel() == (n + 127) // 128
        want = s[name].view(-1).double()
        want = want.sqrt() if root else want
        got = _decoded(codes, scale).view(-1)
        finite = want.isfinite()
        assert got[~finite].isnan().all() and got[finite].isfinite().all()
        unit = torch.pow(2.0, scale.double() - 127).repeat_interleave(128)[:n]
        limit = torch.maximum(want.abs() * (2.0 ** -4 + 2.0 ** -23), unit * 2.0 ** -10)
        if root:
            assert ((got > 0) == (want > 0))[finite].all()
            limit = torch.where(got == unit * 2.0 ** -9, unit * 2.0 ** -9, limit)   # what would be zero is the least number
        assert ((got - want).abs() <= limit)[finite].all()
        # the least power of two that holds the block's largest
        top = torch.where(finite, want.abs(), 0.0)
        top = torch.cat([top, top.new_zeros(-n % 128)]).view(-1, 128).amax(1)
        k = torch.pow(2.0, scale.double() - 127)
        assert (top <= 448 * k * (1 + 2.0 ** -23)).all() and ((top > 224 * k * (1 - 2.0 ** -23)) | (scale == 1)).all()
    assert mine["step"].item() == 3
    # what is smaller than the group's bound stays in 32 bits, as do groups of 32
    for options in ({"state_bits": 8, "min_8bit_size": n + 1}, {}):
        other = AdamW([p], **options)
        other.load_state_dict(state)
        assert other.state[p]["exp_avg"].dtype == torch.float32 and "exp_avg_scale" not in other.state[p]


@pytest.mark.gpu
def test_a_step_after_moments_were_loaded_into_8_bits():
    """The kernel reads the loaded moments as they were written: without gradients they fall by their factors, and the parameter moves by their quotient."""
    from flashfusedmoe_b200 import AdamW
    p, state = _torchs(torch.float32, "cuda", size=5003)
    opt = AdamW([p], state_bits=8, weight_decay=0.0)
    opt.load_state_dict(state)
    s = opt.state[p]
    m = _decoded(s["exp_avg"], s["exp_avg_scale"])
    v = _decoded(s["exp_avg_sq"], s["exp_avg_sq_scale"], root=True)
    group = opt.param_groups[0]
    (b1, b2), lr, eps, decay = group["betas"], group["lr"], group["eps"], group["weight_decay"]
    old = p.detach().double()
    p.grad = torch.zeros_like(p)
    opt.step()
    update = lr / (1 - b1 ** 4) * (b1 * m) / ((b2 * v / (1 - b2 ** 4)).sqrt() + eps)
    want = old * (1 - lr * decay) - update
    # as in test_adamw_gpu: 32 u of the update, 4 u of the parameter, and 4 u of either moment
    assert ((p.detach().double() - want).abs() <= 2.0 ** -24 * (40 * update.abs() + 8 * old.abs())).all()
    assert s["step"].item() == 4


def test_hooks_see_and_change_what_is_loaded():
    """A hook may hand back another state dict (fewer states, other values, other options); hooks after loading see it as it stays."""
    from flashfusedmoe_b200 import AdamW
    p, state = _torchs(torch.bfloat16, "cpu")
    q = torch.nn.Parameter(torch.ones(7))
    theirs = torch.optim.AdamW([p, q], lr=1e-3)
    p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    theirs.step()
    opt = AdamW([p, q])
    seen = []

    def other(_, state_dict):
        first = dict(state_dict["state"][0])
        first["exp_avg"] = first["exp_avg"] * 0.5
        return {"state": {0: first}, "param_groups": [dict(g, lr=0.25) for g in state_dict["param_groups"]]}

    handles = [opt.register_load_state_dict_pre_hook(other),
               opt.register_load_state_dict_post_hook(lambda o: seen.append({k: v.dtype for k, v in o.state[p].items()}))]
    state = theirs.state_dict()
    opt.load_state_dict(state)
    assert torch.equal(opt.state[p]["exp_avg"], state["state"][0]["exp_avg"].float() * 0.5) and not opt.state[q]
    assert opt.param_groups[0]["lr"] == 0.25 and opt.param_groups[0]["state_bits"] == 32
    assert seen == [{"step": torch.int32, "exp_avg": torch.float32, "exp_avg_sq": torch.float32}]
    # a hook that turns a state dict into one that can be loaded, or into one that cannot
    handles[0].remove()
    turn = opt.register_load_state_dict_pre_hook(
        lambda _, s: {**s, "param_groups": [dict(g, amsgrad=not g["amsgrad"]) for g in s["param_groups"]]})
    odd = {**state, "param_groups": [dict(g, amsgrad=True) for g in state["param_groups"]]}
    opt.load_state_dict(odd)
    assert torch.equal(opt.state[p]["exp_avg"], state["state"][0]["exp_avg"].float())
    before = {k: v.clone() for k, v in opt.state[p].items()}
    with pytest.raises(ValueError, match="another step"):
        opt.load_state_dict(state)
    assert all(torch.equal(v, before[k]) for k, v in opt.state[p].items())
    # the hooks that loading itself uses are gone again
    turn.remove()
    assert len(opt._optimizer_load_state_dict_pre_hooks) == 0 and len(opt._optimizer_load_state_dict_post_hooks) == 1
