"""AdamW over all parameters of a model in a launch per group, with its two moments in 32 or in 8 bits."""

import torch

from . import _lib
from .fused_moe import written_by_replays

BLOCK = 128   # values of a tensor that share a scale in an 8-bit state


def _capturing(tensors):
    return bool(tensors) and tensors[0].is_cuda and torch.cuda.is_current_stream_capturing()


@torch.compiler.disable
def adamw_step(params, grads, exp_avgs, exp_avg_sqs, steps, *, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, masters=None,
               exp_avg_scales=None, exp_avg_sq_scales=None, grad_scale=None, seed=0):
    """One AdamW step of the tensors in `params`, in place: m = b1 m + (1 - b1) g, v = b2 v + (1 - b2) g^2,
    p = p (1 - lr weight_decay) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps).

    Lists of CUDA tensors of one device, one entry a parameter: params (bfloat16, float16 or float32, contiguous) and grads
    (any of these types); steps, int32 tensors of one element, raised by one (t is the raised value); exp_avgs and
    exp_avg_sqs, float32. With exp_avg_scales and exp_avg_sq_scales (uint8, one for every 128 values) the moments are held in
    8 bits: exp_avgs[i] are float8_e4m3fn numbers of m over 2^(scale - 127), exp_avg_sqs[i] those of sqrt(v). m is rounded to
    nearest, sqrt(v) at random by `seed`, step and place (the average moves by less than the distance of two such
    numbers), a positive v never to zero; what is not finite becomes NaN.

    masters (float32): the parameters that are updated, of which `params` then are the rounded copies. grad_scale: one
    float32 on the device that multiplies every gradient (a clipping coefficient). lr: a number, or one float32 on the
    device, which a captured step reads at every replay. What is written lies on nothing else of the call. Everything runs on the
    current stream without a host wait and can be captured."""
    capturing = _capturing(params)
    _lib.native().adamw_step(params, grads, exp_avgs, exp_avg_sqs, steps, masters, exp_avg_scales, exp_avg_sq_scales, lr, betas[0],
                             betas[1], eps, weight_decay, grad_scale, seed & 0xFFFFFFFF, capturing)
    if capturing:
        written_by_replays(params)


def _in_8_bits(moment, root):
    """A moment in 32 bits as codes and scales of adamw_step() (of its root). Rounded to nearest, the root too: this is done once, on loading."""
    x = (moment.sqrt() if root else moment).reshape(-1)
    blocks = torch.cat([x, x.new_zeros(-x.numel() % BLOCK)]).view(-1, BLOCK)
    finite = blocks.isfinite()
    top = torch.where(finite, blocks.abs(), 0.0).amax(1)
    mantissa, exponent = torch.frexp(top)   # 448, the largest number, is 0.875 * 2^9
    k = torch.where(top > 0, exponent - 9 + (mantissa > 0.875).int(), -126).clamp(-126, 120)
    codes = torch.where(finite, torch.ldexp(blocks, -k[:, None]), torch.nan).to(torch.float8_e4m3fn).view(torch.uint8)
    if root:
        codes = torch.where(blocks > 0, codes.clamp(min=1), codes)
    return codes.view(-1)[:x.numel()].clone().view(torch.float8_e4m3fn).view(moment.shape), (k + 127).to(torch.uint8)


class AdamW(torch.optim.Optimizer):
    """AdamW with a launch per parameter group. state_bits = 8 holds both moments of tensors of at least `min_8bit_size`
    values in 8 bits (2 bytes a parameter instead of 8; adamw_step() says how), those of smaller ones, where nothing is to
    be saved, in 32. master_weights keeps a float32 copy of parameters of fewer bits, which the updates go to: without it an
    update of less than half a unit of a bfloat16 parameter's last place is lost.

    Parameters are contiguous CUDA tensors. lr may be a float32 tensor on the device: a step that was captured in a graph then
    reads it at every replay. State dicts load and save as torch's do, and one of torch.optim.AdamW can be loaded: its moments go to 8 bits
    where state_bits says so, and the first step makes masters that it does not have (from the parameters as they are then); `step` counts
    on the device."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, *, state_bits=32, master_weights=True,
                 min_8bit_size=4096, seed=0):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        if not torch.is_tensor(lr) and not lr >= 0.0:
            raise ValueError(f"lr must not be negative, got {lr}")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"betas must be in [0, 1), got {betas}")
        if not eps >= 0.0 or not weight_decay >= 0.0:
            raise ValueError(f"eps and weight_decay must not be negative, got {eps} and {weight_decay}")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      master_weights=master_weights, min_8bit_size=min_8bit_size, seed=seed))

    def _state_of(self, p, group):
        state = self.state[p]
        if not state:
            if _capturing([p]):
                raise RuntimeError("a parameter's first AdamW step makes its state and cannot be captured: take one step before")
            state["step"] = torch.zeros((), dtype=torch.int32, device=p.device)
            if group["state_bits"] == 8 and p.numel() >= group["min_8bit_size"]:
                for name in ("exp_avg", "exp_avg_sq"):
                    state[name] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device).view(torch.float8_e4m3fn)
                    state[name + "_scale"] = torch.zeros((p.numel() + BLOCK - 1) // BLOCK, dtype=torch.uint8, device=p.device)
            else:
                for name in ("exp_avg", "exp_avg_sq"):
                    state[name] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        # (also where a loaded state had none: made as late as this, since the parameters may be loaded after it)
        if group["master_weights"] and p.dtype != torch.float32 and "master" not in state:
            if _capturing([p]):
                raise RuntimeError("a parameter's first AdamW step after loading makes its master and cannot be captured: take one step before")
            state["master"] = p.detach().to(torch.float32, memory_format=torch.contiguous_format)
        return state

    def load_state_dict(self, state_dict):
        """As torch's, but every state keeps its own type: there, floating states take their parameter's. Steps and unscaled
        moments of another optimizer become int32 and float32, or 8 bits where the group's state_bits says so; one whose step is another
        is refused."""
        own = [dict(g) for g in self.param_groups]
        given = {}

        def look(_, state_dict):   # what the hooks before made of it
            for group in state_dict["param_groups"]:
                for name in ("amsgrad", "maximize"):
                    if group.get(name):
                        raise ValueError(f"a state dict with {name} is of another step than AdamW's here")
                if group["weight_decay"] != 0 and not group.get("decoupled_weight_decay", True):
                    raise ValueError("a state dict whose weight decay is part of the gradient is of another step than AdamW's here")
            given.update(state_dict)

        # last of the hooks before loading, first of those after it
        hooks = [self.register_load_state_dict_pre_hook(look),
                 self.register_load_state_dict_post_hook(lambda _: self._take_states(given, own), prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    def _take_states(self, state_dict, own):
        for group, mine in zip(self.param_groups, own):   # options that another optimizer's groups do not have
            for name, value in mine.items():
                group.setdefault(name, value)
            group.pop("decoupled_weight_decay", None)   # it always is here
        order = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [(p, g) for g in self.param_groups for p in g["params"]]
        for i, (p, group) in zip(order, params):
            old = {k: v for k, v in state_dict["state"].get(i, {}).items() if torch.is_tensor(v)}
            for name, value in old.items():
                kind = value.dtype
                if name == "step":
                    kind = torch.int32
                elif name in ("exp_avg", "exp_avg_sq") and name + "_scale" not in old:
                    kind = torch.float32
                self.state[p][name] = value.detach().to(p.device, kind, copy=True).contiguous()
            if group["state_bits"] == 8 and p.numel() >= group["min_8bit_size"] and "exp_avg" in old and "exp_avg_scale" not in old:
                for name in ("exp_avg", "exp_avg_sq"):
                    self.state[p][name], self.state[p][name + "_scale"] = _in_8_bits(self.state[p][name], root=name == "exp_avg_sq")

    @torch.no_grad()
    def step(self, closure=None, *, grad_scale=None):
        """Updates every parameter that has a gradient. grad_scale (one float32 on the device) multiplies the gradients."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            # one launch holds one kind of state: 8 or 32 bits, with masters or without, on one device
            kinds = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("AdamW does not take sparse gradients")
                s = self._state_of(p, group)
                kinds.setdefault((p.device, "exp_avg_scale" in s, "master" in s), []).append((p, s))
            for (_, eight, master), entries in kinds.items():
                def column(name, entries=entries):
                    return [s[name] for _, s in entries]

                adamw_step([p for p, _ in entries], [p.grad for p, _ in entries], column("exp_avg"), column("exp_avg_sq"),
                           column("step"), lr=group["lr"], betas=group["betas"], eps=group["eps"],
                           weight_decay=group["weight_decay"], masters=column("master") if master else None,
                           exp_avg_scales=column("exp_avg_scale") if eight else None,
                           exp_avg_sq_scales=column("exp_avg_sq_scale") if eight else None, grad_scale=grad_scale,
                           seed=group["seed"])
        return loss
