"""The norm of all gradients together and clipping by it: the coefficient that AdamW's step takes (grad_scale), or gradients scaled in
place."""

import torch
import torch.distributed as dist

from . import _lib

_KINDS = {2.0: False, float("inf"): True}


def _arguments(max_norm, norm_type):
    norm_type = float(norm_type)
    if norm_type not in _KINDS:
        raise ValueError(f"norm_type must be 2 or inf, got {norm_type}")
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    return max_norm, _KINDS[norm_type]


def _tensors(given):
    return [given] if isinstance(given, torch.Tensor) else list(given)


def _nothing():
    """Stands for the gradients of a rank that has none, on its current device."""
    return torch.empty(0, device="cuda")


def _norm(grads, sharded, like, max_norm, largest, group):
    native, other = _lib.native(), None
    if group is not None:
        other = native.gradient_norm(sharded, like, 0.0, largest, None)[0][:1]
        if largest:
            # MAX of numbers drops a NaN of another rank. As whole numbers the bits of magnitudes compare as those do, and NaN is above all.
            bits = other.view(torch.int64) & 0x7fffffffffffffff
            dist.all_reduce(bits, dist.ReduceOp.MAX, group=group)
            other = bits.view(torch.float64)
        else:
            dist.all_reduce(other, dist.ReduceOp.SUM, group=group)
    else:
        grads = [*grads, *sharded]
    return native.gradient_norm(grads, like, max_norm, largest, other)[1:]


@torch.compiler.disable
def clip_coefficient(grads, max_norm, norm_type=2.0, *, sharded=(), group=None):
    """(norm, coefficient) of the tensors in `grads` (or of the one tensor) together: the root of the sum of all squares (norm_type 2) or the largest
    magnitude (inf), and min(1, max_norm / (norm + 1e-6)); NaN where the norm is NaN. Both are float32 on the device, and the coefficient is
    what AdamW.step(grad_scale=...) and adamw_step() take: gradients are then clipped without a pass of their own.

    CUDA tensors of one device in bfloat16, float16 or float32, in any order of their dimensions (others are copied). Sums are in
    64 bits and in a fixed order. sharded: gradients of which every rank of `group` has others, as of experts under expert parallelism
    (MoELayer.expert_params); their part of the norm is all-reduced over `group`, so every rank calls with as many tensors of its own as it
    has, none included, and gets the same norm. Without a group they count as the others. Everything runs on the current stream without a host wait and can be
    captured."""
    grads, sharded = _tensors(grads), _tensors(sharded)
    max_norm, largest = _arguments(max_norm, norm_type)
    if not grads and not sharded and group is None:
        raise ValueError("there are no gradients")
    return _norm(grads, sharded, (grads + sharded or [_nothing()])[0], max_norm, largest, group)


@torch.compiler.disable
def clip_grad_norm(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False, *, sharded=(), group=None):
    """Scales the gradients of `parameters` (a tensor or an iterable of them) in place so that their norm together is at most `max_norm`,
    as torch.nn.utils.clip_grad_norm_ does, and returns the norm before (float32 on the device): every gradient is multiplied by the
    coefficient of clip_coefficient(), and none is written where that is 1.

    sharded: those of `parameters` of which every rank of `group` has others (see clip_coefficient()). error_if_nonfinite raises
    where the norm is not finite, which waits for the device and cannot be captured. No two gradients may share memory. Parameters without a
    gradient are passed over; without any gradient the norm is 0."""
    parameters = _tensors(parameters)
    max_norm, largest = _arguments(max_norm, norm_type)
    apart = {id(p) for p in _tensors(sharded)}
    if apart and not apart <= {id(p) for p in parameters}:
        raise ValueError("sharded must be some of the parameters")
    if group is None and not error_if_nonfinite:
        norm = _lib.native().clip_grad_norm(parameters, max_norm, largest)
        return torch.zeros((), device=parameters[0].device if parameters else None) if norm is None else norm
    with_grad = [p for p in parameters if p.grad is not None]
    grads = [p.grad for p in with_grad if id(p) not in apart]
    local = [p.grad for p in with_grad if id(p) in apart]
    every = [*grads, *local]
    if not every and group is None:
        return torch.zeros((), device=parameters[0].device if parameters else None)
    norm, coefficient = _norm(grads, local, (every or parameters or [_nothing()])[0], max_norm, largest, group)
    if error_if_nonfinite and not bool(torch.isfinite(norm)):
        raise RuntimeError("The norm of the gradients is not finite, so they cannot be clipped by it")
    _lib.native().scale_gradients(every, coefficient)
    return norm
