"""Cross entropy of hidden rows against a vocabulary, without the logits: the loss behind a model's last layer, beside the MoE
layer's own two losses."""

import torch

from . import _lib, ops
from .fused_moe import _get_compute_dtype, _require_bf16

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


@torch.compiler.disable
def linear_cross_entropy(hidden, weight, target, *, ignore_index=-100, reduction="mean", z_loss_coeff=0.0, _piece_rows=0):
    """Softmax cross entropy of the logits hidden weight^T, which are never stored: with lse = log sum exp of a row's logits,
    lse - logit[target] + z_loss_coeff * lse^2 for every row, 0 where the target is ignore_index.

    hidden [*, D] and weight [V, D] are CUDA tensors, D a multiple of 8, V any number, both on 16 bytes
    (as allocated; rows that are not contiguous are copied); target [*] is int64. As in fused_moe()
    the compute type is the autocast type if autocast is on, else hidden's, and has to be bfloat16; gradients come in the
    tensors' own types (the weight's, where that is float32, without a rounding in between). reduction: "mean" over the rows that
    are not ignored (NaN without any, with zero gradients), "sum", or "none" (float32 [*]). The result is float32.

    With "mean" and "sum" the gradients are computed together with the loss, wherever hidden or weight requires one: under
    torch.no_grad() the call takes a third of the time. With "none" they are computed in the backward pass, which takes the logits a second
    time. Scratch: without gradients 8 bytes for 128 entries; with them 2 bytes an entry (a probability, then its gradient) for as many rows as
    2 GiB hold, 4 V D bytes where that is not all of them and the weight's gradient is not float32, and up to 64 N D bytes for few rows.
    Precision: logits, sums and losses are fp32. Probabilities are fp16 numbers over the largest of 128 neighbouring entries: 11 bits
    down to e^-20 of that one, nothing below e^-27. The gradients of the logits are bf16, as the products' operands; so are gradients of bf16
    operands before the backward pass's factor, where that is not 1, multiplies them.
    Differentiable once, in reverse mode; a device's first call cannot be captured. A target outside of the vocabulary gives NaN, and raises from a
    later call as other device failures do."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"Unknown reduction: {reduction}")
    for t, name in ((hidden, "hidden"), (weight, "weight"), (target, "target")):
        if not t.is_cuda:
            raise RuntimeError(f"{name} must be a CUDA tensor: flashfusedmoe_b200 has no CPU path")
    if not hidden.device == weight.device == target.device:
        raise ValueError("All tensors must be on same device")
    _require_bf16(_get_compute_dtype(hidden.dtype))
    if not (hidden.is_floating_point() and weight.is_floating_point()):
        raise TypeError(f"hidden and weight must be floating-point tensors, got {hidden.dtype} and {weight.dtype}")
    if weight.dim() != 2 or hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"weight must be [V, {hidden.shape[-1] if hidden.dim() else '?'}], got {tuple(weight.shape)}")
    if weight.shape[0] < 1 or weight.shape[1] < 1 or weight.shape[1] % 8 != 0:
        raise ValueError(f"D must be a multiple of 8 and V positive, got {tuple(weight.shape)}")
    if target.shape != hidden.shape[:-1]:
        raise ValueError(f"target must be {tuple(hidden.shape[:-1])}, got {tuple(target.shape)}")
    if target.dtype != torch.int64:
        raise TypeError(f"target must be int64, got {target.dtype}")
    if not z_loss_coeff >= 0.0:
        raise ValueError(f"z_loss_coeff must not be negative, got {z_loss_coeff}")
    if not ops.has_status(hidden.device) and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("the first call on a device cannot be captured: make one before")
    ops.raise_reported(hidden.device)
    return _lib.native().linear_cross_entropy(hidden, weight, target, ignore_index, _REDUCTIONS[reduction], z_loss_coeff, _piece_rows,
                                              ops.status_tensor(hidden.device).data_ptr(), ops.reported_word(hidden.device))
