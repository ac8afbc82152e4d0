"""Layer norm and root-mean-square norm over the last dimension: the norm in front of the MoE layer (MoELayer(pre_norm=...)), forward and
backward in the kernels of libffmoe."""

import torch
import torch.nn as nn

from . import _lib


@torch.compiler.disable
def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension of x [*, D].

    x, weight [D] and bias [D] (None: 1 and 0) are CUDA tensors in bfloat16, float16 or float32, each in its own; y has x's
    type and shape and is contiguous. Statistics are fp32, and so is everything in between. D is any number up to 32768
    (float32: 16384). The rows of x may be further apart than D; other strides are copied. Differentiable once, in reverse mode, with the
    gradients of weight and bias summed in a fixed order."""
    return _lib.native().layer_norm(x, weight, bias, eps)


@torch.compiler.disable
def rms_norm(x, weight=None, eps=1e-6, *, residual=None, weight_offset=0.0, quantize=False):
    """h / sqrt(mean(h^2) + eps) * (weight + weight_offset) over the last dimension of h = x + residual.

    Without a residual h is x, and the result is y. With one (of x's shape and type) the sum is rounded to x's type, and the result is
    (y, h): h is the residual stream to hand on. weight_offset = 1 is for weights that are stored less 1.

    quantize=True makes y the operand of linear_e4m3(): float8_e4m3fn values and a float32 scale for every 128 columns, those of
    quantize_e4m3() for y in fp32; the result is (values, scales) or (values, scales, h). D is a multiple of 16 then, and the call is not differentiable.

    x, residual and weight [D] (None: 1) are CUDA tensors in bfloat16, float16 or float32, the weight in its own; y and h have x's type and
    shape and are contiguous. Everything between is fp32. D is any number up to 32768 (float32: 16384). The rows of x and residual may be further
    apart than D; other strides are copied. Differentiable once, in reverse mode, through y and h, with the weight's gradient summed
    in a fixed order."""
    return _lib.native().rms_norm(x, weight, eps, residual, weight_offset, quantize)


class LayerNorm(nn.Module):
    """layer_norm() with its parameters; names, defaults and initial values of torch.nn.LayerNorm over one dimension."""

    def __init__(self, normalized_shape, eps=1e-5, elementwise_affine=True, bias=True, device=None, dtype=None):
        super().__init__()
        shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(normalized_shape)
        if len(shape) != 1 or shape[0] < 1:
            raise ValueError(f"LayerNorm normalises one dimension, got {shape}")
        self.normalized_shape = shape
        self.eps = eps
        self.elementwise_affine = elementwise_affine
        if elementwise_affine:
            self.weight = nn.Parameter(torch.empty(shape, device=device, dtype=dtype))
        else:
            self.register_parameter("weight", None)
        if elementwise_affine and bias:
            self.bias = nn.Parameter(torch.empty(shape, device=device, dtype=dtype))
        else:
            self.register_parameter("bias", None)
        self.reset_parameters()

    def reset_parameters(self):
        if self.weight is not None:
            nn.init.ones_(self.weight)
        if self.bias is not None:
            nn.init.zeros_(self.bias)

    def forward(self, x):
        if x.shape[-1:] != self.normalized_shape:
            raise ValueError(f"x must end in {self.normalized_shape}, got {tuple(x.shape)}")
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self):
        return f"{self.normalized_shape}, eps={self.eps}, elementwise_affine={self.elementwise_affine}"


class RMSNorm(nn.Module):
    """rms_norm() with its weight; names, defaults and initial values of torch.nn.RMSNorm over one dimension, but for eps=None. forward takes
    rms_norm()'s `residual` and `quantize`."""

    def __init__(self, normalized_shape, eps=1e-6, elementwise_affine=True, device=None, dtype=None, *, weight_offset=0.0):
        super().__init__()
        shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(normalized_shape)
        if len(shape) != 1 or shape[0] < 1:
            raise ValueError(f"RMSNorm normalises one dimension, got {shape}")
        self.normalized_shape = shape
        self.eps = eps
        self.elementwise_affine = elementwise_affine
        self.weight_offset = weight_offset
        if elementwise_affine:
            self.weight = nn.Parameter(torch.empty(shape, device=device, dtype=dtype))
        else:
            self.register_parameter("weight", None)
        self.reset_parameters()

    def reset_parameters(self):
        if self.weight is not None:
            nn.init.constant_(self.weight, 1.0 - self.weight_offset)

    def forward(self, x, residual=None, quantize=False):
        if x.shape[-1:] != self.normalized_shape:
            raise ValueError(f"x must end in {self.normalized_shape}, got {tuple(x.shape)}")
        offset = self.weight_offset if self.weight is not None else 0.0
        return rms_norm(x, self.weight, self.eps, residual=residual, weight_offset=offset, quantize=quantize)

    def extra_repr(self):
        return f"{self.normalized_shape}, eps={self.eps}, elementwise_affine={self.elementwise_affine}, weight_offset={self.weight_offset}"
