"""8-bit operands (e4m3) with a scale for every 128 values, and their products: dense, or grouped by expert with ragged sizes."""

import torch

from . import _lib, ops


@torch.compiler.disable
def quantize_e4m3(x, block_rows=1):
    """(values, scales): x [*, K] as float8_e4m3fn numbers and float32 scales, x close to values * scale in every block.

    block_rows = 1 (activations): a scale for 128 values of a row, scales [*, ceil(K / 128)]. block_rows = 128 (weights): x is [*, N, K] and
    a scale serves 128 x 128 values, scales [*, ceil(N / 128), ceil(K / 128)]. Blocks at the ends may be smaller. The scale is the block's
    largest magnitude / 448, at least 2^-126, and 1 for a block of zeros, and the values are (x / scale).to(torch.float8_e4m3fn), both quotients
    rounded as fp32 division rounds them. NaN values stay NaN and do not count for the scale; a block with an
    infinity has an infinite scale and stands for NaN throughout.

    x: a CUDA tensor in bfloat16, float16 or float32, K a multiple of 16; what is not contiguous (block_rows = 1: whose rows are not) is
    copied. Not differentiable."""
    return _lib.native().quantize_e4m3(x, block_rows)


@torch.compiler.disable
def linear_e4m3(x, x_scale, weight, weight_scale, *, ends=None, out_dtype=torch.bfloat16):
    """x weight^T of e4m3 operands with a scale for every block of 128, as quantize_e4m3() and rms_norm(quantize=True) make them.

    x [*, K] with x_scale [*, ceil(K / 128)], weight [N, K] with weight_scale [ceil(N / 128), ceil(K / 128)]: the result is [*, N] in
    `out_dtype` (bfloat16, float16 or float32), summed in fp32 and rounded once; x_scale * weight_scale is formed in fp32 and has to be a normal
    number or infinite there. K is a multiple of 16, N and the number of rows any.

    Grouped by expert: x [rows, K], weight [experts, N, K], weight_scale [experts, ceil(N / 128), ceil(K / 128)] and ends [experts]
    (int32, on the device): rows ends[e - 1] to ends[e] - 1 of x are multiplied by weight[e]. Experts may have no rows, and rows from the
    last end on belong to none: the result is 0 there. ends must not decrease nor pass the number of rows; a call where they do raises from a
    later one, as other device failures do. At most 1024 experts.

    Everything runs on the current stream without a host wait and can be captured, except for a device's first call. Not differentiable."""
    for t, name in ((x, "x"), (x_scale, "x_scale"), (weight, "weight"), (weight_scale, "weight_scale")):
        if not t.is_cuda:
            raise RuntimeError(f"{name} must be a CUDA tensor: flashfusedmoe_b200 has no CPU path")
    if ops.first_call(x.device) and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("the first call on a device cannot be captured: make one before")
    ops.raise_reported(x.device)
    return _lib.native().linear_e4m3(x, x_scale, weight, weight_scale, ends, out_dtype, ops.status_tensor(x.device).data_ptr(),
                                     ops.reported_word(x.device))
