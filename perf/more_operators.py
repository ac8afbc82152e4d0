"""More operators around the fused MoE layer, over the sizes they are used at: the root-mean-square norm with the residual's
addition (forward and backward, or with an output in 8 bits), quantising to 8 bits with a scale for each block of 128, products of
such operands (dense, and grouped by expert with ragged sizes), and the norm of all gradients with clipping.

A case is one call of a user's program. `run` computes it in plain torch operations, in 32 bits, or with `own` set through the
framework's kernels.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 128          # values that share a scale
TOP = 448.0          # the largest e4m3 number
LEAST = 2.0 ** -126  # the smallest scale
EPS = 1e-6           # of the norm, and what is added to the gradients' norm


# ---------------------------------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------------------------------

def _rms(rows, dim, dtype="bf16", backward=False, residual=True, quantize=False, offset=0.0):
    return dict(op="rms_norm", rows=rows, dim=dim, dtype=dtype, backward=backward, residual=residual, quantize=quantize,
                offset=offset)


def _quantize(matrices, rows, dim, dtype="bf16", block_rows=1):
    return dict(op="quantize", matrices=matrices, rows=rows, dim=dim, dtype=dtype, block_rows=block_rows)


def _linear(rows, width, dim, experts=0, spare=0, skew=0.0, dtype="bf16"):
    """`rows` by width products of dim values; with experts the rows of each lie together, and `spare` rows behind the last
    expert's belong to none. skew: how unevenly they are spread."""
    return dict(op="linear", rows=rows, width=width, dim=dim, experts=experts, spare=spare, skew=skew, dtype=dtype)


def _clip(d_model, ffn_dim, experts, layers=1, dtype="bf16", in_place=True, max_norm=1.0):
    return dict(op="clip", d_model=d_model, ffn_dim=ffn_dim, experts=experts, layers=layers, dtype=dtype, in_place=in_place,
                max_norm=max_norm)


def listed():
    def named(name, case):
        return dict(case, name=name)

    return [
        # one decoded token between two layers, its norm the next product's operand: nothing but latency
        named("rms_decode_1x4096_e4m3", _rms(1, 4096, quantize=True)),
        # the residual stream of the benchmark's training step, forward and backward
        named("rms_train_16384x1024", _rms(16384, 1024, backward=True)),
        # a ragged micro-batch of fp16 rows of odd width, without a residual: no 16-byte accesses
        named("rms_train_4093x2051_fp16", _rms(4093, 2051, dtype="fp16", backward=True, residual=False)),
        # a long prompt in wide rows, out in 8 bits: bandwidth alone
        named("rms_prefill_8192x7168_e4m3", _rms(8192, 7168, quantize=True)),
        # a serving batch's activations, a scale for 128 values of a row
        named("quantize_rows_61x7168", _quantize(1, 61, 7168)),
        # the weights of wide experts, laid out once: a scale for 128 x 128 values
        named("quantize_experts_8x14336x4096", _quantize(8, 14336, 4096, block_rows=128)),
        # one decoded token against a dense projection: the weights are streamed once
        named("linear_decode_1x4096x7168", _linear(1, 4096, 7168)),
        # 48 decoded tokens, six of 64 experts each, in a buffer that holds a few more rows
        named("linear_experts_decode_288x2816x2048", _linear(288, 2816, 2048, experts=64, spare=32, skew=0.3)),
        # a ragged prompt over 16 experts of odd width, the contraction ending inside a block, fp32 out
        named("linear_experts_ragged_9973x2815x2064", _linear(9973, 2815, 2064, experts=16, skew=1.0, dtype="fp32")),
        # the routed rows of a large batch on eight experts: the largest amount of arithmetic
        named("linear_experts_32768x4096x4096", _linear(32768, 4096, 4096, experts=8, skew=0.3)),
        # the coefficient that the optimizer step of a small fp32 layer takes: launches and latency
        named("clip_small_fp32", _clip(256, 128, 1, dtype="fp32", in_place=False)),
        # twelve layers of the benchmark's width, many tensors, clipped in place
        named("clip_layers_in_place", _clip(1024, 2816, 4, layers=12)),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["rms_norm", "rms_norm", "quantize", "linear", "linear", "clip"])
    if op == "rms_norm":
        # rows from one token to a large micro-batch; widths of any value, in 8 bits multiples of 16 (the products' operands)
        dim, quantize = log_int(64, 8192), rng.random() < 0.4
        if quantize or rng.random() < 0.5:
            dim = max(64, dim // 16 * 16)
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"]) if dim <= 3500 else "bf16"
        return _rms(log_int(1, 16384 if dim <= 3500 else 8192), dim, dtype, not quantize and rng.random() < 0.7,
                    rng.random() < 0.7, quantize, rng.choice([0.0, 0.0, 1.0]))
    if op == "quantize":
        dim = 16 * log_int(4, 448)
        if rng.random() < 0.5:
            return _quantize(1, log_int(1, 16384), dim, rng.choice(["bf16", "bf16", "fp16", "fp32"]))
        return _quantize(rng.randint(1, 8), log_int(64, 8192), dim, rng.choice(["bf16", "fp32"]), 128)
    if op == "linear":
        # contractions are multiples of 16; widths and numbers of rows of any value
        rows, width, dim = log_int(1, 16384), log_int(64, 4096), 16 * log_int(8, 256)
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        if rng.random() < 0.4:
            return _linear(rows, width, dim, dtype=dtype)
        return _linear(rows, width, dim, log_int(2, 32), rng.choice([0, 0, rng.randint(1, 200)]), rng.uniform(0.0, 1.0), dtype)
    # odd widths put the tensors' ends at any place
    return _clip(log_int(64, 2048), 2 * log_int(32, 1024), rng.randint(1, 4), rng.randint(1, 6),
                 rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.random() < 0.5, rng.choice([0.5, 1.0, 1e4]))


# ---------------------------------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rows(rows, dim, g):
    """Activations of a residual stream: rows of different scale, a few channels that stand out."""
    scale = torch.rand(rows, 1, device="cuda", generator=g) * 2.0 + 0.5
    x = torch.randn(rows, dim, device="cuda", generator=g) * scale
    x[:, :: max(1, dim // 8)] *= 5.0
    return x


def _prepare_rms(case, g):
    rows, dim, dtype = case["rows"], case["dim"], DTYPES[case["dtype"]]
    state = {"x": _rows(rows, dim, g).to(dtype), "residual": None}
    state["weight"] = (1.0 - case["offset"] + 0.2 * torch.randn(dim, device="cuda", generator=g)).to(dtype)
    if case["residual"]:
        state["residual"] = (2.0 * _rows(rows, dim, g)).to(dtype)
    if case["backward"]:
        for name in ("x", "residual", "weight"):
            if state[name] is not None:
                state[name].requires_grad_()
        state["grad"] = torch.randn(rows, dim, device="cuda", generator=g).to(dtype)
        state["grad_h"] = torch.randn(rows, dim, device="cuda", generator=g).to(dtype) if case["residual"] else None
    return state


def _prepare_quantize(case, g):
    x = _rows(case["matrices"] * case["rows"], case["dim"], g)
    if case["block_rows"] == 128:   # weights
        x = x.mul_(0.02).view(case["matrices"], case["rows"], case["dim"])
    return {"x": x.to(DTYPES[case["dtype"]])}


def _sizes(case, seed):
    """Rows of each expert."""
    rng = torch.Generator().manual_seed(seed)
    share = torch.softmax(case["skew"] * torch.randn(case["experts"], generator=rng), dim=0)
    of = torch.multinomial(share, case["rows"], replacement=True, generator=rng)
    return torch.bincount(of, minlength=case["experts"])


def _prepare_linear(case, g, seed):
    rows, width, dim, experts = case["rows"] + case["spare"], case["width"], case["dim"], case["experts"]
    x, x_scale = _quantize_plain(_rows(rows, dim, g), 1)
    shape = (experts, width, dim) if experts else (width, dim)
    weight = torch.randn(shape, device="cuda", generator=g).mul_(dim ** -0.5)
    weight, weight_scale = _quantize_plain(weight, 128)
    state = {"x": x, "x_scale": x_scale, "weight": weight, "weight_scale": weight_scale, "ends": None}
    if experts:
        sizes = _sizes(case, seed)
        state["most"] = max(1, int(sizes.max()))   # for the plain form's batch of equal sizes
        state["ends"] = sizes.cumsum(0).to(device="cuda", dtype=torch.int32)
    return state


def _elements(case):
    """Elements of each tensor: per layer a norm's weight, the gate, the experts' two projections."""
    d, f, e = case["d_model"], case["ffn_dim"], case["experts"]
    return [d, e * d, e * f * d, e * d * (f // 2)] * case["layers"]


def _prepare_clip(case, g):
    """The tensors lie in a flat buffer, each from a multiple of BLOCK on; what lies between them is zero and stays it."""
    sizes = _elements(case)
    room = [(n + BLOCK - 1) // BLOCK * BLOCK for n in sizes]
    starts = [sum(room[:i]) for i in range(len(room))]
    # gradients of very different size from tensor to tensor and row to row, as in training
    scale = torch.exp(torch.randn(sum(room) // BLOCK, 1, device="cuda", generator=g) * 2.0 - 6.0)
    grad = (torch.randn(sum(room) // BLOCK, BLOCK, device="cuda", generator=g) * scale).view(-1)
    for start, n, r in zip(starts, sizes, room):
        grad[start + n:start + r] = 0.0
    grad = grad.to(DTYPES[case["dtype"]])
    params = [torch.nn.Parameter(torch.empty_like(grad[s:s + n])) for s, n in zip(starts, sizes)]
    for p, s in zip(params, starts):
        p.grad = grad[s:s + p.numel()]
    return {"flat": grad, "params": params, "grads": [p.grad for p in params]}


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] == "linear":
        state = _prepare_linear(case, g, seed)
    else:
        state = {"rms_norm": _prepare_rms, "quantize": _prepare_quantize, "clip": _prepare_clip}[case["op"]](case, g)
    state["case"] = case
    return state


# ---------------------------------------------------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------------------------------------------------

def _quantize_plain(x, block_rows):
    """e4m3 numbers and the scales of their blocks: 128 values of a row, or 128 x 128 of a matrix."""
    rows, dim = x.shape[-2:]
    down, across = (rows + block_rows - 1) // block_rows, (dim + BLOCK - 1) // BLOCK
    blocks = torch.nn.functional.pad(x.float(), (0, across * BLOCK - dim, 0, down * block_rows - rows))
    blocks = blocks.unflatten(-1, (across, BLOCK)).unflatten(-3, (down, block_rows))
    top = blocks.abs().amax(dim=(-3, -1), keepdim=True)
    scale = torch.where(top > 0, (top / TOP).clamp(min=LEAST), 1.0)
    values = (blocks / scale).to(torch.float8_e4m3fn).flatten(-2).flatten(-3, -2)
    return values[..., :rows, :dim].contiguous(), scale.squeeze(-1).squeeze(-2)


def _dequantize_plain(values, scale, block_rows):
    rows, dim = values.shape[-2:]
    spread = scale.repeat_interleave(BLOCK, dim=-1)[..., :dim]
    if block_rows > 1:
        spread = spread.repeat_interleave(block_rows, dim=-2)[..., :rows, :]
    return values.float() * spread


def _rms_plain(s):
    case = s["case"]
    with torch.no_grad():
        h = s["x"].float()
        out = {}
        if s["residual"] is not None:
            out["h"] = (h + s["residual"].float()).to(s["x"].dtype)
            h = out["h"].float()
        w = s["weight"].float() + case["offset"]
        r = torch.rsqrt(h.square().mean(dim=1, keepdim=True) + EPS)
        y = h * r * w
        if case["quantize"]:
            out["values"], out["scale"] = _quantize_plain(y, 1)
            return out
        out["y"] = y.to(s["x"].dtype)
        if case["backward"]:
            dy, xh = s["grad"].float(), h * r
            g = dy * w
            dx = r * (g - xh * (g * xh).mean(dim=1, keepdim=True))
            if s["residual"] is not None:
                dx = dx + s["grad_h"].float()
                out["dresidual"] = dx.to(s["x"].dtype)
            out["dx"] = dx.to(s["x"].dtype)
            out["dweight"] = (dy * xh).sum(dim=0).to(s["weight"].dtype)
        return out


def _linear_plain(s):
    case = s["case"]
    with torch.no_grad():
        x = _dequantize_plain(s["x"], s["x_scale"], 1)
        w = _dequantize_plain(s["weight"], s["weight_scale"], 128)
        if s["ends"] is None:
            return {"out": (x @ w.t()).to(DTYPES[case["dtype"]])}
        # every expert's rows in a batch of equal sizes, and back
        row = torch.arange(x.shape[0], device=x.device)
        expert = torch.searchsorted(s["ends"], row.int(), right=True)
        used = expert < case["experts"]
        expert = expert.clamp(max=case["experts"] - 1)
        start = torch.nn.functional.pad(s["ends"], (1, 0))[expert]
        place = torch.where(used, expert * s["most"] + row - start, case["experts"] * s["most"])
        batch = x.new_zeros(case["experts"] * s["most"] + 1, x.shape[1]).index_copy_(0, place, x)
        out = torch.bmm(batch[:-1].view(case["experts"], s["most"], -1), w.transpose(1, 2)).flatten(0, 1)
        out = out[place.clamp(max=out.shape[0] - 1)]
        return {"out": torch.where(used[:, None], out, 0.0).to(DTYPES[case["dtype"]])}


def _clip_plain(s):
    case = s["case"]
    with torch.no_grad():
        g = s["flat"].float()
        norm = g.double().square_().sum().sqrt().float()
        coefficient = (case["max_norm"] / (norm + EPS)).clamp(max=1.0)
        if not case["in_place"]:
            return {"norm": norm, "coefficient": coefficient}
        s["flat"].copy_(g * coefficient)
        return {"norm": norm, "grads": s["flat"]}


# ---------------------------------------------------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------------------------------------------------

def _rms_own(s):
    from flashfusedmoe_b200 import rms_norm
    case = s["case"]
    options = dict(residual=s["residual"], weight_offset=case["offset"])
    if case["quantize"]:
        with torch.no_grad():
            out = rms_norm(s["x"], s["weight"], EPS, quantize=True, **options)
        return dict(zip(("values", "scale", "h"), out))
    if not case["backward"]:
        with torch.no_grad():
            out = rms_norm(s["x"], s["weight"], EPS, **options)
        return {"y": out} if s["residual"] is None else {"y": out[0], "h": out[1]}
    out = rms_norm(s["x"], s["weight"], EPS, **options)
    if s["residual"] is None:
        dx, dweight = torch.autograd.grad(out, [s["x"], s["weight"]], s["grad"])
        return {"y": out.detach(), "dx": dx, "dweight": dweight}
    dx, dresidual, dweight = torch.autograd.grad(out, [s["x"], s["residual"], s["weight"]], [s["grad"], s["grad_h"]])
    return {"y": out[0].detach(), "h": out[1].detach(), "dx": dx, "dresidual": dresidual, "dweight": dweight}


def _quantize_own(s):
    from flashfusedmoe_b200 import quantize_e4m3
    values, scale = quantize_e4m3(s["x"], s["case"]["block_rows"])
    return {"values": values, "scale": scale}


def _linear_own(s):
    from flashfusedmoe_b200 import linear_e4m3
    return {"out": linear_e4m3(s["x"], s["x_scale"], s["weight"], s["weight_scale"], ends=s["ends"],
                               out_dtype=DTYPES[s["case"]["dtype"]])}


def _clip_own(s):
    from flashfusedmoe_b200 import clip_coefficient, clip_grad_norm
    case = s["case"]
    if case["in_place"]:
        return {"norm": clip_grad_norm(s["params"], case["max_norm"]), "grads": s["flat"]}
    norm, coefficient = clip_coefficient(s["grads"], case["max_norm"])
    return {"norm": norm, "coefficient": coefficient}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"rms_norm": _rms_own, "quantize": _quantize_own, "linear": _linear_own, "clip": _clip_own}[op](state)
    if op == "quantize":
        values, scale = _quantize_plain(state["x"], state["case"]["block_rows"])
        return {"values": values, "scale": scale}
    return {"rms_norm": _rms_plain, "linear": _linear_plain, "clip": _clip_plain}[op](state)


# ---------------------------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "rms_norm":
        rows, dim = case["rows"], case["dim"]
        n, streams = rows * dim, 4 if case["residual"] else 2   # x (and the residual) in, y (and the sum) out
        if case["quantize"]:
            return {"bytes": n * (size * (streams - 1) + 1) + 4 * rows * math.ceil(dim / BLOCK) + dim * size, "flops": 8 * n}
        if case["backward"]:   # the gradients of the outputs in, and one out for both inputs; the weight's
            return {"bytes": n * size * (streams + (3 if case["residual"] else 2)) + 2 * dim * size, "flops": 16 * n}
        return {"bytes": n * size * streams + dim * size, "flops": 6 * n}
    if case["op"] == "quantize":
        n = case["matrices"] * case["rows"] * case["dim"]
        return {"bytes": n * (size + 1) + 4 * n / (BLOCK * case["block_rows"]), "flops": 3 * n}
    if case["op"] == "linear":
        rows, width, dim, experts = case["rows"], case["width"], case["dim"], case["experts"]
        # experts that some row falls on, were they spread evenly
        hit = experts * (1.0 - (1.0 - 1.0 / experts) ** rows) if experts else 1.0
        scales = 4.0 / BLOCK
        return {"bytes": rows * dim * (1 + scales) + hit * width * dim * (1 + scales / BLOCK) + (rows + case["spare"]) * width * size,
                "flops": 2 * rows * width * dim}
    n = sum(_elements(case))
    # in for the norm; clipping changes what was read, so in and out again
    return {"bytes": n * size * (3 if case["in_place"] else 1), "flops": (3 if case["in_place"] else 2) * n}


# ---------------------------------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------

def _scaled_exact(y, block_rows):
    """What the 8-bit numbers round, and their blocks' scales."""
    rows, dim = y.shape[-2:]
    scale = torch.nn.functional.max_pool2d(y.abs().view(-1, 1, rows, dim), (block_rows, BLOCK), ceil_mode=True)
    scale = torch.where(scale > 0, torch.clamp(scale / TOP, min=LEAST), torch.ones_like(scale))
    scale = scale.view(*y.shape[:-2], *scale.shape[-2:])
    down, across = (torch.arange(n, device=y.device) // b for n, b in ((rows, block_rows), (dim, BLOCK)))
    return y / scale[..., down, :][..., across], scale


def _rms_exact(s, case):
    h = s["x"].detach().double()
    out = {}
    if s["residual"] is not None:
        h = h + s["residual"].detach().double()
        out["h"] = h
        h = h.to(s["x"].dtype).double()   # the norm is that of the sum as it is handed on
    w = s["weight"].detach().double() + case["offset"]
    sigma = ((h * h).sum(dim=1, keepdim=True) / h.shape[1] + EPS).sqrt()
    xh = h / sigma
    if case["quantize"]:
        out["values"], out["scale"] = _scaled_exact(xh * w, 1)
        return out
    out["y"] = xh * w
    if case["backward"]:
        dy = s["grad"].double()
        inner = torch.einsum("rd,rd,d->r", dy, xh, w)[:, None] / h.shape[1]
        dx = (dy * w - xh * inner) / sigma
        if s["residual"] is not None:
            dx = dx + s["grad_h"].double()
            out["dresidual"] = dx
        out["dx"] = dx
        out["dweight"] = torch.einsum("rd,rd->d", dy, xh)
    return out


def _linear_exact(s, case):
    def wide(values, scale, block_rows):
        down, across = (torch.arange(n, device=values.device) // b for n, b in zip(values.shape, (block_rows, BLOCK)))
        return values.double() * scale.double()[down][:, across]

    if s["ends"] is None:
        return {"out": wide(s["x"], s["x_scale"], 1) @ wide(s["weight"], s["weight_scale"], 128).t()}
    out = torch.zeros(s["x"].shape[0], case["width"], dtype=torch.float64, device="cuda")
    begin = 0
    for e, end in enumerate(s["ends"].tolist()):
        x = wide(s["x"][begin:end], s["x_scale"][begin:end], 1)
        out[begin:end] = x @ wide(s["weight"][e], s["weight_scale"][e], 128).t()
        begin = end
    return {"out": out}


def _clip_exact(s, case):
    g = s["flat"].double()
    norm = torch.linalg.vector_norm(g)
    coefficient = torch.minimum(torch.ones_like(norm), case["max_norm"] / (norm + EPS))
    return {"norm": norm, "grads": g * coefficient} if case["in_place"] else {"norm": norm, "coefficient": coefficient}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "quantize":
            values, scale = _scaled_exact(s["x"].double(), case["block_rows"])
            return {"values": values, "scale": scale}
        return {"rms_norm": _rms_exact, "linear": _linear_exact, "clip": _clip_exact}[case["op"]](s, case)
