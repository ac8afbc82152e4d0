"""The operators a training step needs around the fused MoE layer, over the sizes they are used at: layer norm (forward and
backward), the linear cross entropy over a vocabulary (scoring and training) and the AdamW step over many tensors with states
in 32 or 8 bits.

A case is one call of a user's program. `run` computes it in plain torch operations, in 32 bits, or with `own` set through the
framework's kernels.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 128          # values that share a scale in an 8-bit state
IGNORE = -100
BETA1, BETA2, EPS, DECAY, RATE = 0.9, 0.95, 1e-8, 0.1, 3e-4


# ---------------------------------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------------------------------

def _norm(rows, dim, dtype="bf16", backward=True, bias=True):
    return dict(op="layer_norm", rows=rows, dim=dim, dtype=dtype, backward=backward, bias=bias, eps=1e-5)


def _loss(rows, dim, vocab, backward=True, ignored=0.0, z=0.0):
    return dict(op="linear_cross_entropy", rows=rows, dim=dim, vocab=vocab, backward=backward, ignored=ignored, z=z)


def _adamw(d_model, ffn_dim, experts, layers=1, dtype="bf16", bits=32, master=False):
    return dict(op="adamw", d_model=d_model, ffn_dim=ffn_dim, experts=experts, layers=layers, dtype=dtype, bits=bits,
                master=master)


def listed():
    def named(name, case):
        return dict(case, name=name)

    return [
        # the norm in front of the layer for one decoded token: nothing but latency
        named("norm_decode_1x4096", _norm(1, 4096, backward=False)),
        # the norm of the benchmark's training step
        named("norm_train_16384x1024", _norm(16384, 1024)),
        # a ragged micro-batch of fp16 rows of odd width: no 16-byte accesses
        named("norm_train_4093x2051_fp16", _norm(4093, 2051, dtype="fp16")),
        # a large micro-batch of wide rows: bandwidth alone
        named("norm_train_32768x7168", _norm(32768, 7168)),
        # log-probability of one decoded token under the benchmark model's vocabulary: the weights are streamed once
        named("loss_score_1x1024x50257", _loss(1, 1024, 50257, backward=False)),
        # a serving batch scored over a wider vocabulary
        named("loss_score_61x4096x100352", _loss(61, 4096, 100352, backward=False)),
        # a small training step with ignored (padding) targets and the z-loss
        named("loss_train_1999x2048x32003", _loss(1999, 2048, 32003, ignored=0.3, z=1e-4)),
        # a training step at the benchmark's width
        named("loss_train_16384x1024x50257", _loss(16384, 1024, 50257)),
        # a training step over a large vocabulary and wide rows: the largest amount of arithmetic
        named("loss_train_8192x4096x131072", _loss(8192, 4096, 131072)),
        # the gate and norm of a small layer in fp32: launches and latency
        named("adamw_small_fp32", _adamw(256, 128, 1, dtype="fp32")),
        # twelve layers of the benchmark's width, bf16 parameters with fp32 masters, 32-bit states, many tensors
        named("adamw_layers_master32", _adamw(1024, 2816, 4, layers=12, master=True)),
        # one wide layer in bf16 with 8-bit states: the largest, where the state's bytes are what counts
        named("adamw_wide_8bit", _adamw(4096, 14336, 4, bits=8)),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["layer_norm", "linear_cross_entropy", "adamw"])
    if op == "layer_norm":
        # rows from one token to a large micro-batch, widths of any value
        dim = log_int(64, 8192)
        if rng.random() < 0.5:
            dim = max(64, dim // 64 * 64)
        return _norm(log_int(1, 32768), dim, rng.choice(["bf16", "bf16", "fp16", "fp32"]) if dim <= 3500 else "bf16",
                     rng.random() < 0.7, rng.random() < 0.7)
    if op == "linear_cross_entropy":
        # widths are multiples of 8 (16-byte rows); vocabularies of any value
        dim = 8 * log_int(32, 512)
        if rng.random() < 0.3:
            return _loss(log_int(1, 256), dim, log_int(1000, 131072), backward=False)
        return _loss(log_int(16, 8192), dim, log_int(1000, 131072), True, rng.choice([0.0, 0.1, 0.5]),
                     rng.choice([0.0, 1e-4]))
    # odd widths put the tensors' ends at any place
    d = log_int(64, 2048)
    f = 2 * log_int(32, 2048)
    return _adamw(d, f, rng.randint(1, 8), rng.randint(1, 6), rng.choice(["bf16", "bf16", "fp32"]), rng.choice([32, 8]),
                  rng.random() < 0.4)


# ---------------------------------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------------------------------

def _sizes(case):
    """Elements of each tensor: per layer a norm's weight and bias, the gate, the experts' two projections."""
    d, f, e = case["d_model"], case["ffn_dim"], case["experts"]
    return [d, d, e * d, e * f * d, e * d * (f // 2)] * case["layers"]


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _prepare_norm(case, g):
    rows, dim, dtype = case["rows"], case["dim"], DTYPES[case["dtype"]]
    # activations of a residual stream: rows of different scale with a mean, a few channels that stand out
    scale = torch.rand(rows, 1, device="cuda", generator=g) * 2.0 + 0.5
    x = torch.randn(rows, dim, device="cuda", generator=g) * scale + 0.3
    x[:, :: max(1, dim // 8)] *= 5.0
    state = {"x": x.to(dtype), "weight": (1.0 + 0.2 * torch.randn(dim, device="cuda", generator=g)).to(dtype), "bias": None}
    if case["bias"]:
        state["bias"] = (0.2 * torch.randn(dim, device="cuda", generator=g)).to(dtype)
    if case["backward"]:
        state["grad"] = torch.randn(rows, dim, device="cuda", generator=g).to(dtype)
        for name in ("x", "weight", "bias"):
            if state[name] is not None:
                state[name].requires_grad_()
    return state


def _prepare_loss(case, g):
    rows, dim, vocab = case["rows"], case["dim"], case["vocab"]
    weight = torch.empty(vocab, dim, dtype=torch.bfloat16, device="cuda").normal_(0.0, dim ** -0.5, generator=g)
    target = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    # hidden rows of a model in training: some tokens are predicted well, some not at all
    sure = torch.rand(rows, 1, device="cuda", generator=g) * 14.0
    hidden = torch.randn(rows, dim, device="cuda", generator=g) + sure * weight[target].float()
    if case["ignored"] > 0.0:
        target = torch.where(torch.rand(rows, device="cuda", generator=g) < case["ignored"], IGNORE, target)
    state = {"hidden": hidden.bfloat16(), "weight": weight, "target": target}
    if case["backward"]:
        state["hidden"].requires_grad_()
        state["weight"].requires_grad_()
    return state


def _power(k):
    """2^k in fp32, exactly, for whole k from -126 to 127."""
    return ((k.to(torch.int32) + 127) << 23).view(torch.float32)


def _scaled(x, k):
    """The blocks of x times 2^k of each."""
    return (x.view(-1, BLOCK) * _power(k)[:, None]).view(-1)


def _prepare_adamw(case, g):
    """The tensors lie in flat buffers, each from a multiple of BLOCK on; what lies between them is zero and stays it."""
    dtype = DTYPES[case["dtype"]]
    sizes = _sizes(case)
    room = [(n + BLOCK - 1) // BLOCK * BLOCK for n in sizes]
    starts = [sum(room[:i]) for i in range(len(room))]
    total = sum(room)
    # gradients of very different size from tensor to tensor and row to row, as in training; their ends are padding
    scale = torch.exp(torch.randn(total // BLOCK, 1, device="cuda", generator=g) * 2.0 - 8.0)
    grad = (torch.randn(total // BLOCK, BLOCK, device="cuda", generator=g) * scale).view(-1)
    first = (torch.randn(total // BLOCK, BLOCK, device="cuda", generator=g) * scale * 0.3).view(-1)
    second = (grad * torch.rand(total, device="cuda", generator=g).add_(0.5)).square_()
    param = torch.randn(total, device="cuda", generator=g) * 0.02
    for start, n, r in zip(starts, sizes, room):
        for t in (grad, first, second, param):
            t[start + n:start + r] = 0.0
    state = {"starts": torch.tensor(starts, device="cuda"), "room": torch.tensor(room, device="cuda"), "seed": 12345,
             "steps": torch.full((len(sizes),), 9, dtype=torch.int32, device="cuda"), "param": param.to(dtype),
             "grad": grad.to(dtype), "master": param if case["master"] and dtype != torch.float32 else None}
    if case["bits"] == 8:
        for name, value in (("first", first), ("second", second.sqrt_())):
            top = value.view(-1, BLOCK).abs().amax(dim=1)
            mantissa, exponent = torch.frexp(top)
            exponent = torch.where(top > 0, exponent - 9 + (mantissa > 0.875).int(), -126).clamp(-126, 120)
            state[name] = _scaled(value, -exponent).to(torch.float8_e4m3fn)
            state[name + "_scale"] = (exponent + 127).to(torch.uint8)
    else:
        state["first"], state["second"] = first, second
    cut = lambda t: None if t is None else [t[s:s + n] for s, n in zip(starts, sizes)]  # noqa: E731
    state["lists"] = {name: cut(state[name]) for name in ("param", "grad", "first", "second", "master")}
    for name in ("first_scale", "second_scale"):
        t = state.get(name)
        state["lists"][name] = None if t is None else [t[s // BLOCK:(s + r) // BLOCK] for s, r in zip(starts, room)]
    state["lists"]["steps"] = list(state["steps"].unbind())
    return state


def prepare(case, seed):
    g = _generator(seed)
    state = {"layer_norm": _prepare_norm, "linear_cross_entropy": _prepare_loss, "adamw": _prepare_adamw}[case["op"]](case, g)
    state["case"] = case
    return state


# ---------------------------------------------------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------------------------------------------------

def _norm_plain(s):
    case = s["case"]
    with torch.no_grad():
        x, w = s["x"].float(), s["weight"].float()
        centred = x - x.mean(dim=1, keepdim=True)
        r = torch.rsqrt(centred.square().mean(dim=1, keepdim=True) + case["eps"])
        xh = centred * r
        y = xh * w
        if s["bias"] is not None:
            y = y + s["bias"].float()
        out = {"y": y.to(s["x"].dtype)}
        if case["backward"]:
            dy = s["grad"].float()
            g = dy * w
            dx = r * (g - g.mean(dim=1, keepdim=True) - xh * (g * xh).mean(dim=1, keepdim=True))
            out["dx"] = dx.to(s["x"].dtype)
            out["dweight"] = (dy * xh).sum(dim=0).to(s["weight"].dtype)
            if s["bias"] is not None:
                out["dbias"] = dy.sum(dim=0).to(s["bias"].dtype)
        return out


def _loss_plain(s):
    case = s["case"]
    with torch.no_grad():
        x, w, target = s["hidden"].float(), s["weight"].float(), s["target"]
        logits = x @ w.t()
        top = logits.amax(dim=1, keepdim=True)
        e = torch.exp(logits - top)
        total = e.sum(dim=1, keepdim=True)
        lse = (torch.log(total) + top)[:, 0]
        valid = target != IGNORE
        safe = torch.where(valid, target, 0)
        nll = lse - logits.gather(1, safe[:, None])[:, 0] + case["z"] * lse.square()
        nll = torch.where(valid, nll, 0.0)
        if not case["backward"]:
            return {"nll": nll}
        share = valid.float() / valid.sum().float()
        d = e / total * (1.0 + 2.0 * case["z"] * lse)[:, None]
        d[torch.arange(target.numel(), device=target.device), safe] -= 1.0
        d *= share[:, None]
        return {"loss": nll.double().mul(share).sum().float(), "dhidden": (d @ w).bfloat16(), "dweight": (d.t() @ x).bfloat16()}


def _random16(index, key):
    """Sixteen random bits per element, as a number between 0 and 1: the low and the high half of a 32-bit hash of a counter of
    pairs."""
    h = ((index >> 1) * 0x9E3779B1 + key) & 0xFFFFFFFF
    h = ((h ^ (h >> 16)) * 0x85EBCA6B) & 0xFFFFFFFF
    h = ((h ^ (h >> 13)) * 0xC2B2AE35) & 0xFFFFFFFF
    h = h ^ (h >> 16)
    return (((h >> 16 * (index & 1)) & 0xFFFF).float() + 0.5) * (1.0 / 65536.0)


def _block_exponent(x):
    """The least k for which no magnitude of the block is over 448 * 2^k (448 = 0.875 * 2^9 is e4m3's largest)."""
    top = x.view(-1, BLOCK).abs().amax(dim=1)
    mantissa, exponent = torch.frexp(top)
    return torch.where(top > 0, exponent - 9 + (mantissa > 0.875).int(), -126).clamp(-126, 120)


def _adamw_plain(s):
    case, eight = s["case"], s["case"]["bits"] == 8
    with torch.no_grad():
        s["steps"].add_(1)
        t = s["steps"].double().repeat_interleave(s["room"])
        rate = (RATE / (1.0 - BETA1 ** t)).float()
        inverse = (1.0 / (1.0 - BETA2 ** t).sqrt()).float()
        g = s["grad"].float()
        m, v = s["first"], s["second"]
        if eight:
            km, kv = (s[n].to(torch.int32) - 127 for n in ("first_scale", "second_scale"))
            m, v = _scaled(m.float(), km), _scaled(v.float(), kv).square()
        m = m * BETA1 + g * (1.0 - BETA1)
        v = v * BETA2 + (g * (1.0 - BETA2)) * g
        p = (s["param"] if s["master"] is None else s["master"]).float()
        root = v.sqrt()
        p = p * (1.0 - RATE * DECAY) - rate * (m / (root * inverse + EPS))
        s["param"].copy_(p)
        if s["master"] is not None:
            s["master"].copy_(p)
        if not eight:
            s["first"].copy_(m)
            s["second"].copy_(v)
            out = {"exp_avg": s["first"], "exp_avg_sq": s["second"]}
        else:
            km, kv = _block_exponent(m), _block_exponent(root)
            s["first"].copy_(_scaled(m, -km).to(torch.float8_e4m3fn))
            x = _scaled(root, -kv)
            index = torch.arange(x.numel(), device=x.device) - s["starts"].repeat_interleave(s["room"])
            key = (s["steps"].long() * 0x85EBCA77 + s["seed"] * 0xC2B2AE3D).repeat_interleave(s["room"]) & 0xFFFFFFFF
            step = _power(torch.frexp(x)[1].sub(1).clamp(min=-6).sub(3))
            code = torch.floor(x / step + _random16(index, key)) * step
            code = torch.where(x > 0, code.clamp(min=2.0 ** -9), 0.0)
            s["second"].copy_(code.to(torch.float8_e4m3fn))
            s["first_scale"].copy_(km + 127)
            s["second_scale"].copy_(kv + 127)
            out = _adamw_states(s)
        return _adamw_outputs(s, out)


def _adamw_states(s):
    """8-bit states as the values they stand for: e4m3 numbers and the blocks' powers of two."""
    scales = {n: _power(s[k].int() - 127) for n, k in (("exp_avg_scale", "first_scale"), ("exp_avg_sq_scale", "second_scale"))}
    return {"exp_avg": s["first"], "exp_avg_sq": s["second"], **scales}


def _adamw_outputs(s, out):
    out = dict(out, param=s["param"], steps=s["steps"])
    if s["master"] is not None:
        out["master"] = s["master"]
    return out


# ---------------------------------------------------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------------------------------------------------

def _norm_own(s):
    from flashfusedmoe_b200 import layer_norm
    case = s["case"]
    if not case["backward"]:
        with torch.no_grad():
            return {"y": layer_norm(s["x"], s["weight"], s["bias"], case["eps"])}
    s["x"].grad = s["weight"].grad = None
    y = layer_norm(s["x"], s["weight"], s["bias"], case["eps"])
    if s["bias"] is not None:
        s["bias"].grad = None
    y.backward(s["grad"])
    out = {"y": y.detach(), "dx": s["x"].grad, "dweight": s["weight"].grad}
    if s["bias"] is not None:
        out["dbias"] = s["bias"].grad
    return out


def _loss_own(s):
    from flashfusedmoe_b200 import linear_cross_entropy
    case = s["case"]
    if not case["backward"]:
        with torch.no_grad():
            return {"nll": linear_cross_entropy(s["hidden"], s["weight"], s["target"], ignore_index=IGNORE, reduction="none",
                                                z_loss_coeff=case["z"])}
    s["hidden"].grad = s["weight"].grad = None
    loss = linear_cross_entropy(s["hidden"], s["weight"], s["target"], ignore_index=IGNORE, z_loss_coeff=case["z"])
    loss.backward()
    return {"loss": loss.detach(), "dhidden": s["hidden"].grad, "dweight": s["weight"].grad}


def _adamw_own(s):
    from flashfusedmoe_b200 import adamw_step
    lists = s["lists"]
    adamw_step(lists["param"], lists["grad"], lists["first"], lists["second"], lists["steps"], lr=RATE, betas=(BETA1, BETA2),
               eps=EPS, weight_decay=DECAY, masters=lists["master"], exp_avg_scales=lists["first_scale"],
               exp_avg_sq_scales=lists["second_scale"], seed=s["seed"])
    if s["case"]["bits"] == 8:
        return _adamw_outputs(s, _adamw_states(s))
    return _adamw_outputs(s, {"exp_avg": s["first"], "exp_avg_sq": s["second"]})


def run(state):
    op = state["case"]["op"]
    if own:
        return {"layer_norm": _norm_own, "linear_cross_entropy": _loss_own, "adamw": _adamw_own}[op](state)
    return {"layer_norm": _norm_plain, "linear_cross_entropy": _loss_plain, "adamw": _adamw_plain}[op](state)


# ---------------------------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------

def work(case):
    if case["op"] == "layer_norm":
        n = case["rows"] * case["dim"]
        size = 4 if case["dtype"] == "fp32" else 2
        vectors = (2 if case["bias"] else 1) * case["dim"] * size
        # x in, y out; with gradients dy in and dx out too, and a gradient for every vector
        if case["backward"]:
            return {"bytes": 4 * n * size + 2 * vectors, "flops": 20 * n}
        return {"bytes": 2 * n * size + vectors, "flops": 8 * n}
    if case["op"] == "linear_cross_entropy":
        rows, dim, vocab = case["rows"], case["dim"], case["vocab"]
        product = 2 * rows * dim * vocab
        operands = 2 * (rows + vocab) * dim
        if case["backward"]:  # logits, and their gradient against either operand
            return {"bytes": 2 * operands + 8 * rows, "flops": 3 * product}
        return {"bytes": operands + 12 * rows, "flops": product}
    n = sum(_sizes(case))
    size = 4 if case["dtype"] == "fp32" else 2
    # parameter and both states in and out, gradient in; with a master its 4 bytes are read in the parameter's place
    states = 16 if case["bits"] == 32 else 4 + 4 / BLOCK
    param = 2 * size if not (case["master"] and size == 2) else 8 + size
    return {"bytes": n * (param + size + states), "flops": 16 * n}


# ---------------------------------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------

def _norm_exact(s, case):
    x, w = s["x"].detach().double(), s["weight"].detach().double()
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    sigma = (var + case["eps"]).sqrt()
    b = 0.0 if s["bias"] is None else s["bias"].detach().double()
    out = {"y": (x - mean) / sigma * w + b}
    if case["backward"]:
        dy = s["grad"].double()
        xh = (x - mean) / sigma
        n = x.shape[1]
        inner = torch.einsum("rd,rd,d->r", dy, xh, w)[:, None]
        total = (dy @ w)[:, None]
        out["dx"] = (dy * w - (total + xh * inner) / n) / sigma
        out["dweight"] = torch.einsum("rd,rd->d", dy, xh)
        if s["bias"] is not None:
            out["dbias"] = dy.sum(dim=0)
    return out


def _loss_exact(s, case):
    h, w, target = s["hidden"].detach().double(), s["weight"].detach().double(), s["target"]
    valid = target.ne(IGNORE)
    rows = valid.nonzero()[:, 0]
    logits = torch.mm(h[rows], w.t())
    lse = torch.logsumexp(logits, dim=1)
    value = lse - logits[torch.arange(rows.numel(), device=rows.device), target[rows]] + case["z"] * lse * lse
    if not case["backward"]:
        return {"nll": torch.zeros(target.numel(), dtype=torch.float64, device=h.device).index_copy_(0, rows, value)}
    d = torch.exp(logits - lse[:, None])
    d.mul_(1.0 + 2.0 * case["z"] * lse[:, None])
    d.scatter_add_(1, target[rows][:, None], torch.full_like(d[:, :1], -1.0))
    d.div_(rows.numel())
    dh = torch.zeros_like(h).index_copy_(0, rows, torch.mm(d, w))
    return {"loss": value.mean(), "dhidden": dh, "dweight": torch.mm(d.t(), h[rows])}


def _adamw_exact(s, case):
    eight = case["bits"] == 8

    def value(name):
        x = s[name].double()
        return x if not eight else (x.view(-1, BLOCK) * torch.pow(2.0, s[name + "_scale"].double() - 127.0)[:, None]).view(-1)

    t = (s["steps"].double() + 1.0).repeat_interleave(s["room"])
    g = s["grad"].double()
    m = value("first").lerp_(g, 1.0 - BETA1)
    v = value("second")
    v = torch.addcmul((v * v if eight else v).mul_(BETA2), g, g, value=1.0 - BETA2)
    m_hat, v_hat = m / (1.0 - torch.pow(BETA1, t)), v / (1.0 - torch.pow(BETA2, t))
    p = s["param" if s["master"] is None else "master"].double()
    p = p - RATE * DECAY * p - RATE * m_hat / (v_hat.sqrt() + EPS)
    out = {"param": p, "steps": s["steps"] + 1, "exp_avg": None, "exp_avg_sq": None}
    if s["master"] is not None:
        out["master"] = p
    if not eight:
        out.update(exp_avg=m, exp_avg_sq=v)
        return out
    # e4m3 values: multiples of 2^(e-3) in the binade of 2^e, and of 2^-9 below 2^-6
    for name, x in (("exp_avg", m), ("exp_avg_sq", v.sqrt())):
        x = x.view(-1, BLOCK)
        scale = torch.pow(2.0, torch.ceil(torch.log2(x.abs().amax(dim=1, keepdim=True).clamp(min=1e-300) / 448.0)))
        scale = scale.clamp(min=2.0 ** -126)
        x = x / scale
        grid = torch.pow(2.0, torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3.0)
        if name == "exp_avg":
            x = torch.round(x / grid) * grid
        else:
            index = torch.cat([torch.arange(int(n), device=x.device) for n in s["room"].tolist()])
            step = (s["steps"].long() + 1).repeat_interleave(s["room"])
            key = (step * 0x85EBCA77 + s["seed"] * 0xC2B2AE3D) % 2 ** 32
            h = (index // 2 * 0x9E3779B1 + key) % 2 ** 32
            h = (h ^ (h // 2 ** 16)) * 0x85EBCA6B % 2 ** 32
            h = (h ^ (h // 2 ** 13)) * 0xC2B2AE35 % 2 ** 32
            h = h ^ (h // 2 ** 16)
            u = (torch.where(index % 2 == 1, h // 2 ** 16, h % 2 ** 16).double() + 0.5) / 2 ** 16
            x = torch.where(x > 0, (torch.floor(x / grid + u.view_as(x)) * grid).clamp(min=2.0 ** -9), x)
        out[name], out[name + "_scale"] = x.reshape(-1), None  # a power of two has no rounding to speak of
    return out


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"layer_norm": _norm_exact, "linear_cross_entropy": _loss_exact, "adamw": _adamw_exact}[case["op"]](state, case)
