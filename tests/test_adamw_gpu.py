"""AdamW over many tensors against a 64-bit evaluation, states in 32 and 8 bits.

Bounds, with u = 2^-24: m and v are two rounded products and a rounded sum (v: one product more), 4 u of the terms. The update
is off by 32 u of itself (constants rounded to fp32, root, quotient) and the parameter by 4 u more of itself, and then half a
unit of its type. In 8 bits m is rounded to the nearest e4m3 number (half a step: 2^-4 of it, or 2^-10 of the scale), sqrt(v)
to one of its two neighbours (a whole step: 2^-3 of it, or 2^-9 of the scale)."""

import pytest
import torch

U = 2.0 ** -24
BLOCK = 128
# around a thread's eight, a scale's block, a block's chunk of 2048; several chunks
SIZES = [1, 7, 8, 127, 128, 129, 1000, 2047, 2048, 2049, 4096, 4097, 5003, 8192, 70001]
HYPER = dict(lr=3e-3, betas=(0.9, 0.97), eps=1e-6, weight_decay=0.1)


def decode(codes, scale, root=False):
    n = codes.numel()
    s = torch.pow(2.0, scale.double() - 127).repeat_interleave(BLOCK)[:n]
    x = codes.reshape(-1).double() * s
    return (x * x if root else x).view(codes.shape)


class Tensors:
    def __init__(self, sizes, dtype, bits, master=False, grad_dtype=None, shift=0, seed=0, step=3):
        gen = torch.Generator(device="cuda").manual_seed(seed)

        def normal(n, std, kind):
            room = torch.randn(n + shift, device="cuda", generator=gen) * std
            return room.to(kind)[shift:]

        self.params = [normal(n, 0.5, dtype) for n in sizes]
        self.grads = [normal(n, 10.0 ** -(i % 5), grad_dtype or dtype) for i, n in enumerate(sizes)]
        self.steps = [torch.tensor(step + i % 2, dtype=torch.int32, device="cuda") for i in range(len(sizes))]
        self.masters = [p.float() + normal(n, 1e-4, torch.float32) for p, n in zip(self.params, sizes)] if master else None
        self.m = [g.float() * 0.5 + normal(n, 1e-3, torch.float32) for g, n in zip(self.grads, sizes)]
        self.v = [g.float().square() + normal(n, 1e-3, torch.float32).square() for g, n in zip(self.grads, sizes)]
        if shift:
            self.m, self.v = ([torch.cat([t.new_zeros(shift), t])[shift:] for t in ts] for ts in (self.m, self.v))
        self.m_scale = self.v_scale = None
        if bits == 8:
            self.m_scale, self.v_scale, states = [], [], ([], [])
            for x, y in zip(self.m, self.v):
                for values, scales, into in ((x, self.m_scale, states[0]), (y.sqrt(), self.v_scale, states[1])):
                    n = values.numel()
                    blocks = torch.cat([values, values.new_zeros(-n % BLOCK)]).view(-1, BLOCK)
                    k = torch.ceil(torch.log2(blocks.abs().amax(1).clamp(min=1e-30) / 448)).int()
                    scales.append((k + 127).to(torch.uint8))
                    codes = torch.ldexp(blocks, -k[:, None]).to(torch.float8_e4m3fn).view(-1)[:n].view(torch.uint8)
                    into.append(torch.cat([codes.new_zeros(shift), codes])[shift:].view(torch.float8_e4m3fn))
            self.m, self.v = states

    def exact(self, grad_scale=1.0, **h):
        """(m, v, p, bounds of each) per tensor, in 64 bits, from the state as it is."""
        h = {**HYPER, **h}
        b1, b2 = h["betas"]
        found = []
        for i, p in enumerate(self.params):
            m, v = (self.m[i].double(), self.v[i].double()) if self.m_scale is None else \
                (decode(self.m[i], self.m_scale[i]), decode(self.v[i], self.v_scale[i], root=True))
            g = self.grads[i].double() * grad_scale
            t = self.steps[i].item() + 1
            m_off, v_off = 4 * U * (b1 * m.abs() + (1 - b1) * g.abs()), 4 * U * (b2 * v + (1 - b2) * g * g)
            m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
            denominator = (v / (1 - b2 ** t)).sqrt() + h["eps"]
            update = h["lr"] / (1 - b1 ** t) * m / denominator
            old = (p if self.masters is None else self.masters[i]).double()
            new = old * (1 - h["lr"] * h["weight_decay"]) - update
            p_off = 32 * U * update.abs() + h["lr"] / (1 - b1 ** t) * m_off / denominator + 4 * U * (old.abs() + new.abs())
            found.append((m, v, new, m_off, v_off, p_off))
        return found

    def step(self, **h):
        from flashfusedmoe_b200 import adamw_step
        adamw_step(self.params, self.grads, self.m, self.v, self.steps, masters=self.masters, exp_avg_scales=self.m_scale,
                   exp_avg_sq_scales=self.v_scale, **{**HYPER, **h})

    def check(self, found, before):
        for i, (m, v, p, m_off, v_off, p_off) in enumerate(found):
            assert self.steps[i].item() == before[i] + 1
            if self.masters is not None:
                assert ((self.masters[i].double() - p).abs() <= p_off).all()
                assert torch.equal(self.params[i], self.masters[i].to(self.params[i].dtype))
            half = torch.finfo(self.params[i].dtype).eps / 2
            assert ((self.params[i].double() - p).abs() <= p_off * (1 + half) + half * p.abs() + 2.0 ** -25).all()
            if self.m_scale is None:
                assert ((self.m[i].double() - m).abs() <= m_off).all() and ((self.v[i].double() - v).abs() <= v_off).all()
                continue
            for exact, off, codes, scale, step in ((m, m_off, self.m[i], self.m_scale[i], 2.0 ** -4),
                                                   (v.sqrt(), v_off.sqrt() * 0 + 4 * U * v.sqrt(), self.v[i], self.v_scale[i], 2.0 ** -3)):
                n = exact.numel()
                s = torch.pow(2.0, scale.double() - 127)
                top = torch.cat([exact.abs(), exact.new_zeros(-n % BLOCK)]).view(-1, BLOCK).amax(1)
                # the least power of two for which the largest fits, up to its own rounding
                assert (top <= 448 * s * (1 + 8 * U)).all() and (top >= 224 * s * (1 - 8 * U)).all()
                s = s.repeat_interleave(BLOCK)[:n]
                got = decode(codes, scale)
                assert ((got - exact).abs() <= off + torch.maximum(step * exact.abs() * (1 + 4 * U), s * 2.0 ** -6 * step)).all()
            assert (decode(self.v[i], self.v_scale[i])[v > 0] > 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,grad_dtype,master", [(torch.bfloat16, None, False), (torch.bfloat16, None, True), (torch.float32, None, False),
                                                     (torch.float16, None, False), (torch.float16, None, True), (torch.float16, torch.float32, True),
                                                     (torch.float32, torch.bfloat16, False), (torch.bfloat16, torch.float16, False)])
@pytest.mark.parametrize("shift", [0, 1])
def test_a_step_over_tensors_of_every_size(bits, dtype, grad_dtype, master, shift):
    t = Tensors(SIZES, dtype, bits, master, grad_dtype, shift)
    before = [s.item() for s in t.steps]
    found = t.exact()
    t.step()
    t.check(found, before)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [0, 1, 32, 33, 256, 257, 600])
def test_any_number_of_tensors(count, bits):
    t = Tensors([5 + 37 * i % 300 for i in range(count)], torch.bfloat16, bits)
    if count > 40:
        for name in ("params", "grads", "m", "v"):
            getattr(t, name)[37] = getattr(t, name)[37][:0]
        if bits == 8:
            t.m_scale[37], t.v_scale[37] = t.m_scale[37][:0], t.v_scale[37][:0]
    before = [s.item() for s in t.steps]
    found = t.exact()
    t.step()
    t.check([f for i, f in enumerate(found) if True] if count <= 40 else found[:37], before)
    assert [s.item() for s in t.steps] == [b + 1 for b in before]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_of_different_types_in_one_call(bits):
    parts = [Tensors([300, 9000], dtype, bits, False, grad, seed=k) for k, (dtype, grad) in enumerate(
        [(torch.bfloat16, None), (torch.float32, None), (torch.float16, None), (torch.float32, torch.bfloat16), (torch.bfloat16, None)])]
    t = Tensors([], torch.float32, bits)
    for name in ("params", "grads", "steps", "m", "v") + (("m_scale", "v_scale") if bits == 8 else ()):
        setattr(t, name, [x for p in parts for x in getattr(p, name)])
    before = [s.item() for s in t.steps]
    found = t.exact()
    t.step()
    t.check(found, before)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [0.0, 1e-20])
def test_tiny_gradients_and_eps(bits, eps):
    """v around and below the smallest normal number; the quotient of two small numbers is still about 1. In 8 bits no positive v is
    lost. v itself is fp32: 2^-149 off (a whole of it where nothing is left)."""
    t = Tensors([5000], torch.float32, bits)
    t.grads[0].copy_(torch.logspace(-24, -16, 5000, device="cuda"))
    t.m[0].view(torch.uint8).zero_()
    t.v[0].view(torch.uint8).zero_()
    m, v, p, _, _, p_off = t.exact(eps=eps)[0]
    t.step(eps=eps)
    normal = v > 2.0 ** -126
    assert ((t.params[0].double() - p).abs() <= p_off)[normal].all() and t.params[0].isfinite()[v > 2.0 ** -148].all()
    if bits == 8:
        root, got = v.sqrt(), decode(t.v[0], t.v_scale[0])
        assert (got[normal] > 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_device_scalars_and_a_first_step(bits):
    t = Tensors([300, 4000], torch.float32, bits, step=0)
    for s in t.steps:
        s.zero_()
    found = t.exact(grad_scale=0.25, lr=1.0 / 64)
    t.step(lr=torch.tensor(1.0 / 64, device="cuda"), grad_scale=torch.tensor([0.25], device="cuda"))
    t.check(found, [0, 0])


@pytest.mark.gpu
def test_rounding_of_the_second_moment_is_even_handed():
    """Up and down in proportion: the mean of the rounded roots is off by at most 5 standard errors (half a step's each), and by
    half of the random fraction's last place. Other seeds and steps draw other numbers; the same draws the same."""
    n = 1 << 20
    drawn = []
    for seed, step in ((1, 5), (1, 5), (2, 5), (1, 6)):
        t = Tensors([n], torch.float32, 8, step=step)
        t.grads[0].fill_(1.0)
        t.m[0].view(torch.uint8).zero_()
        t.v[0].view(torch.uint8).zero_()
        t.grads[0][::2] = torch.linspace(0.001, 1.0, n // 2, device="cuda")
        _, v, *_ = t.exact()[0]
        t.step(seed=seed)
        got, root = decode(t.v[0], t.v_scale[0]), v.sqrt()
        s = torch.pow(2.0, t.v_scale[0].double() - 127).repeat_interleave(BLOCK)
        step_size = torch.maximum(root / 8, s * 2.0 ** -9)
        error = (got - root) / step_size
        assert abs(error.mean().item()) <= 5 * 0.5 / n ** 0.5 + 2.0 ** -16
        drawn.append(got)
    assert torch.equal(drawn[0], drawn[1]) and not torch.equal(drawn[0], drawn[2]) and not torch.equal(drawn[0], drawn[3])


@pytest.mark.gpu
def test_codes_do_not_depend_on_how_the_root_was_taken():
    """The states do not depend on eps, so a call whose eps wants exact roots and quotients stores the codes of one whose eps does
    not. One value in 2^20 lies where a root one unit off gives another code: 32 or so of these 2^25 at either step."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    n = 1 << 25
    grad = torch.randn(n, device="cuda", generator=gen).mul_(1e-3)
    one, other = ([torch.zeros(n, device="cuda")] + [torch.zeros(n, device="cuda", dtype=torch.float8_e4m3fn) for _ in range(2)]
                  + [torch.full((n // BLOCK,), 1, dtype=torch.uint8, device="cuda") for _ in range(2)]
                  + [torch.zeros((), dtype=torch.int32, device="cuda")] for _ in range(2))
    from flashfusedmoe_b200 import adamw_step
    for _ in range(2):
        for (p, m, v, ms, vs, step), eps in ((one, 1e-6), (other, 1e-30)):
            adamw_step([p], [grad], [m], [v], [step], exp_avg_scales=[ms], exp_avg_sq_scales=[vs], **{**HYPER, "eps": eps})
        for x, y in zip(one[1:5], other[1:5]):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.gpu
def test_a_small_average_keeps_moving_in_8_bits():
    """Gradients fall to nothing: v = b2^t v then, 2 % of sqrt(v) a step, far less than the distance of two e4m3 numbers."""
    from flashfusedmoe_b200 import adamw_step
    n = 1 << 16
    p, g = torch.zeros(n, device="cuda"), torch.full((n,), 1e-3, device="cuda")
    m, v = (torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
    ms, vs = (torch.zeros(n // BLOCK, dtype=torch.uint8, device="cuda") for _ in range(2))
    step = torch.zeros((), dtype=torch.int32, device="cuda")
    exact = 0.0
    for k in range(60):
        if k == 1:
            g.zero_()
        adamw_step([p], [g], [m], [v], [step], lr=0.0, betas=(0.9, 0.96), exp_avg_scales=[ms], exp_avg_sq_scales=[vs], seed=3)
        exact = 0.96 * exact + (0.04 * 1e-6 if k == 0 else 0.0)
    # the mean root follows (its rounding is even-handed); squaring adds the spread, 60 draws of at most half a step each
    assert decode(v, vs).mean().item() == pytest.approx(exact ** 0.5, rel=0.05)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_values_that_are_not_finite_stay_where_they_are(bits):
    t = Tensors([1000], torch.float32, bits)
    t.grads[0][5] = float("nan")
    t.grads[0][300] = float("inf")
    before = [s.item() for s in t.steps]
    found = t.exact()
    t.step()
    bad = [5, 300]
    assert t.params[0][bad].isnan().all() and not t.params[0].isnan().sum() > 2
    m = t.m[0].double() if bits == 32 else decode(t.m[0], t.m_scale[0])
    assert m.isfinite().sum() == 1000 - len(bad) if bits == 32 else m[5].isnan() and m[300].isnan()
    rest = torch.ones(1000, dtype=torch.bool, device="cuda")
    rest[0:128] = rest[256:384] = False   # the scales of these blocks are those of infinity
    _, _, p, _, _, off = found[0]
    assert ((t.params[0].double() - p).abs() <= off)[rest].all() and t.steps[0].item() == before[0] + 1


@pytest.mark.gpu
def test_zero_gradients_and_states_change_nothing_but_the_decay():
    for bits in (32, 8):
        t = Tensors([513], torch.float32, bits)
        t.grads[0].zero_()
        (t.m[0] if bits == 32 else t.m[0].view(torch.uint8)).zero_()
        (t.v[0] if bits == 32 else t.v[0].view(torch.uint8)).zero_()
        old = t.params[0].clone()
        t.step(weight_decay=0.0)
        assert torch.equal(t.params[0], old) and not t.m[0].float().any() and not t.v[0].float().any()


def _models(dtype, **options):
    from flashfusedmoe_b200 import AdamW
    torch.manual_seed(1)
    shapes = [(64, 128), (128,), (3, 50, 70), (1,)]
    params = [torch.nn.Parameter(torch.randn(s, device="cuda").to(dtype)) for s in shapes]
    groups = [{"params": params[:2], "weight_decay": 0.1}, {"params": params[2:], "lr": 2e-3}]
    return params, AdamW(groups, lr=1e-3, betas=(0.9, 0.95), weight_decay=0.0, **options)


@pytest.mark.gpu
def test_optimizer_follows_torch_in_32_bits():
    """Twenty steps beside torch.optim.AdamW in fp64 on the same gradients: each step adds at most 40 u of an update and 4 u of
    the parameter."""
    params, opt = _models(torch.float32)
    twins = [torch.nn.Parameter(p.detach().double()) for p in params]
    other = torch.optim.AdamW([{"params": twins[:2], "weight_decay": 0.1}, {"params": twins[2:], "lr": 2e-3}], lr=1e-3,
                              betas=(0.9, 0.95), weight_decay=0.0)
    for k in range(20):
        for p, q in zip(params, twins):
            p.grad = torch.randn_like(p)
            q.grad = p.grad.double()
        if k == 7:
            params[1].grad = twins[1].grad = None   # a parameter without a gradient keeps its step
        opt.step()
        other.step()
    for p, q in zip(params, twins):
        limit = 20 * (40 * U * 2e-3 * 5 + 4 * U * (q.detach().abs() + 0.1))
        assert ((p.double() - q).abs() <= limit).all()
    assert opt.state[params[1]]["step"].item() == 19 and opt.state[params[0]]["step"].item() == 20


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,options", [(torch.float32, {}), (torch.bfloat16, {}), (torch.bfloat16, {"master_weights": False}),
                                           (torch.bfloat16, {"state_bits": 8, "min_8bit_size": 1000})])
def test_state_dict_resumes_bit_for_bit(dtype, options):
    def drive(params, opt, lo, hi):
        for k in range(lo, hi):
            gen = torch.Generator(device="cuda").manual_seed(k)
            for p in params:
                p.grad = torch.randn(p.shape, device="cuda", generator=gen).to(dtype)
            opt.step()

    params, opt = _models(dtype, **options)
    drive(params, opt, 0, 5)
    saved = [p.detach().clone() for p in params], opt.state_dict()
    saved = (saved[0], {"state": {i: {k: v.clone() for k, v in s.items()} for i, s in saved[1]["state"].items()},
                        "param_groups": saved[1]["param_groups"]})
    drive(params, opt, 5, 9)
    again, resumed = _models(dtype, **options)
    with torch.no_grad():
        for p, q in zip(again, saved[0]):
            p.copy_(q)
    resumed.load_state_dict(saved[1])
    for p in again:
        for name, value in resumed.state[p].items():
            assert value.dtype == opt.state[params[[q is p for q in again].index(True)]][name].dtype, name
    drive(again, resumed, 5, 9)
    assert all(torch.equal(p, q) for p, q in zip(params, again))
    eight = options.get("state_bits") == 8
    assert ("exp_avg_scale" in opt.state[params[0]]) == eight and "exp_avg_scale" not in opt.state[params[1]]
    assert ("master" in opt.state[params[0]]) == (dtype != torch.float32 and options.get("master_weights", True))


@pytest.mark.gpu
def test_a_state_dict_of_torchs_optimizer_goes_on():
    """Five steps with torch.optim.AdamW, then ten with either; the bound is that of twenty steps above."""
    params, opt = _models(torch.float32)
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    other = torch.optim.AdamW([{"params": twins[:2], "weight_decay": 0.1}, {"params": twins[2:], "lr": 2e-3}], lr=1e-3,
                              betas=(0.9, 0.95), weight_decay=0.0)

    def gradients(k):
        gen = torch.Generator(device="cuda").manual_seed(k)
        for p, q in zip(params, twins):
            q.grad = torch.randn(q.shape, device="cuda", generator=gen)
            p.grad = q.grad.clone()

    for k in range(5):
        gradients(k)
        other.step()
    with torch.no_grad():
        for p, q in zip(params, twins):
            p.copy_(q)
    opt.load_state_dict(other.state_dict())
    assert all(opt.state[p]["step"].dtype == torch.int32 and opt.state[p]["step"].item() == 5 for p in params)
    for k in range(5, 15):
        gradients(k)
        opt.step()
        other.step()
    for p, q in zip(params, twins):
        assert ((p - q).abs() <= 2 * 20 * (40 * U * 2e-3 * 5 + 4 * U * (q.detach().abs() + 0.1))).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_replay_to_the_eager_bits(bits):
    """Two graphs of one optimizer, replayed in turn, with the rate read from the device."""
    def make():
        params, opt = _models(torch.bfloat16, state_bits=bits, min_8bit_size=1000)
        lr = torch.tensor(1e-3, device="cuda")
        for g in opt.param_groups:
            g["lr"] = lr
        for p in params:
            p.grad = torch.ones_like(p)
        opt.step()
        return params, opt, lr

    params, opt, lr = make()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            opt.step()
        graphs.append(g)
    twins, eager, rate = make()
    for k in range(6):
        for p, q in zip(params, twins):
            p.grad.copy_(torch.randn_like(p))
            q.grad.copy_(p.grad)
        lr.fill_(1e-3 / (k + 1))
        rate.copy_(lr)
        graphs[k % 2].replay()
        eager.step()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(params, twins))
    assert all(opt.state[p]["step"].item() == 7 for p in params)


@pytest.mark.gpu
def test_the_first_step_of_a_parameter_is_not_captured():
    params, opt = _models(torch.float32)
    for p in params:
        p.grad = torch.ones_like(p)
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="cannot be captured"):
        with torch.cuda.graph(g):
            opt.step()


@pytest.mark.gpu
def test_calls_on_two_streams_at_once():
    streams = [torch.cuda.Stream() for _ in range(2)]
    jobs = [[Tensors([300000, 777], torch.bfloat16, 8, seed=s) for s in (1, 2)] for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for stream, t in zip(streams, jobs[0]):
            with torch.cuda.stream(stream):
                t.step()
    torch.cuda.synchronize()
    for t in jobs[1]:
        for _ in range(5):
            t.step()
    for a, b in zip(*jobs):
        assert all(torch.equal(p, q) for p, q in zip(a.params, b.params))
        assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(a.v, b.v))


@pytest.mark.gpu
def test_a_step_is_seen_by_whoever_watches_versions():
    t = Tensors([100], torch.float32, 32)
    leaf = t.params[0].requires_grad_()
    loss = (leaf * leaf).sum()
    version = leaf._version
    t.step()
    assert leaf._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.gpu
def test_refusals():
    from flashfusedmoe_b200 import adamw_step

    def refused(error, match, change, bits=32, **h):
        t = Tensors([100, 200], torch.float32, bits, master=False)
        change(t)
        old = [p.clone() for p in t.params]
        with pytest.raises(error, match=match):
            t.step(**h)
        torch.cuda.synchronize()
        assert all(torch.equal(p.cpu(), q.cpu()) for p, q in zip(t.params, old))

    refused(ValueError, "one tensor for each", lambda t: t.grads.pop())
    refused(ValueError, "twice", lambda t: (t.params.__setitem__(1, t.params[0]), t.grads.__setitem__(1, t.grads[0]),
                                            t.m.__setitem__(1, t.m[1][:100]), t.v.__setitem__(1, t.v[1][:100])))
    refused(ValueError, "twice", lambda t: t.steps.__setitem__(1, t.steps[0]))
    refused(ValueError, "shape", lambda t: t.grads.__setitem__(0, t.grads[0][:50]))
    refused(ValueError, "elements", lambda t: t.m.__setitem__(0, t.m[0][:50]))
    refused(ValueError, "contiguous", lambda t: t.v.__setitem__(0, t.v[0].repeat(2)[::2]))
    refused(TypeError, "float32", lambda t: t.m.__setitem__(0, t.m[0].bfloat16()))
    refused(TypeError, "float8", lambda t: t.m.__setitem__(0, t.m[0].float()), bits=8)
    refused(ValueError, "elements", lambda t: t.v_scale.__setitem__(1, t.v_scale[1][:1]), bits=8)
    refused(TypeError, "int32", lambda t: t.steps.__setitem__(0, t.steps[0].float()))
    refused(RuntimeError, "no CPU path", lambda t: t.grads.__setitem__(0, t.grads[0].cpu()))
    refused(ValueError, "betas", lambda t: None, betas=(1.0, 0.9))
    refused(ValueError, "lr", lambda t: None, lr=-1.0)
    refused(TypeError, "grad_scale", lambda t: None, grad_scale=torch.ones(1, device="cuda").double())
    with pytest.raises(ValueError, match="8-bit"):
        t = Tensors([100], torch.float32, 8)
        adamw_step(t.params, t.grads, t.m, t.v, t.steps, lr=0.1, exp_avg_scales=t.m_scale)


@pytest.mark.gpu
def test_tensors_that_share_memory_are_refused():
    from flashfusedmoe_b200 import adamw_step

    def call(p, g, m, v, step, **h):
        adamw_step([*p], [*g], [*m], [*v], [*step], lr=1e-3, **h)

    room = torch.zeros(100000, device="cuda")
    step = torch.zeros(4, dtype=torch.int32, device="cuda")
    piece = [room[1000 * k:1000 * k + 1000] for k in range(9)]
    call(piece[:2], piece[2:4], piece[4:6], piece[6:8], (step[0], step[1]))   # side by side is not on another
    call(piece[:2], [piece[2]] * 2, piece[4:6], piece[6:8], (step[0], step[1]))   # gradients are only read
    shifted = room[999:1999]
    for p, g, m in (((piece[0], shifted), piece[2:4], piece[4:6]), (piece[:2], (shifted, piece[3]), piece[4:6]),
                    ((piece[0], piece[5]), piece[2:4], (piece[4], shifted)), (piece[:2], (piece[2], piece[0]), piece[4:6])):
        with pytest.raises(ValueError, match="lies on another"):
            call(p, g, m, piece[6:8], (step[0], step[1]))
    with pytest.raises(ValueError, match="lies on another"):
        call(piece[:1], piece[1:2], piece[2:3], piece[3:4], (step[0],), grad_scale=room[500:501])
    assert step.tolist() == [2, 2, 0, 0] and not room.any()
