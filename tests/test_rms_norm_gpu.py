"""GPU: root-mean-square norm with the residual's addition against the formula in 64 bits: forward, the 8-bit output, gradients.

Bounds count roundings: half a step of the type (eps / 2) of the result, and C steps of fp32 for what lies before it: a row's sum is added up
over at most 64 values in a thread, five steps in a warp and 32 warps; the root, the quotient and three products follow."""

import pytest
import torch

from flashfusedmoe_b200 import MoELayer, RMSNorm, rms_norm

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
C = 128 * 2.0 ** -24


def _inputs(rows, dim, dtype, residual=True, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    x = (rand(rows, dim) * (0.5 + 2 * torch.rand(rows, 1, device="cuda", generator=g))).to(dtype)
    return x, (3 * rand(rows, dim)).to(dtype) if residual else None, (1 + 0.2 * rand(dim)).to(dtype)


def _formula(x, residual, weight, eps, offset=0.0):
    """h, xh, y, r in 64 bits; h rounded as it is handed on."""
    h = x.double() if residual is None else (x.float() + residual.float()).to(x.dtype).double()
    r = 1.0 / (h.square().mean(-1, keepdim=True) + eps).sqrt()
    w = 1.0 if weight is None else weight.double()
    return h, h * r, h * r * (w + offset), r


def _close(got, want, extra=0.0):
    """extra: the sum of magnitudes that fp32 roundings are relative to, where it is not the result itself"""
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps
    bound = half * want.abs() + C * (want.abs() + extra) * (1 + half) + tiny
    off = (got.double() - want).abs()
    assert got.shape == want.shape and bool((off <= bound).all()), float((off / bound).max())


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,dim", [(1, 1), (1, 4096), (3, 7), (5, 64), (2, 8192), (7, 1000), (300, 1024), (149, 2051), (2, 16384), (700, 127),
                                      (1200, 520), (65, 7168)])
@pytest.mark.parametrize("residual", [True, False])
def test_forward(rows, dim, dtype, residual):
    x, more, w = _inputs(rows, dim, DTYPES[dtype], residual)
    h, _, y, _ = _formula(x, more, w, 1e-6)
    out = rms_norm(x, w, residual=more)
    if residual:
        out, got_h = out
        assert got_h.dtype == x.dtype and torch.equal(got_h.double(), h)
    assert out.dtype == x.dtype
    _close(out, y)


def test_forward_of_the_longest_rows_and_options():
    for dtype, dim in ((torch.bfloat16, 32768), (torch.float32, 16384)):
        x, more, _ = _inputs(3, dim, dtype)
        y, h = rms_norm(x, None, 0.5, residual=more)
        _close(y, _formula(x, more, None, 0.5)[2])
    x, more, w = _inputs(9, 200, torch.bfloat16)
    _close(rms_norm(x, w.float(), 1e-6, weight_offset=1.0), _formula(x, None, w, 1e-6, 1.0)[2])          # a weight of another type
    _close(rms_norm(x.float(), w, 1e-6, weight_offset=-0.25), _formula(x.float(), None, w, 1e-6, -0.25)[2])
    assert rms_norm(x.view(3, 3, 200)).shape == (3, 3, 200)
    assert rms_norm(x[:0], w).shape == (0, 200)


def test_strides_and_alignment():
    x, more, w = _inputs(40, 512, torch.bfloat16)
    wide = torch.zeros(40, 1024, dtype=x.dtype, device="cuda")
    for at in (0, 8, 3):       # rows further apart, on 16 bytes and off them
        wide[:, at:at + 512] = x
        y, h = rms_norm(wide[:, at:at + 512], w, residual=more)
        want, want_h = rms_norm(x, w, residual=more)
        assert torch.equal(h, want_h)
        _close(y, _formula(x, more, w, 1e-6)[2])
    _close(rms_norm(x.t().contiguous().t(), w), _formula(x, None, w, 1e-6)[2])
    flat = torch.zeros(513, dtype=x.dtype, device="cuda")
    flat[1:] = w
    _close(rms_norm(x, flat[1:]), _formula(x, None, w, 1e-6)[2])
    values, scale = rms_norm(wide[:, 3:515].copy_(x), flat[1:], quantize=True)
    want, want_scale = rms_norm(x, w, quantize=True)
    assert torch.equal(values.view(torch.uint8), want.view(torch.uint8)) and torch.equal(scale, want_scale)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,dim", [(1, 16), (1, 4096), (3, 144), (300, 1024), (149, 2064), (2, 16384), (65, 7168), (3000, 128), (1, 8192)])
def test_8_bit_output(rows, dim, dtype):
    x, more, w = _inputs(rows, dim, DTYPES[dtype])
    x[-1] = 0
    more[-1] = 0      # a row of zeros has scale 1
    if dim >= 256:
        w[128:256] = 0
    values, scale, h = rms_norm(x, w, residual=more, quantize=True)
    want_h, _, y, _ = _formula(x, more, w, 1e-6)
    assert torch.equal(h.double(), want_h) and values.dtype == torch.float8_e4m3fn
    blocks = (dim + 127) // 128
    y = torch.nn.functional.pad(y, (0, blocks * 128 - dim)).view(rows, blocks, 128)
    top = y.abs().amax(2)
    want = torch.where(top > 0, top / 448, 1.0)
    assert scale.shape == want.shape and bool(((scale.double() - want).abs() <= C * want).all())
    got = torch.nn.functional.pad(values.double(), (0, blocks * 128 - dim)).view(rows, blocks, 128)
    # half a step of e4m3: 2^-4 of the value, 2^-10 where numbers are no multiples of a smaller one; and fp32's before it
    off, over = (got * scale.double()[:, :, None] - y).abs(), scale.double()[:, :, None]
    assert bool((off <= torch.maximum(2.0 ** -4 * y.abs(), 2.0 ** -10 * over) * (1 + 2.0 ** -10) + C * y.abs()).all())


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows", [5, 6000])
def test_8_bit_codes_are_the_rounded_quotients(rows, dtype):
    """h = k / 256 with whole k, and eps such that the root is 1: y = k m / 256 and the scale m / 256 are exact. k halfway between two e4m3 numbers
    goes to the even one, and a scale or a reciprocal that is a rounding off would put some of them on the other side."""
    half = [17 + 2 * i for i in range(8)] + [34 + 4 * i for i in range(8)] + [68 + 8 * i for i in range(8)] + [136 + 16 * i for i in range(8)]
    half = torch.tensor(half + [448] + [3] * 95, dtype=torch.float32)
    g = torch.Generator().manual_seed(0)
    k = torch.stack([half[torch.rand(rows, 128, generator=g).argsort(1)] for _ in range(2)], 1).view(rows, 256)
    k *= torch.where(torch.rand(rows, 256, generator=g) < 0.5, -1.0, 1.0)
    eps = 1.0 - float(2 * half.double().square().sum()) * 2.0 ** -24
    for m in (7.0, 13.0, 15.0, 61.0):
        values, scale = rms_norm((k / 256).to(DTYPES[dtype]).cuda(), torch.full((256,), m, device="cuda"), eps, quantize=True)
        assert bool((scale == m / 256).all())
        assert torch.equal(values.cpu().view(torch.uint8), k.to(torch.float8_e4m3fn).view(torch.uint8))


def test_8_bit_output_of_extreme_rows():
    w = torch.ones(256, device="cuda")
    x = torch.randn(4, 256, device="cuda")
    x[0] *= 1e-30                       # eps alone is under the root: values about 1e-27
    x[1, 5] = float("nan")
    x[2, 200] = float("inf")
    values, scale = rms_norm(x, w, quantize=True)
    want = (x[0].double() / 1e-3).view(2, 128)
    assert bool(((values[0].double().view(2, 128) * scale[0].double()[:, None] - want).abs() <= 2.0 ** -4 * want.abs().amax()).all())
    assert bool(values[1].float().isnan().all())
    assert bool(torch.isnan(values[2, 200:201].float() * scale[2, 1]).all())
    _close(rms_norm(x[3:], w), _formula(x[3:], None, w, 1e-6)[2])


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,dim", [(1, 1), (1, 4096), (3, 7), (5, 64), (2, 8192), (7, 1000), (700, 1024), (149, 2051), (3, 16384), (700, 127),
                                      (1200, 520), (5000, 64), (600, 7168), (400, 16384), (400, 9216), (5, 32768), (40, 12001)])
@pytest.mark.parametrize("residual", [True, False])
def test_gradients(rows, dim, dtype, residual):
    if dtype == "fp32" and dim > 16384:
        pytest.skip("fp32 rows end at 16384")
    x, more, w = _inputs(rows, dim, DTYPES[dtype], residual)
    dy, dh, _ = _inputs(rows, dim, DTYPES[dtype], seed=1)
    leaves = [t.requires_grad_() for t in (x, more, w) if t is not None]
    out = rms_norm(x, w, residual=more)
    got = torch.autograd.grad(out, leaves, [dy, dh] if residual else dy)
    with torch.no_grad():
        _, xh, _, r = _formula(x, more, w, 1e-6)
        g = dy.double() * w.double()
        inner = (g * xh).mean(-1, keepdim=True)
        dx = r * (g - xh * inner)
        extra = r * (g.abs() + xh.abs() * (g * xh).abs().mean(-1, keepdim=True))
        if residual:
            dx, extra = dx + dh.double(), extra + dh.double().abs()
            assert torch.equal(got[0], got[1])
        _close(got[0], dx, extra)
        each = dy.double() * xh
        # a column's sum runs over the rows: at most so many additions
        _close(got[-1], each.sum(0), each.abs().sum(0) * (rows + 128) / 128)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows", [6, 25000])
@pytest.mark.parametrize("residual", [True, False])
def test_gradients_of_tiny_rows(rows, dtype, residual):
    """Rows of whole multiples of 2^-66, whose squares are exact sums in fp32, without eps: the root's inverse is about 2^66, its square is infinite."""
    g = torch.Generator(device="cuda").manual_seed(0)
    x = (torch.randint(-2, 3, (rows, 256), device="cuda", generator=g) * 2.0 ** -66).to(DTYPES[dtype])
    more = torch.zeros_like(x) if residual else None
    _, _, w = _inputs(1, 256, DTYPES[dtype])
    dy, _, _ = _inputs(rows, 256, DTYPES[dtype], seed=1)
    x.requires_grad_(), w.requires_grad_()
    out = rms_norm(x, w, 0.0, residual=more)
    got = torch.autograd.grad(out, [x, w], [dy, torch.zeros_like(dy)] if residual else dy)
    with torch.no_grad():
        _, xh, y, r = _formula(x, None, w, 0.0)
        _close(out[0] if residual else out, y)
        g = dy.double() * w.double()
        dx = r * (g - xh * (g * xh).mean(-1, keepdim=True))
        _close(got[0], dx, r * (g.abs() + xh.abs() * (g * xh).abs().mean(-1, keepdim=True)))
        each = dy.double() * xh
        _close(got[1], each.sum(0), each.abs().sum(0) * (rows + 128) / 128)


def test_gradients_of_some_inputs():
    x, more, w = _inputs(50, 384, torch.bfloat16)
    dy, dh, _ = _inputs(50, 384, torch.bfloat16, seed=1)

    def grads(*wanted, used=(True, True), residual=more):
        for t in (x, more, w):
            t.requires_grad_(any(t is u for u in wanted))
        out = rms_norm(x, w, residual=residual)
        pairs = [(o, g) for o, g, u in zip(out if residual is not None else [out], (dy, dh), used) if u]
        return torch.autograd.grad([p[0] for p in pairs], wanted, [p[1] for p in pairs])

    dx, dmore, dw = grads(x, more, w)
    assert torch.equal(grads(w)[0], dw) and torch.equal(grads(more)[0], dmore) and torch.equal(grads(x)[0], dx)
    only_h = grads(x, more, w, used=(False, True))
    assert torch.equal(only_h[0], dh) and torch.equal(only_h[1], dh) and not bool(only_h[2].any())
    only_y = grads(x, w, used=(True, False))
    assert torch.equal(only_y[1], dw) and not torch.equal(only_y[0], dx)
    x.requires_grad_()
    y = rms_norm(x)
    assert torch.equal(torch.autograd.grad(y, x, dy)[0], torch.autograd.grad(rms_norm(x, torch.ones_like(w).detach()), x, dy)[0])
    # without a weight, with a residual of which alone a gradient is asked for; the same tensor as both
    x.requires_grad_(False), more.requires_grad_()
    dy, dh, _ = _inputs(50, 384, torch.bfloat16, seed=2)
    alone = torch.autograd.grad(rms_norm(x, residual=more), more, [dy, dh])[0]
    ones = torch.ones_like(w).detach()
    assert torch.equal(alone, torch.autograd.grad(rms_norm(x, ones, residual=more), more, [dy, dh])[0])
    x.requires_grad_()
    twice, = torch.autograd.grad(rms_norm(x, w.detach(), residual=x), x, [dy, dh])
    again = x.detach().clone().requires_grad_()
    once, = torch.autograd.grad(rms_norm(x, w.detach(), residual=again), x, [dy, dh])
    assert torch.equal(twice, once + once)
    # an expanded gradient, and one that is not contiguous
    a = torch.autograd.grad(rms_norm(x, w).sum(), x)[0]
    assert torch.equal(a, torch.autograd.grad(rms_norm(x, w), x, torch.ones_like(x))[0])
    b = torch.autograd.grad(rms_norm(x, w), x, dy.t().contiguous().t())[0]
    assert torch.equal(b, torch.autograd.grad(rms_norm(x, w), x, dy)[0])
    with pytest.raises(RuntimeError, match="once"):
        g, = torch.autograd.grad(rms_norm(x, w), x, dy, create_graph=True)
        g.sum().backward()


def test_gradients_against_differences():
    """fp32: the difference quotient over 2 t is off by t^2 |f'''| / 6 and by the roundings of f over t."""
    x, more, w = (t[:4, :24].contiguous() if t.dim() == 2 else t[:24].contiguous() for t in _inputs(4, 24, torch.float32))
    dy, dh = (torch.randn(4, 24, device="cuda") for _ in range(2))
    leaves = [t.requires_grad_() for t in (x, more, w)]

    def value():
        y, h = rms_norm(x, w, residual=more)
        return (y.double() * dy).sum() + (h.double() * dh).sum()

    got = torch.autograd.grad(value(), leaves)
    t = 2.0 ** -7
    for leaf, g in zip(leaves, got):
        for i in range(0, leaf.numel(), 11):
            with torch.no_grad():
                flat = leaf.view(-1)
                was = flat[i].clone()
                flat[i] = was + t
                up, ahead = value(), flat[i].double()
                flat[i] = was - t
                down, behind = value(), flat[i].double()
                flat[i] = was
                # f''' of the norm of rows of scale 1 and more is of order 1; a hundred roundings of values up to 10 over 2 t
                assert abs(float((up - down) / (ahead - behind) - g.view(-1)[i].double())) < 10 * t * t + 100 * 10 * 2.0 ** -24 / (2 * t) * 4


def test_same_bits_again_and_in_graphs_on_other_streams():
    x, more, w = _inputs(3000, 1024, torch.bfloat16)
    dy, dh, _ = _inputs(3000, 1024, torch.bfloat16, seed=1)
    leaves = [t.requires_grad_() for t in (x, more, w)]

    def step():
        return torch.autograd.grad(rms_norm(x, w, residual=more), leaves, [dy, dh])

    first = step()
    assert all(torch.equal(a, b) for a, b in zip(first, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, out))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
        with torch.no_grad():
            q = rms_norm(x, w, residual=more, quantize=True)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(first, out))
    with torch.no_grad():
        x.copy_(dy)
        graph.replay()
        want = rms_norm(x, w, residual=more, quantize=True)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(q, want))
    assert all(torch.equal(a, b) for a, b in zip(step(), out))


def test_rows_beyond_32_bits():
    rows, dim = 2 ** 19 + 3, 4104
    if torch.cuda.get_device_properties(0).total_memory < 60e9:
        pytest.skip("needs 20 GB")
    x = torch.randn(rows, dim, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(dim, dtype=torch.bfloat16, device="cuda")
    y, h = rms_norm(x, w, residual=x)
    for at in (slice(0, 2), slice(rows - 2, rows)):
        _close(y[at], _formula(x[at], x[at], w, 1e-6)[2])
        assert torch.equal(h[at], x[at] * 2)


def test_module_and_layer():
    norm = RMSNorm(96, dtype=torch.bfloat16, device="cuda")
    x = torch.randn(5, 96, dtype=torch.bfloat16, device="cuda")
    _close(norm(x), _formula(x, None, norm.weight.detach(), 1e-6)[2])
    layer = MoELayer(256, 512, 4, pre_norm="rms").cuda().bfloat16()
    x = torch.randn(64, 256, dtype=torch.bfloat16, device="cuda")
    plain = MoELayer(256, 512, 4).cuda().bfloat16()
    plain.load_state_dict({k: v for k, v in layer.state_dict().items() if not k.startswith("norm")})
    out, _ = layer(x)
    want, _ = plain(rms_norm(x, layer.norm.weight, 1e-5))
    assert torch.equal(out, want)
    out.sum().backward()
    assert layer.norm.weight.grad is not None


# Rows enough for the kernels that go through them in a ring, with teams of 1 to 512 threads a row on 148 SMs; widths that end inside a chunk of a
# thread's, or inside a block of 128
MANY = [(5000, 1024), (4800, 520), (600, 7168), (80000, 64), (1600, 2056), (700, 8192), (25000, 200)]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,dim", MANY + [(160000, 8)])
@pytest.mark.parametrize("residual", [True, False])
def test_forward_of_many_rows(rows, dim, dtype, residual):
    test_forward(rows, dim, dtype, residual)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,dim", [(5000, 1024), (5000, 144), (700, 7168), (1600, 2064), (5000, 16), (700, 8192)])
def test_8_bit_output_of_many_rows(rows, dim, dtype):
    test_8_bit_output(rows, dim, dtype)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,dim", MANY)
@pytest.mark.parametrize("residual", [True, False])
def test_gradients_of_many_rows(rows, dim, dtype, residual):
    test_gradients(rows, dim, dtype, residual)


def test_options_of_many_rows():
    rows, dim = 5000, 1024
    x, more, w = _inputs(rows, dim, torch.bfloat16)
    y, h = rms_norm(x, None, 0.5, residual=more)
    want, _, out, _ = _formula(x, more, None, 0.5)
    assert torch.equal(h.double(), want)
    _close(y, out)
    _close(rms_norm(x, w.float(), weight_offset=1.0), _formula(x, None, w, 1e-6, 1.0)[2])
    wide = torch.zeros(rows, 2 * dim, dtype=x.dtype, device="cuda")   # rows further apart
    wide[:, 8:8 + dim], wide[:, dim + 8:] = x, 0
    y, h = rms_norm(wide[:, 8:8 + dim], w, residual=more)
    assert torch.equal(h.double(), _formula(x, more, w, 1e-6)[0])
    _close(y, _formula(x, more, w, 1e-6)[2])
    values, scale = rms_norm(wide[:, 8:8 + dim], w, quantize=True)
    again = rms_norm(x, w, quantize=True)
    assert torch.equal(values.view(torch.uint8), again[0].view(torch.uint8)) and torch.equal(scale, again[1])
    x[17, 5], x[4999, 1000] = float("nan"), float("inf")     # stay in their rows
    y = rms_norm(x, w)
    rest = torch.ones(rows, dtype=torch.bool, device="cuda")
    rest[17] = rest[4999] = False
    assert bool(y[17].isnan().all()) and bool(y[4999, 1000].isnan()) and not bool(y[4999, :1000].any())
    _close(y[rest], _formula(x[rest], None, w, 1e-6)[2])
    dy = _inputs(rows, dim, torch.bfloat16, seed=1)[0]
    dx, = torch.autograd.grad(rms_norm(x.requires_grad_(), w), x, dy)
    assert bool(dx[17].isnan().all()) and bool(dx[rest].isfinite().all())
