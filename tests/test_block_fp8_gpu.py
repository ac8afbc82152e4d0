"""GPU: e4m3 operands with a scale for every 128 values, and their products, against the formula in 64 bits."""

import pytest
import torch

from flashfusedmoe_b200 import linear_e4m3, ops, quantize_e4m3, rms_norm

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _spread(scale, block_rows, shape):
    s = scale.double().repeat_interleave(128, dim=-1)[..., :shape[-1]]
    return s if block_rows == 1 else s.repeat_interleave(block_rows, dim=-2)[..., :shape[-2], :]


def _wide(values, scale, block_rows):
    return values.double() * _spread(scale, block_rows, values.shape)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("block_rows,shape", [(1, (1, 16)), (1, (5, 128)), (1, (61, 7168)), (1, (3, 2, 272)), (1, (1000, 144)), (1, (16,)), (128, (1, 16)),
                                              (128, (128, 128)), (128, (129, 144)), (128, (3, 300, 272)), (128, (2, 2, 64, 1024)), (128, (1000, 128))])
def test_quantize(block_rows, shape, dtype):
    x = (torch.randn(shape, device="cuda") * torch.rand(shape[:-1] + (1,), device="cuda") * 5).to(DTYPES[dtype])
    if len(shape) > 1:   # blocks of zeros
        x[..., :1, :] = 0
        x[..., -1, 128:] = 0
    values, scale = quantize_e4m3(x, block_rows)
    K = shape[-1]
    lead = shape[:-1] + ((K + 127) // 128,) if block_rows == 1 else shape[:-2] + ((shape[-2] + 127) // 128, (K + 127) // 128)
    assert values.shape == x.shape and values.dtype == torch.float8_e4m3fn and tuple(scale.shape) == lead and scale.dtype == torch.float32
    # the block's largest magnitude over 448, one rounding
    top = torch.nn.functional.max_pool2d(x.double().abs().reshape(-1, 1, *((1, K) if len(shape) == 1 else shape[-2:])), (block_rows, 128),
                                         ceil_mode=True).view(lead)
    want = torch.where(top > 0, top / 448, 1.0)
    assert bool(((scale.double() - want).abs() <= 2.0 ** -24 * want).all())
    # half a step of e4m3, 2^-4 of the value or 2^-10 scales, and the roundings of the inverse and the product
    y = x.double()
    bound = torch.maximum(2.0 ** -4 * y.abs(), 2.0 ** -10 * _spread(scale, block_rows, shape)) * (1 + 2.0 ** -20)
    assert bool(((_wide(values, scale, block_rows) - y).abs() <= bound).all())


def test_quantize_extremes_and_strides():
    x = torch.randn(4, 256, device="cuda")
    x[0] *= 1e-41          # below fp32's normal numbers: the scale stays 2^-126
    x[1, 3] = float("nan")
    x[2, 130] = float("-inf")
    x[3, :128] = 3e38
    values, scale = quantize_e4m3(x)
    assert bool((scale[0] == 2.0 ** -126).all()) and bool(((_wide(values[:1], scale[:1], 1) - x[:1].double()).abs() <= 2.0 ** -136).all())
    rest = x[1, :128].double()
    finite = ~rest.isnan()
    assert bool(values[1, 3].float().isnan()) and bool((scale[1, 0].double() - rest[finite].abs().max() / 448).abs() <= 2.0 ** -24 * scale[1, 0].double())
    assert bool((_wide(values[2:3], scale[2:3], 1)[0, 128:]).isnan().all()) and not bool(values[2, :128].float().isnan().any())
    assert bool(((_wide(values[3:], scale[3:], 1)[0, :128] - 3e38).abs() <= 2.0 ** -20 * 3e38).all())
    wide = torch.zeros(4, 600, device="cuda", dtype=torch.bfloat16)
    x = torch.randn(4, 256, device="cuda").bfloat16()
    for at in (0, 8, 5):
        wide[:, at:at + 256] = x
        for a, b in zip(quantize_e4m3(wide[:, at:at + 256]), quantize_e4m3(x)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        for a, b in zip(quantize_e4m3(wide[:, at:at + 256], 128), quantize_e4m3(x, 128)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    for shape, block_rows in (((0, 64), 1), ((0, 64), 128), ((0, 5, 64), 128), ((3, 0, 64), 128)):
        values, scale = quantize_e4m3(torch.empty(shape, device="cuda"), block_rows)
        assert values.shape == shape and scale.numel() == 0


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("block_rows,rows,K", [(1, 61, 7168), (1, 3000, 272), (128, 300, 2064)])
def test_codes_are_the_rounded_quotients(block_rows, rows, K, dtype):
    """Values halfway between two e4m3 numbers, which 16-bit inputs often are, go to the even one: the codes are those of the quotient in fp32."""
    x = torch.randn(rows, K).to(DTYPES[dtype])
    # k m with k halfway between two e4m3 numbers, against a scale of m: a rounded 1 / m puts some of them on the other side
    halfway = torch.tensor([17.0 + 2 * i for i in range(8)] + [34.0 + 4 * i for i in range(8)] + [0.5 + i for i in range(8)])
    for i, m in enumerate((7.0, 13.0, 15.0, 61.0, 63.0)):
        at = slice(128 * (i % 2), 128 * (i % 2) + 128)
        where = i // 2 * block_rows
        x[where:where + block_rows, at] = 0
        x[where, at.start:at.start + 24] = (halfway * m).to(x.dtype)
        x[where, at.start + 24:at.start + 48] = (-halfway * m).to(x.dtype)
        x[where, at.start + 127] = 448 * m
    values, scale = quantize_e4m3(x.cuda(), block_rows)
    spread = _spread(scale.cpu(), block_rows, x.shape).float()
    assert [float(scale[i // 2, i % 2]) for i in range(5)] == [7.0, 13.0, 15.0, 61.0, 63.0]
    assert torch.equal(values.cpu().view(torch.uint8), (x.float() / spread).to(torch.float8_e4m3fn).view(torch.uint8))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("block_rows", [1, 128])
def test_extreme_values_of_all_types(block_rows, dtype):
    """The type's smallest numbers, NaN in either half of a word and in whole words, zeros of both signs: codes and scales of a division on the host."""
    x = torch.randn(4 * block_rows, 256).to(DTYPES[dtype])
    tiny = torch.finfo(DTYPES[dtype]).tiny * torch.finfo(DTYPES[dtype]).eps
    x[:block_rows, :128] = (torch.randint(-7, 8, (block_rows, 128)) * tiny).to(x.dtype)
    x[block_rows, [0, 3, 10, 11, 127]] = float("nan")
    x[2 * block_rows, 128:] = -0.0
    x[2 * block_rows + 1 if block_rows > 1 else 2, 5] = 448.0
    x[3 * block_rows, 7] = float("-inf")
    values, scale = quantize_e4m3(x.cuda(), block_rows)
    # NaN counts as 0 for the scale
    top = torch.nn.functional.max_pool2d(x.float().nan_to_num(0.0, float("inf"), -float("inf")).abs()[None, None], (block_rows, 128))[0, 0]
    want = torch.where(top > 0, (top / 448).clamp(min=2.0 ** -126), 1.0)
    assert torch.equal(scale.cpu(), want)
    codes = (x.float() / _spread(want, block_rows, x.shape).float()).to(torch.float8_e4m3fn)
    nan = codes.float().isnan()
    assert torch.equal(values.cpu().float().isnan(), nan) and int(nan.sum()) == 6
    assert torch.equal(values.cpu().view(torch.uint8)[~nan], codes.view(torch.uint8)[~nan])


def _operands(rows, N, K, experts=None, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, K, device="cuda", generator=g) * (0.2 + 3 * torch.rand(rows, 1, device="cuda", generator=g))
    w = torch.randn((N, K) if experts is None else (experts, N, K), device="cuda", generator=g) * K ** -0.5
    w *= 0.1 + 2 * torch.rand(w.shape[:-1] + (1,), device="cuda", generator=g)
    return (*quantize_e4m3(x), *quantize_e4m3(w, 128))


def _check(out, x, xs, w, ws):
    """The products of 8-bit numbers are exact in fp32. A sum of K of them, in any order and with a rounding for every block's scales, is off by
    at most K + 2 ceil(K / 128) + 2 half steps of fp32 of the sum of magnitudes, twice that if a sum is cut off instead of rounded."""
    a, b = _wide(x, xs, 1), _wide(w, ws, 128)
    want, size = a @ b.t(), a.abs() @ b.abs().t()
    K = x.shape[-1]
    bound = 2 * (K + 2 * ((K + 127) // 128) + 2) * 2.0 ** -24 * size
    half = torch.finfo(out.dtype).eps / 2
    bound = bound * (1 + half) + half * want.abs() + torch.finfo(out.dtype).tiny * torch.finfo(out.dtype).eps
    off = (out.double() - want).abs()
    assert out.shape == want.shape and bool((off <= bound).all()), float((off / bound).nan_to_num(0).max())


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("block_rows,rows,K", [(1, 61, 7168), (1, 3000, 272), (128, 300, 2064)])
def test_codes_are_the_rounded_quotients(block_rows, rows, K, dtype):
    """Values halfway between two e4m3 numbers, which 16-bit inputs often are, go to the even one: the codes are those of the quotient in fp32."""
    x = torch.randn(rows, K).to(DTYPES[dtype])
    # k m with k halfway between two e4m3 numbers, against a scale of m: a rounded 1 / m puts some of them on the other side
    halfway = torch.tensor([17.0 + 2 * i for i in range(8)] + [34.0 + 4 * i for i in range(8)] + [0.5 + i for i in range(8)])
    for i, m in enumerate((7.0, 13.0, 15.0, 61.0)):
        row, col = i // 2 * block_rows, i % 2 * 128
        x[row:row + block_rows, col:col + 128] = 0
        x[row, col:col + 24] = (halfway * m).to(x.dtype)
        x[row, col + 24:col + 48] = (-halfway * m).to(x.dtype)
        x[row, col + 127] = 448 * m
    values, scale = quantize_e4m3(x.cuda(), block_rows)
    spread = _spread(scale.cpu(), block_rows, x.shape).float()
    assert spread[0, 0] == 7.0 and spread[0, 128] == 13.0 and spread[block_rows, 0] == 15.0
    assert torch.equal(values.cpu().view(torch.uint8), (x.float() / spread).to(torch.float8_e4m3fn).view(torch.uint8))


@pytest.mark.parametrize("block_rows", [1, 128])
def test_codes_beside_borders_at_all_scales(block_rows):
    """Values at, one step above and one below the borders between e4m3 numbers, for scales of every size: the codes of a division all the same."""
    g = torch.Generator().manual_seed(0)
    rows = 20000 if block_rows == 1 else 300
    scale = (1 + torch.rand(rows, generator=g)) * torch.exp2(torch.randint(-126, 119, (rows,), generator=g).float())
    # mantissas at which quotients come closest to the middle between two fp32 numbers
    near = torch.arange(8, 16).repeat_interleave(33) * 2 ** 20 + torch.arange(-16, 17).repeat(8)
    near = near[near >= 2 ** 23].float()
    scale[:near.numel()] = (near * torch.exp2(torch.randint(-80, 80, (near.numel(),), generator=g).float()))[:rows]
    scale[-8:] = torch.tensor([2.0 ** -126, 1e-38, 2.0 ** -80, 2.0 ** -79, 2.0 ** -79 * 1.5, 7e35, 2.0 ** -149, 0.0])
    top = (448 * scale).clamp(max=3.4e38)
    scale = torch.where(top > 0, (top / 448).clamp(min=2.0 ** -126), 1.0)
    border = torch.arange(16, 32).float() / 16 * torch.exp2(torch.randint(-10, 8, (rows, 16), generator=g).float()) * scale[:, None]
    x = torch.cat([border, torch.nextafter(border, border * 2), torch.nextafter(border, border * 0)], 1)
    x = torch.cat([x, -x, torch.zeros(rows, 1), -torch.zeros(rows, 1), torch.rand(rows, 29, generator=g) * top[:, None], top[:, None]], 1)
    x = torch.minimum(torch.maximum(x, -top[:, None]), top[:, None])
    if block_rows == 128:   # a block for each
        x, where = torch.zeros(rows * 128, 128), x
        x[torch.arange(rows) * 128 + torch.arange(rows) % 128] = where
        scale = scale.repeat_interleave(128)
    values, got = quantize_e4m3(x.cuda(), block_rows)
    assert torch.equal(got.cpu().view(-1), scale[::block_rows])
    assert torch.equal(values.cpu().view(torch.uint8), (x / scale[:, None]).to(torch.float8_e4m3fn).view(torch.uint8))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,N,K", [(1, 1, 16), (1, 128, 128), (1, 4096, 7168), (3, 130, 144), (16, 64, 272), (17, 129, 256), (64, 500, 1040), (65, 256, 128),
                                      (128, 128, 128), (129, 127, 400), (300, 1000, 2064), (1000, 3001, 512), (4096, 2048, 1024), (200, 40000, 64),
                                      (1, 3001, 2064), (1, 40000, 272), (1, 200000, 64), (1, 130, 16384), (1, 130, 16400), (1, 257, 528), (1, 14000, 4096), (2, 4096, 7168)])
def test_dense(rows, N, K, dtype):
    x, xs, w, ws = _operands(rows, N, K)
    out = linear_e4m3(x, xs, w, ws, out_dtype=DTYPES[dtype])
    assert out.dtype == DTYPES[dtype]
    _check(out, x, xs, w, ws)
    ops.check_status()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,N,K", [(33, 700, 2048), (64, 4096, 2064), (20, 1000, 2048), (17, 130, 4096), (64, 129, 16400), (48, 257, 2064)])
def test_dense_rows_of_a_tile_whose_contraction_is_shared(rows, N, K, dtype):
    test_dense(rows, N, K, dtype)


# rows of each expert, and rows behind the last
GROUPS = [([1], 0), ([0], 3), ([5, 0, 1, 64, 0, 65], 2), ([0, 0, 0, 0], 7), ([128, 0, 129, 1, 300, 127], 0), ([1000, 3, 0, 0, 700], 130),
          ([3] * 40, 5), ([0] * 33 + [200] + [0] * 31 + [1], 1), ([400, 300, 500, 2], 0)]


@pytest.mark.parametrize("sizes,spare", GROUPS)
@pytest.mark.parametrize("N,K,dtype", [(257, 400, "bf16"), (384, 1024, "fp32"), (1000, 144, "fp16")])
def test_grouped(sizes, spare, N, K, dtype):
    rows = sum(sizes) + spare
    x, xs, w, ws = _operands(rows, N, K, len(sizes))
    ends = torch.tensor(sizes).cumsum(0).int().cuda()
    out = linear_e4m3(x, xs, w, ws, ends=ends, out_dtype=DTYPES[dtype])
    begin = 0
    for e, n in enumerate(sizes):
        _check(out[begin:begin + n], x[begin:begin + n], xs[begin:begin + n], w[e], ws[e])
        begin += n
    assert not bool(out[begin:].any())
    ops.check_status()


@pytest.mark.parametrize("rows,N,K,experts", [(288, 2816, 2048, 64), (100, 4096, 1024, 8), (700, 1000, 2064, 40), (6000, 1400, 528, 48)])
def test_many_tiles_a_block_of_threads(rows, N, K, experts):
    """Tiles follow one another on an SM: every one of them, and the same bits each time."""
    x, xs, w, ws = _operands(rows, N, K, experts)
    sizes = torch.bincount(torch.randint(0, experts, (rows,), generator=torch.Generator().manual_seed(1)), minlength=experts)
    ends = sizes.cumsum(0).int().cuda()
    outs = [linear_e4m3(x, xs, w, ws, ends=ends) for _ in range(8)]
    assert all(torch.equal(o, outs[0]) for o in outs)
    begin = 0
    for e, n in enumerate(sizes.tolist()):
        _check(outs[0][begin:begin + n], x[begin:begin + n], xs[begin:begin + n], w[e], ws[e])
        begin += n


def test_groups_do_not_reach_into_one_another():
    """NaN rows and weights of one expert stay in its rows, and those behind the last in none."""
    for sizes, spare in (([5, 7, 3], 4), ([200, 130, 300], 40)):
        rows, N, K = sum(sizes) + spare, 300, 272
        x, xs, w, ws = _operands(rows, N, K, 3)
        ends = torch.tensor(sizes).cumsum(0).int().cuda()
        want = linear_e4m3(x, xs, w, ws, ends=ends)
        xs[sizes[0]:sizes[0] + sizes[1]] = float("nan")
        x.view(torch.uint8)[sizes[0] + sizes[1] + sizes[2]:] = 0x7f
        ws[1] = float("inf")
        out = linear_e4m3(x, xs, w, ws, ends=ends)
        assert torch.equal(out[:sizes[0]], want[:sizes[0]]) and torch.equal(out[sizes[0] + sizes[1]:], want[sizes[0] + sizes[1]:])
        assert bool(out[sizes[0]:sizes[0] + sizes[1]].isnan().all())


def test_strides_shapes_and_alignment():
    x, xs, w, ws = _operands(24, 200, 256)
    want = linear_e4m3(x, xs, w, ws)
    wide = torch.zeros(24, 1024, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    for at in (0, 16, 5):
        wide.view(torch.uint8)[:, at:at + 256] = x.view(torch.uint8)
        assert torch.equal(linear_e4m3(wide[:, at:at + 256], xs, w, ws), want)
    assert torch.equal(linear_e4m3(x.view(2, 12, 256), xs.view(2, 12, 2), w, ws), want.view(2, 12, 200))
    assert torch.equal(linear_e4m3(x[0], xs[0], w, ws), linear_e4m3(x[:1], xs[:1], w, ws)[0])
    assert torch.equal(linear_e4m3(x, xs.t().contiguous().t(), w, ws.t().contiguous().t()), want)
    back = torch.zeros(200 * 256 + 8, dtype=torch.uint8, device="cuda")
    back[8:] = w.view(torch.uint8).view(-1)
    assert torch.equal(linear_e4m3(x, xs, back[8:].view(torch.float8_e4m3fn).view(200, 256), ws), want)
    assert linear_e4m3(x[:0], xs[:0], w, ws).shape == (0, 200)


def test_bad_ends_are_reported_and_stay_in_bounds():
    x, xs, w, ws = _operands(50, 160, 128, 3)
    for ends in ([10, 5, 50], [10, 20, 51], [-1, 20, 50], [2 ** 31 - 1, -2 ** 31, 7]):
        out = linear_e4m3(x, xs, w, ws, ends=torch.tensor(ends, dtype=torch.int32, device="cuda"))
        assert out.shape == (50, 160)
        with pytest.raises(RuntimeError, match="104"):
            torch.cuda.synchronize()
            linear_e4m3(x, xs, w, ws, ends=torch.tensor([10, 20, 50], dtype=torch.int32, device="cuda"))
    want = linear_e4m3(x, xs, w, ws, ends=torch.tensor([10, 20, 50], dtype=torch.int32, device="cuda"))
    ops.check_status()
    assert bool(want.isfinite().all())


def test_same_bits_in_graphs_with_other_ends():
    x, xs, w, ws = _operands(300, 512, 1024, 6)
    ends = torch.tensor([10, 20, 20, 150, 280, 300], dtype=torch.int32, device="cuda")
    other = torch.tensor([0, 200, 220, 250, 280, 290], dtype=torch.int32, device="cuda")
    want, want_other = (linear_e4m3(x, xs, w, ws, ends=e) for e in (ends, other))
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(linear_e4m3(x, xs, w, ws, ends=ends))
    for g in graphs:
        g.replay()
    assert all(torch.equal(o, want) for o in outs)
    ends.copy_(other)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graphs[1].replay()
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want_other) for o in outs)
    ops.check_status()


@pytest.mark.parametrize("rows,N,K,experts", [(1, 1000, 1040, None), (2, 4096, 1024, None), (60, 700, 2048, None), (3, 300, 512, 4), (100, 4096, 512, 16)])
def test_calls_of_few_rows_in_graphs(rows, N, K, experts):
    x, xs, w, ws = _operands(rows, N, K, experts)
    ends = None if experts is None else torch.linspace(0, rows, experts + 1)[1:].int().cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = linear_e4m3(x, xs, w, ws, ends=ends)
    for seed in range(3):
        other = _operands(rows, N, K, experts, seed)
        for a, b in zip((x, xs, w, ws), other):
            a.copy_(b)
        graph.replay()
        assert torch.equal(out, linear_e4m3(*other, ends=ends))


def test_one_row_with_values_that_are_not_finite():
    x, xs, w, ws = _operands(1, 400, 384)
    want = linear_e4m3(x, xs, w, ws)
    w.view(torch.uint8)[7, 300] = 0x7f
    ws[2, 1] = float("inf")
    out = linear_e4m3(x, xs, w, ws)[0]
    bad = torch.zeros(400, dtype=torch.bool, device="cuda")
    bad[7] = bad[256:384] = True
    assert torch.equal(out[~bad], want[0, ~bad]) and not bool(out[bad].isfinite().any())


def test_outputs_beyond_32_bits():
    rows, N, K = 70000, 32768, 16
    x, xs, w, ws = _operands(rows, N, K)
    out = linear_e4m3(x, xs, w, ws)
    for at in (slice(0, 3), slice(rows - 3, rows)):
        _check(out[at], x[at], xs[at], w, ws)
    del out
    x = torch.zeros(2 ** 20 + 3, 2064, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    xs = torch.ones(2 ** 20 + 3, 17, device="cuda")
    x[-2:] = torch.randn(2, 2064, device="cuda").to(torch.float8_e4m3fn)
    w, ws = quantize_e4m3(torch.randn(64, 2064, device="cuda"), 128)
    _check(linear_e4m3(x, xs, w, ws)[-2:], x[-2:], xs[-2:], w, ws)


def test_norm_quantised_into_the_experts_products():
    """The chain as a model runs it: residual and norm, the experts' product of its 8-bit rows, and back to a row of 8 bits."""
    D, H, sizes = 512, 768, [30, 0, 97, 1]
    rows = sum(sizes)
    x, res = (torch.randn(rows, D, device="cuda").bfloat16() for _ in range(2))
    w, ws = quantize_e4m3(torch.randn(4, H, D, device="cuda") * D ** -0.5, 128)
    down, down_s = quantize_e4m3(torch.randn(4, D, H, device="cuda") * H ** -0.5, 128)
    ends = torch.tensor(sizes).cumsum(0).int().cuda()
    q, s, h = rms_norm(x, torch.ones(D, device="cuda"), residual=res, quantize=True)
    up = linear_e4m3(q, s, w, ws, ends=ends)
    q2, s2 = quantize_e4m3(up)
    out = linear_e4m3(q2, s2, down, down_s, ends=ends, out_dtype=torch.float32)
    begin = 0
    for e, n in enumerate(sizes):
        at = slice(begin, begin + n)
        _check(up[at], q[at], s[at], w[e], ws[e])
        _check(out[at], q2[at], s2[at], down[e], down_s[e])
        # against the product in full precision: a step of e4m3 on each of four operands, roots of sums of independent errors
        want = torch.nn.functional.rms_norm(h[at].double(), (D,), eps=1e-6) @ _wide(w[e], ws[e], 128).t()
        assert n == 0 or float((up[at].double() - want).norm() / want.norm()) < 2.0 ** -4
        begin += n


def test_experts_of_a_layer_by_their_products():
    """Router, rows by expert, gated activation and weighted sum as the documentation has them: `ends` from the sorted experts, each product as above."""
    T, D, H, experts, k = 150, 256, 320, 6, 2
    g = torch.Generator(device="cuda").manual_seed(0)
    y, stream = (torch.randn(T, D, device="cuda", generator=g).bfloat16() for _ in range(2))
    up, up_scale = quantize_e4m3(torch.randn(experts, 2 * H, D, device="cuda", generator=g) * D ** -0.5, block_rows=128)
    down, down_scale = quantize_e4m3(torch.randn(experts, D, H, device="cuda", generator=g) * H ** -0.5, block_rows=128)
    logits = torch.randn(T, experts, device="cuda", generator=g)
    logits[:, 3] -= 100   # an expert without rows
    share, chosen = torch.topk(logits.softmax(-1), k)
    x, x_scale, stream = rms_norm(y, torch.ones(D, device="cuda"), residual=stream, quantize=True)
    expert, order = chosen.flatten().sort(stable=True)
    ends = torch.searchsorted(expert, torch.arange(experts, device="cuda"), right=True).int()
    token = order // k
    both = linear_e4m3(x[token], x_scale[token], up, up_scale, ends=ends)
    gate, value = both.chunk(2, -1)
    hidden = quantize_e4m3(torch.nn.functional.silu(gate) * value)
    out = linear_e4m3(*hidden, down, down_scale, ends=ends, out_dtype=torch.float32)
    result = torch.zeros(T, D, device="cuda").index_add_(0, token, out * share.flatten()[order, None])
    want = torch.zeros(T, D, dtype=torch.float64, device="cuda")
    begin = 0
    for e, end in enumerate(ends.tolist()):
        at = slice(begin, end)
        rows = torch.nonzero((chosen == e).any(1))[:, 0]
        assert torch.equal(token[at], rows) and (e != 3 or begin == end)
        _check(both[at], x[rows], x_scale[rows], up[e], up_scale[e])
        _check(out[at], hidden[0][at], hidden[1][at], down[e], down_scale[e])
        want[rows] += out[at].double() * share.double()[chosen == e][:, None]
        begin = end
    assert begin == T * k
    # a product and a sum in fp32 for each of two experts
    size = torch.zeros(T, D, dtype=torch.float64, device="cuda").index_add_(0, token, (out.double() * share.double().flatten()[order, None]).abs())
    assert bool(((result.double() - want).abs() <= 4 * 2.0 ** -24 * size).all())
