"""Layer norm, forward and backward, against 64-bit evaluations of its formulas.

Bounds, with u = 2^-24 and h = eps / 2 of the type that a result is rounded to: sums of a row go through at most 64 additions
(16 values a thread, 5 exchanges in a warp, 32 warps), so statistics are off by 64 u of the sums of magnitudes, and so is what is
computed from them; a result is then rounded once. Sums over the rows go through at most rows + 64 additions."""

import pytest
import torch

U = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
# one value, a partial chunk, widths on either side of a chunk, a warp's row, two warps, odd ones, the benchmark's, wide ones with
# four chunks a thread, the widest
WIDTHS = [1, 7, 8, 33, 64, 255, 256, 257, 264, 520, 1024, 2051, 4096, 7168, 8193, 16384]


def reference(x, w, b, eps, dy=None):
    x, w = x.double(), torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if w is None else w.double()
    mu = x.mean(-1, keepdim=True)
    r = 1.0 / ((x - mu).square().mean(-1, keepdim=True) + eps).sqrt()
    xh = (x - mu) * r
    size = (x.abs() + x.abs().mean(-1, keepdim=True)) * r      # what xh is the difference of
    off = 64 * U * size + 64 * U * xh.abs()                    # of xh
    out = {"y": xh * w + (0.0 if b is None else b.double())}
    bound = {"y": off * w.abs() + 4 * U * out["y"].abs()}
    if dy is not None:
        dy = dy.double()
        g = dy * w
        s1, s2 = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
        a1, a2 = g.abs().mean(-1, keepdim=True), (g * xh).abs().mean(-1, keepdim=True)
        out["dx"] = r * (g - s1 - xh * s2)
        bound["dx"] = r * (64 * U * (g.abs() + a1 + xh.abs() * a2) + off * a2 + xh.abs() * (g.abs() * off).mean(-1, keepdim=True))
        n = dy.reshape(-1, dy.shape[-1])
        rows = n.shape[0]
        flat, foff = xh.reshape(n.shape), off.reshape(n.shape)
        out["dw"], out["db"] = (n * flat).sum(0), n.sum(0)
        bound["dw"] = (rows + 64) * U * (n * flat).abs().sum(0) + (n.abs() * foff).sum(0)
        bound["db"] = (rows + 64) * U * n.abs().sum(0)
    return out, bound


def check(got, out, bound, name):
    assert got.shape == out[name].shape
    half = torch.finfo(got.dtype).eps / 2
    smallest = torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps
    limit = bound[name] * (1 + half) + half * out[name].abs() + smallest
    wrong = (got.double() - out[name]).abs() > limit
    assert not wrong.any(), (name, wrong.sum().item(), ((got.double() - out[name]).abs() / limit).max().item())


def inputs(rows, width, dtype, seed, offset=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, width, device="cuda", generator=g) * 2 + 0.5 + offset).to(dtype)
    w = (1 + 0.3 * torch.randn(width, device="cuda", generator=g)).to(dtype)
    b = (0.3 * torch.randn(width, device="cuda", generator=g)).to(dtype)
    dy = torch.randn(rows, width, device="cuda", generator=g).to(dtype)
    return x, w, b, dy


def run(x, w, b, dy, eps=1e-5):
    from flashfusedmoe_b200 import layer_norm
    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, w, b)]
    y = layer_norm(*leaves, eps)
    assert y.dtype == x.dtype and y.is_contiguous()
    y.backward(dy)
    return y.detach(), [None if t is None else t.grad for t in leaves]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_forward_and_backward(width, dtype):
    for rows in (1, 37, 1500 if width <= 1024 else 300):
        x, w, b, dy = inputs(rows, width, dtype, width + rows)
        out, bound = reference(x, w, b, 1e-5, dy)
        y, (dx, dw, db) = run(x, w, b, dy)
        for got, name in ((y, "y"), (dx, "dx"), (dw, "dw"), (db, "db")):
            check(got, out, bound, name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [8, 64, 256, 264, 1024, 1400, 4096, 8192, 1, 2, 9, 33, 127, 255, 257, 511, 1023, 2051, 4099, 7001])
def test_many_rows(width, dtype):
    """More rows than the device has teams for: several of them one after the other, the last round not full."""
    rows = 148 * 1024 // min(1024, max(1, width // 32)) * 3 + 5
    x, w, b, dy = inputs(rows, width, dtype, width)
    out, bound = reference(x, w, b, 1e-5, dy)
    y, (dx, dw, db) = run(x, w, b, dy)
    for got, name in ((y, "y"), (dx, "dx"), (dw, "dw"), (db, "db")):
        check(got, out, bound, name)
    again, grads = run(x, w, b, dy)
    assert torch.equal(y, again) and all(torch.equal(p, q) for p, q in zip((dx, dw, db), grads))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("room,start", [(1040, 8), (1040, 1), (1037, 5), (1025, 0), (1026, 2)])
def test_many_rows_with_a_distance(room, start, dtype):
    base = torch.randn(9000, room, device="cuda").to(dtype)
    x, (_, w, b, dy) = base[:, start:start + 1024], inputs(9000, 1024, dtype, 21)
    out, bound = reference(x, w, b, 1e-5, dy)
    y, (dx, dw, db) = run(x, w, b, dy)
    for got, name in ((y, "y"), (dx, "dx"), (dw, "dw"), (db, "db")):
        check(got, out, bound, name)


@pytest.mark.gpu
def test_widest_rows():
    for width, dtype in ((32768, torch.bfloat16), (20001, torch.float16), (16384, torch.float32), (9000, torch.float32)):
        x, w, b, dy = inputs(5, width, dtype, 3)
        out, bound = reference(x, w, b, 1e-5, dy)
        y, (dx, dw, db) = run(x, w, b, dy)
        for got, name in ((y, "y"), (dx, "dx"), (dw, "dw"), (db, "db")):
            check(got, out, bound, name)


@pytest.mark.gpu
@pytest.mark.parametrize("w_type,b_type", [(torch.float32, torch.float32), (None, torch.bfloat16), (torch.float16, None), (None, None)])
def test_vectors_of_other_types_or_absent(w_type, b_type):
    x, w, b, dy = inputs(65, 520, torch.bfloat16, 5)
    w, b = w if w_type is None else w.to(w_type), b if b_type is None else b.to(b_type)
    w, b = None if w_type is None else w, None if b_type is None else b
    out, bound = reference(x, w, b, 1e-5, dy)
    y, grads = run(x, w, b, dy)
    check(y, out, bound, "y")
    for got, name in zip(grads, ("dx", "dw", "db")):
        if got is not None:
            check(got, out, bound, name)
            assert name == "dx" or got.dtype == (w_type if name == "dw" else b_type)


@pytest.mark.gpu
def test_a_mean_far_from_zero_keeps_the_variance():
    """Differences of squared sums would have nothing left at 4096 with a spread of 2."""
    x, w, b, dy = inputs(64, 1024, torch.float32, 7, offset=4096.0)
    out, bound = reference(x, w, b, 1e-5, dy)
    y, (dx, dw, db) = run(x, w, b, dy)
    for got, name in ((y, "y"), (dx, "dx"), (dw, "dw"), (db, "db")):
        check(got, out, bound, name)


@pytest.mark.gpu
def test_strides_and_addresses():
    """Rows further apart than their width, rows that start off a 16-byte boundary, transposed and expanded inputs."""
    base = torch.randn(3, 40, 2, 272, device="cuda").bfloat16()
    w, b = torch.randn(256, device="cuda").bfloat16(), torch.randn(256, device="cuda").bfloat16()
    views = [base[:, :, 0, :256], base[:, :, 1, 8:264], base[:, :, 0, 1:257], base[0, :, :, 3:259].transpose(0, 1),
             base[:, ::3, 1, :256], base[:1, :1, 0, :256].expand(4, 5, 256), base.permute(3, 1, 2, 0)[:256].permute(3, 1, 2, 0)]
    for x in views:
        dy = torch.randn(x.shape, device="cuda").bfloat16()
        out, bound = reference(x, w, b, 1e-5, dy)
        y, (dx, dw, db) = run(x, w, b, dy)
        for got, name in ((y, "y"), (dx, "dx"), (dw, "dw"), (db, "db")):
            check(got, out, bound, name)
    # a weight that starts off the boundary, an expanded gradient
    x, big = base[0, :, 0, :256], torch.randn(600, device="cuda").bfloat16()
    dy = torch.randn((), device="cuda").bfloat16().expand(x.shape)
    out, bound = reference(x, big[1:257], big[303:559], 1e-5, dy)
    y, (dx, dw, db) = run(x, big[1:257], big[303:559], dy)
    for got, name in ((y, "y"), (dx, "dx"), (dw, "dw"), (db, "db")):
        check(got, out, bound, name)


@pytest.mark.gpu
def test_constant_rows_infinities_and_nan_stay_in_their_rows():
    x, w, b, dy = inputs(9, 384, torch.float32, 11)
    x[1] = 3.0
    x[3, 5] = float("inf")
    x[4, 100] = float("nan")
    out, bound = reference(x, w, b, 1e-5, dy)
    y, (dx, dw, db) = run(x, w, b, dy)
    rest = [0, 1, 2, 5, 6, 7, 8]
    for got, name in ((y, "y"), (dx, "dx")):
        check(got[rest], {name: out[name][rest]}, {name: bound[name][rest]}, name)
        assert got[[3, 4]].isnan().any(dim=1).all()
    assert torch.equal(y[1], b)


@pytest.mark.gpu
def test_no_rows_give_zero_sums():
    x, w, b, dy = inputs(0, 64, torch.bfloat16, 1)
    y, (dx, dw, db) = run(x, w, b, dy)
    assert y.shape == dx.shape == (0, 64) and not dw.any() and not db.any()


@pytest.mark.gpu
def test_only_wanted_gradients_and_equal_bits():
    from flashfusedmoe_b200 import layer_norm
    x, w, b, dy = inputs(777, 1024, torch.bfloat16, 13)
    y, (dx, dw, db) = run(x, w, b, dy)
    again, grads = run(x, w, b, dy)
    assert torch.equal(y, again) and all(torch.equal(p, q) for p, q in zip((dx, dw, db), grads))
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b), y)
    for mask in range(1, 8):
        leaves = [t.detach().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, w, b))]
        layer_norm(*leaves).backward(dy)
        for i, (leaf, full) in enumerate(zip(leaves, (dx, dw, db))):
            assert (leaf.grad is None) == (mask >> i & 1 == 0) and (leaf.grad is None or torch.equal(leaf.grad, full))


@pytest.mark.gpu
def test_gradient_against_differences():
    """Central differences of the forward pass in fp32: the truncation is h^2 / 6 of the third derivative (of size 1 here), the
    forward's rounding 2^-20 of the loss's terms over h."""
    from flashfusedmoe_b200 import layer_norm
    x, w, b, dy = inputs(3, 40, torch.float32, 17)
    _, (dx, dw, db) = run(x, w, b, dy)
    h = 2.0 ** -6
    terms = (layer_norm(x, w, b).double() * dy.double()).abs().sum().item()
    for leaf, grad in ((x, dx), (w, dw), (b, db)):
        flat = leaf.view(-1)
        for i in range(0, flat.numel(), 7):
            keep = flat[i].item()
            values = []
            for step in (h, -h):
                flat[i] = keep + step
                values.append((layer_norm(x, w, b).double() * dy.double()).sum().item())
            flat[i] = keep
            assert abs((values[0] - values[1]) / (2 * h) - grad.view(-1)[i].item()) <= h * h * 8 + 2.0 ** -20 * terms / h


@pytest.mark.gpu
def test_captured_and_on_another_stream():
    from flashfusedmoe_b200 import layer_norm
    x, w, b, dy = inputs(513, 1024, torch.bfloat16, 19)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    with torch.cuda.stream(side):
        for _ in range(2):
            layer_norm(*leaves).backward(dy)
            for t in leaves:
                t.grad = None
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = layer_norm(*leaves)
        grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        x.copy_(torch.randn_like(x))
        dy.copy_(torch.randn_like(dy))
    graph.replay()
    torch.cuda.synchronize()
    eager, full = run(x, w, b, dy)
    assert torch.equal(y, eager) and all(torch.equal(p, q) for p, q in zip(grads, full))


@pytest.mark.gpu
def test_layer_with_a_norm_in_front():
    """MoELayer(pre_norm=True)(x) is the layer of norm(x), gradients included, bit for bit; its parameters are dense ones."""
    from flashfusedmoe_b200 import LayerNorm, MoELayer, get_dense_params
    torch.manual_seed(0)
    layer = MoELayer(128, 256, 4, top_k=2, aux_loss_coeff=0.01, pre_norm=True).cuda().bfloat16()
    plain = MoELayer(128, 256, 4, top_k=2, aux_loss_coeff=0.01).cuda().bfloat16()
    norm = LayerNorm(128).cuda().bfloat16()
    with torch.no_grad():
        layer.norm.weight.normal_(1.0, 0.2)
        layer.norm.bias.normal_(0.0, 0.2)
    state = layer.state_dict()
    norm.load_state_dict({k[5:]: state.pop(k) for k in ("norm.weight", "norm.bias")})
    plain.load_state_dict(state)
    x = torch.randn(2, 50, 128, device="cuda").bfloat16()
    a, c = x.clone().requires_grad_(), x.clone().requires_grad_()
    out, losses = layer(a)
    other, others = plain(norm(c))
    assert torch.equal(out, other) and torch.equal(losses["aux_loss"], others["aux_loss"])
    (out.float().square().sum() + losses["aux_loss"]).backward()
    (other.float().square().sum() + others["aux_loss"]).backward()
    assert torch.equal(a.grad, c.grad)
    assert torch.equal(layer.norm.weight.grad, norm.weight.grad) and torch.equal(layer.norm.bias.grad, norm.bias.grad)
    assert any(p is layer.norm.weight for p in get_dense_params(layer))


@pytest.mark.gpu
def test_refusals():
    from flashfusedmoe_b200 import layer_norm
    x, w, b, _ = inputs(4, 64, torch.bfloat16, 1)
    with pytest.raises(TypeError, match="bfloat16, float16 or float32"):
        layer_norm(x.double(), w, b)
    with pytest.raises(ValueError, match=r"weight must be \[64\]"):
        layer_norm(x, w[:32], b)
    with pytest.raises(RuntimeError, match="no CPU path"):
        layer_norm(x, w.cpu(), b)
    with pytest.raises(ValueError, match="eps"):
        layer_norm(x, w, b, -1.0)
    with pytest.raises(RuntimeError, match="not supported"):
        layer_norm(torch.zeros(1, 32776, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="last dimension"):
        layer_norm(x[0, 0])


@pytest.mark.gpu
def test_a_recorded_backward_pass_refuses_a_second_derivative():
    from flashfusedmoe_b200 import layer_norm, ops
    x, w, b, dy = inputs(4, 64, torch.float32, 1)
    out, bound = reference(x, w, b, 1e-5, dy)
    x = x.requires_grad_()
    before = ops.operator_launches()
    grad, = torch.autograd.grad(layer_norm(x, w, b), x, dy, create_graph=True)
    assert ops.operator_launches() == before + 2
    check(grad.detach(), out, bound, "dx")
    with pytest.raises(RuntimeError, match="twice"):
        grad.sum().backward()


@pytest.mark.gpu
def test_saved_input_may_not_change():
    from flashfusedmoe_b200 import layer_norm
    x, w, b, dy = inputs(4, 64, torch.float32, 1)
    w.requires_grad_()
    y = layer_norm(x, w, b)
    x.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dy)


@pytest.mark.gpu
def test_a_capture_beside_an_eager_graph_of_the_same_leaves_is_refused():
    """The gradients of such leaves would be added on the default stream, which takes no part in the capture."""
    from flashfusedmoe_b200 import layer_norm, linear_cross_entropy
    x = torch.randn(40, 64, device="cuda").bfloat16()
    w = torch.randn(64, device="cuda", requires_grad=True)
    head = torch.randn(100, 64, device="cuda").bfloat16().requires_grad_()
    t = torch.randint(0, 100, (40,), device="cuda")
    side = torch.cuda.Stream()
    for call, leaf in ((lambda: layer_norm(x, w).float().sum(), w), (lambda: linear_cross_entropy(x, head, t), head)):
        eager = call()
        want, = torch.autograd.grad(eager, leaf, retain_graph=True)
        torch.cuda.synchronize()
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            with pytest.raises(RuntimeError, match="before the capture"):
                call()
            with torch.no_grad():
                call()
        del eager
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got, = torch.autograd.grad(call(), leaf)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
