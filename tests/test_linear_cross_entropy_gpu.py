"""Linear cross entropy and its gradients against 64-bit evaluations of the formulas.

Bounds, with u = 2^-24. A logit is a sum of D exact products, 16 at a time in fp32: off by (D / 16 + 1) 2^-22 of the sum of
magnitudes A. So is lse, and both are off by 16 u more of themselves. An entry of dl is off by twice the logits' bound times itself, by 2^-11 (the exponential
in fp16) and 2^-8 of itself (dl in bf16), and by 2^-25 of the row's factor where fp16 has nothing left; the target's entry p - 1 by
the logits' bound times the factor and 2^-8 of itself. Those go through the product with the other operand, whose sum of n
terms adds (n / 16 + 1) 2^-22 of the magnitudes, and the result is rounded to its type."""

import pytest
import torch

U = 2.0 ** -24
IGNORE = -100


def inputs(n, d, v, seed=0, ignored=0.0, scale=1.0, sure=6.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = (torch.randn(v, d, device="cuda", generator=g) * d ** -0.5 * scale).bfloat16()
    t = torch.randint(0, v, (n,), device="cuda", generator=g)
    h = (torch.randn(n, d, device="cuda", generator=g) + sure * torch.rand(n, 1, device="cuda", generator=g) * w[t].float()).bfloat16()
    if ignored:
        t = torch.where(torch.rand(n, device="cuda", generator=g) < ignored, IGNORE, t)
    return h, w, t


def reference(h, w, t, z=0.0, ignore=IGNORE, row_grad=None, reduction="mean"):
    h, w = h.double(), w.double()
    n, d = h.shape
    v = w.shape[0]
    counts = t != ignore
    safe = torch.where(counts, t, 0)
    logits = h @ w.t()
    size = (h.abs() @ w.abs().t())
    off = (d / 16 + 1) * 2.0 ** -22 * size.amax(1)
    lse = torch.logsumexp(logits, 1)
    lt = logits.gather(1, safe[:, None])[:, 0]
    out = {"nll": torch.where(counts, lse - lt + z * lse * lse, 0.0)}
    off = off + 16 * U * (1 + lse.abs() + lt.abs())
    bound = {"nll": 2 * off * (1 + 2 * z * lse.abs()) + 4 * U * out["nll"].abs()}
    scale = counts.double()
    if reduction == "mean":
        scale = scale / counts.sum()
    if row_grad is not None:
        scale = scale * row_grad.double()
    out["loss"], bound["loss"] = (scale * out["nll"]).sum(), (scale.abs() * bound["nll"]).sum() + 2 * U * (scale * out["nll"]).sum().abs()
    p = torch.exp(logits - lse[:, None])
    zf = 1 + 2 * z * lse
    dl = p * zf[:, None]
    e = dl.abs() * (2 * off[:, None] + 2.0 ** -11 + 2.0 ** -8) + 2.0 ** -25 * zf.abs()[:, None]
    one = torch.zeros_like(p).scatter_(1, safe[:, None], 1.0)
    dl = dl - one
    e = torch.where(one > 0, dl.abs() * 2.0 ** -8 + (2 * off * (p * one).sum(1) * zf.abs())[:, None] + 16 * U, e)
    dl, e = dl * scale[:, None], e * scale.abs()[:, None] * (1 + 4 * U)
    out["dh"], out["dw"] = dl @ w, dl.t() @ h
    bound["dh"] = e @ w.abs() + (v / 16 + 20) * 2.0 ** -22 * (dl.abs() @ w.abs())
    bound["dw"] = e.t() @ h.abs() + (n / 16 + 20) * 2.0 ** -22 * (dl.abs().t() @ h.abs())
    return out, bound


def check(got, out, bound, name):
    assert got.shape == out[name].shape, (name, got.shape)
    half = torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 0.0
    limit = bound[name] * (1 + half) + half * out[name].abs() + 1e-38
    wrong = ~((got.double() - out[name]).abs() <= limit)
    assert not wrong.any(), (name, wrong.sum().item(), ((got.double() - out[name]).abs() / limit).max().item())


def run(h, w, t, factor=None, **options):
    from flashfusedmoe_b200 import linear_cross_entropy, ops
    h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
    loss = linear_cross_entropy(h, w, t, **options)
    assert loss.dtype == torch.float32
    loss.backward(factor)
    ops.check_status()
    return loss.detach(), h.grad, w.grad


SHAPES = [(1, 8, 1), (3, 64, 2), (7, 64, 127), (130, 64, 128), (129, 72, 129), (257, 136, 1000), (300, 256, 257), (64, 1024, 5003),
          (1000, 128, 777), (513, 264, 4099), (100, 128, 40001), (2048, 64, 300)]


@pytest.mark.gpu
@pytest.mark.parametrize("n,d,v", SHAPES)
@pytest.mark.parametrize("z,ignored", [(0.0, 0.0), (1e-3, 0.4)])
def test_loss_and_gradients(n, d, v, z, ignored):
    from flashfusedmoe_b200 import linear_cross_entropy
    h, w, t = inputs(n, d, v, seed=n + d + v, ignored=ignored)
    t[0] = v - 1
    out, bound = reference(h, w, t, z)
    loss, dh, dw = run(h, w, t, z_loss_coeff=z)
    check(loss, out, bound, "loss")
    check(dh, out, bound, "dh")
    check(dw, out, bound, "dw")
    with torch.no_grad():
        nll = linear_cross_entropy(h, w, t, reduction="none", z_loss_coeff=z)
        check(nll, out, bound, "nll")
        check(linear_cross_entropy(h, w, t, z_loss_coeff=z), out, bound, "loss")


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 2, 5, 8, 9, 16, 17, 31, 33, 64, 65, 128, 129])
@pytest.mark.parametrize("d,v", [(64, 1000), (1024, 5003), (2056, 129)])
def test_scoring_of_a_few_rows(n, d, v):
    from flashfusedmoe_b200 import linear_cross_entropy
    h, w, t = inputs(n, d, v, seed=n, ignored=0.2)
    out, bound = reference(h, w, t, 1e-4)
    with torch.no_grad():
        check(linear_cross_entropy(h, w, t, reduction="none", z_loss_coeff=1e-4), out, bound, "nll")


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["sum", "none"])
def test_other_reductions(reduction):
    h, w, t = inputs(333, 128, 1500, ignored=0.2)
    factor = torch.randn(333, device="cuda") if reduction == "none" else None
    out, bound = reference(h, w, t, 1e-3, row_grad=factor, reduction=reduction)
    loss, dh, dw = run(h, w, t, factor, reduction=reduction, z_loss_coeff=1e-3)
    check(loss, out, bound, "nll" if reduction == "none" else "loss")
    check(dh, out, bound, "dh")
    check(dw, out, bound, "dw")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_pieces_of_rows(dtype):
    """700 rows, 256 at a time: the weight's gradient is summed in fp32; the last piece is not full."""
    h, w, t = inputs(700, 128, 1333, ignored=0.1)
    out, bound = reference(h, w, t)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss, dh, dw = run(h.to(dtype), w.to(dtype), t, _piece_rows=256)
    assert dh.dtype == dw.dtype == dtype
    check(loss, out, bound, "loss")
    check(dh.bfloat16(), out, bound, "dh")
    check(dw, out, bound, "dw")
    whole = run(h, w, t)
    assert torch.equal(loss, whole[0]) and torch.equal(dh.bfloat16(), whole[1])
    from flashfusedmoe_b200 import linear_cross_entropy
    with torch.no_grad():
        nll = linear_cross_entropy(h, w, t, reduction="none")
        assert torch.equal(linear_cross_entropy(h, w, t, reduction="none", _piece_rows=256), nll)
        check(nll, out, bound, "nll")


@pytest.mark.gpu
def test_fp32_operands_under_autocast():
    h, w, t = inputs(200, 64, 500)
    out, bound = reference(h, w, t)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss, dh, dw = run(h.float(), w.float(), t)
        mixed = run(h, w.float(), t)
    assert dh.dtype == dw.dtype == torch.float32 and mixed[1].dtype == torch.bfloat16
    check(loss, out, bound, "loss")
    check(dh.bfloat16(), out, bound, "dh")
    check(dw, out, bound, "dw")   # no rounding to bf16
    assert torch.equal(mixed[2], dw)


@pytest.mark.gpu
def test_large_logits():
    """Logits of hundreds: rows that are certain (their own entry of dl is p - 1 of a p close to 1), and rows that are surely wrong."""
    h, w, t = inputs(256, 128, 2000, scale=8.0, sure=3.0)
    out, bound = reference(h, w, t)
    loss, dh, dw = run(h, w, t)
    assert out["nll"].max() > 30 and out["nll"].min() < 1e-6
    check(loss, out, bound, "loss")
    check(dh, out, bound, "dh")
    check(dw, out, bound, "dw")


@pytest.mark.gpu
def test_rows_that_do_not_count():
    from flashfusedmoe_b200 import linear_cross_entropy
    h, w, t = inputs(100, 64, 300)
    loss, dh, dw = run(h, w, torch.full_like(t, IGNORE))
    assert loss.isnan() and not dh.any() and not dw.any()
    loss, dh, dw = run(h, w, torch.full_like(t, IGNORE), reduction="sum")
    assert loss == 0 and not dh.any() and not dw.any()
    # an entry of the vocabulary as the index to ignore; NaN and infinities in rows that do not count
    t[::3] = 7
    bad = h.clone()
    bad[0], bad[3] = float("nan"), float("inf")
    out, bound = reference(h, w, t, ignore=7)
    loss, dh, dw = run(bad, w, t, ignore_index=7)
    check(loss, out, bound, "loss")
    check(dh, out, bound, "dh")
    assert not dh[::3].any()
    for empty in ("mean", "sum", "none"):
        loss, dh, dw = run(h[:0], w, t[:0], torch.zeros(0, device="cuda") if empty == "none" else None, reduction=empty)
        assert dh.shape == (0, 64) and not dw.any()
        assert loss.isnan() if empty == "mean" else not loss.any()
    with torch.no_grad():
        assert linear_cross_entropy(h[:0], w, t[:0], reduction="none").shape == (0,)


@pytest.mark.gpu
def test_values_that_are_not_finite_stay_in_their_rows():
    from flashfusedmoe_b200 import linear_cross_entropy
    h, w, t = inputs(50, 64, 400)
    out, bound = reference(h, w, t)
    bad = h.clone()
    bad[7, 3], bad[20, 0] = float("nan"), float("inf")
    with torch.no_grad():
        nll = linear_cross_entropy(bad, w, t, reduction="none")
    assert nll[[7, 20]].isnan().all()
    keep = torch.ones(50, dtype=torch.bool, device="cuda")
    keep[[7, 20]] = False
    check(nll[keep], {"nll": out["nll"][keep]}, {"nll": bound["nll"][keep]}, "nll")


@pytest.mark.gpu
def test_a_target_outside_of_the_vocabulary_is_reported():
    from flashfusedmoe_b200 import linear_cross_entropy, ops
    h, w, t = inputs(50, 64, 400)
    out, bound = reference(h, w, t)
    for wrong in (400, -1, 1 << 40):
        bad = t.clone()
        bad[9] = wrong
        leaf = h.detach().requires_grad_()
        nll = linear_cross_entropy(leaf, w, bad, reduction="none")
        nll.backward(torch.ones_like(nll))
        torch.cuda.synchronize()
        assert nll[9].isnan() and not leaf.grad[9].any()
        keep = [i for i in range(50) if i != 9]
        check(nll.detach()[keep], {"nll": out["nll"][keep]}, {"nll": bound["nll"][keep]}, "nll")
        with pytest.raises(RuntimeError, match="104"):
            linear_cross_entropy(h, w, t)
        ops.check_status()


@pytest.mark.gpu
def test_shapes_strides_and_frozen_operands():
    from flashfusedmoe_b200 import linear_cross_entropy
    h, w, t = inputs(120, 64, 300)
    out, bound = reference(h, w, t)
    loss, dh, dw = run(h, w, t)
    other = run(h.view(4, 30, 64), w, t.view(4, 30))
    assert torch.equal(other[0], loss) and torch.equal(other[1], dh.view(4, 30, 64)) and torch.equal(other[2], dw)
    wide = torch.zeros(120, 80, device="cuda").bfloat16()
    wide[:, 8:72] = h
    other = run(wide[:, 8:72], w.t().contiguous().t(), t[None].expand(2, 120)[1])
    assert torch.equal(other[0], loss) and torch.equal(other[1], dh) and torch.equal(other[2], dw)
    for frozen in (0, 1):
        leaves = [h.detach().requires_grad_(frozen != 0), w.detach().requires_grad_(frozen != 1)]
        linear_cross_entropy(*leaves, t).backward()
        assert leaves[frozen].grad is None and torch.equal(leaves[1 - frozen].grad, (dh, dw)[1 - frozen])


@pytest.mark.gpu
def test_factors_and_a_second_backward_pass():
    from flashfusedmoe_b200 import linear_cross_entropy
    h, w, t = inputs(120, 64, 300)
    loss, dh, dw = run(h, w, t)
    h, w = h.requires_grad_(), w.requires_grad_()
    loss = linear_cross_entropy(h, w, t)
    (loss * 0.25).backward(retain_graph=True)
    first = h.grad, w.grad
    assert torch.equal(first[0], dh * 0.25) and torch.equal(first[1], dw * 0.25)
    h.grad = w.grad = None
    (loss * 2.0).backward()
    assert torch.equal(h.grad, dh * 2.0) and torch.equal(w.grad, dw * 2.0) and torch.equal(first[0], dh * 0.25)
    again = run(h, w, t)
    assert torch.equal(again[1], dh) and torch.equal(again[2], dw)
    g, = torch.autograd.grad(linear_cross_entropy(h, w, t), h, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.float().sum().backward()
    loss = linear_cross_entropy(h, w, t, reduction="none")
    with torch.no_grad():
        w.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.sum().backward()


@pytest.mark.gpu
def test_gradient_against_differences():
    """Central differences of the loss along random directions. Steps of 2^-3 of representable numbers; the third derivative along
    a direction of size s is at most s^3, the loss is off by the bound on it."""
    from flashfusedmoe_b200 import linear_cross_entropy
    h, w, t = inputs(16, 64, 200, sure=0.0)
    h, w = (h * 8).round() / 8, (w * 64).round() / 64
    _, dh, dw = run(h, w, t)
    out, bound = reference(h, w, t)
    g = torch.Generator(device="cuda").manual_seed(3)
    for which in (0, 1):
        for _ in range(4):
            x = (h, w)[which]
            step = (torch.randint(0, 3, x.shape, device="cuda", generator=g) - 1).bfloat16() / (8 if which == 0 else 64)
            moved = [(h + s * step, w) if which == 0 else (h, w + s * step) for s in (1, -1)]
            assert torch.equal(moved[0][which] - step, x)   # nothing was rounded
            with torch.no_grad():
                values = [linear_cross_entropy(a, b, t).item() for a, b in moved]
            along = ((dh, dw)[which].double() * step.double()).sum().item()
            size = (step.double().abs() @ w.double().abs().t()).amax().item() if which == 0 else (h.double().abs() @ step.double().abs().t()).amax().item()
            limit = size ** 3 + bound["loss"].item() + (bound[("dh", "dw")[which]] * step.double().abs()).sum().item() + abs(along) * 2.0 ** -7
            assert abs((values[0] - values[1]) / 2 - along) <= limit
            assert abs(along) > 1e-4


@pytest.mark.gpu
def test_captured_and_on_another_stream():
    from flashfusedmoe_b200 import linear_cross_entropy
    h, w, t = inputs(300, 128, 1000)
    h, w = h.requires_grad_(), w.requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(linear_cross_entropy(h, w, t), (h, w))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        loss = linear_cross_entropy(h, w, t)
        grads = torch.autograd.grad(loss, (h, w))
    with torch.no_grad():
        h.copy_(torch.randn_like(h))
        t.copy_(torch.randint_like(t, 0, 1000))
    graph.replay()
    torch.cuda.synchronize()
    eager = run(h, w, t)
    assert torch.equal(loss.detach(), eager[0]) and torch.equal(grads[0], eager[1]) and torch.equal(grads[1], eager[2])


@pytest.mark.gpu
def test_no_matrix_of_logits():
    """Scoring keeps 8 bytes for 128 entries; a training step 2 bytes an entry for one piece of rows and its gradients."""
    from flashfusedmoe_b200 import linear_cross_entropy
    n, d, v = 4096, 64, 50257
    h, w, t = inputs(n, d, v)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with torch.no_grad():
        linear_cross_entropy(h, w, t)
    assert torch.cuda.max_memory_allocated() - before < n * v // 8
    torch.cuda.reset_peak_memory_stats()
    linear_cross_entropy(h.requires_grad_(), w.requires_grad_(), t, _piece_rows=512).backward()
    assert torch.cuda.max_memory_allocated() - before < 512 * v * 4 + v * d * 8 + (8 << 20)


@pytest.mark.gpu
def test_refusals():
    from flashfusedmoe_b200 import linear_cross_entropy
    h, w, t = inputs(10, 64, 30)
    for error, match, args, options in (
            (NotImplementedError, "bfloat16", (h.float(), w, t), {}), (ValueError, "weight must be", (h, w[:, :32], t), {}),
            (ValueError, "target must be", (h, w, t[:5]), {}), (TypeError, "int64", (h, w, t.int()), {}),
            (ValueError, "reduction", (h, w, t), {"reduction": "max"}), (ValueError, "z_loss", (h, w, t), {"z_loss_coeff": -1.0}),
            (ValueError, "multiple of 8", (h[:, :60].contiguous(), w[:, :60].contiguous(), t), {}),
            (RuntimeError, "no CPU path", (h.cpu(), w, t), {}), (RuntimeError, "no CPU path", (h, w, t.cpu()), {})):
        with pytest.raises(error, match=match):
            linear_cross_entropy(*args, **options)
    room = torch.zeros(10 * 64 + 1, device="cuda").bfloat16()
    with pytest.raises(RuntimeError, match="16 bytes|not supported"):
        linear_cross_entropy(room[1:].view(10, 64), w, t)


@pytest.mark.gpu
def test_the_first_call_on_a_device_is_not_captured(monkeypatch):
    from flashfusedmoe_b200 import linear_cross_entropy, ops
    monkeypatch.setattr(ops, "_status", {})
    h, w, t = inputs(10, 64, 30)
    torch.cuda.synchronize()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(RuntimeError, match="cannot be captured"):
            linear_cross_entropy(h, w, t)
    linear_cross_entropy(h, w, t)
    ops.check_status()
