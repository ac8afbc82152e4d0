"""GPU: the RMS norm, the 8-bit products and clipping among torch's other ways of calling: refusals, saved-tensor hooks, captures and streams, and
a training step of them together, captured and replayed."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from flashfusedmoe_b200 import (AdamW, MoELayer, RMSNorm, clip_coefficient, clip_grad_norm, linear_cross_entropy, linear_e4m3, ops, quantize_e4m3,
                                rms_norm)

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _refused(call, error, match):
    with pytest.raises(error, match=match):
        call()


def test_operands_that_do_not_fit():
    x, w = torch.randn(6, 64, device=DEV).bfloat16(), torch.ones(64, device=DEV)
    for call, error, match in (
            (lambda: rms_norm(x, w[:63]), ValueError, "weight must be"), (lambda: rms_norm(x, w.double()), TypeError, "bfloat16, float16 or float32"),
            (lambda: rms_norm(x.double(), w), TypeError, "bfloat16, float16 or float32"), (lambda: rms_norm(x, w, -1.0), ValueError, "eps"),
            (lambda: rms_norm(x, w, residual=x[:5]), ValueError, "residual must be"), (lambda: rms_norm(x, w, residual=x.float()), TypeError, "x's type"),
            (lambda: rms_norm(x, w, weight_offset=float("inf")), ValueError, "finite"), (lambda: rms_norm(x[0, 0]), ValueError, "last dimension"),
            (lambda: rms_norm(x[:, :40].contiguous(), quantize=True), ValueError, "16 values"),
            (lambda: rms_norm(x, w.requires_grad_(), quantize=True), RuntimeError, "not differentiable"),
            (lambda: rms_norm(torch.zeros(1, 40000, device=DEV)), RuntimeError, "ffm_rms_norm_forward"),
            (lambda: rms_norm(x, w.cpu()), RuntimeError, "no CPU path"), (lambda: rms_norm(x.to_sparse()), ValueError, "dense"),
            (lambda: quantize_e4m3(x, 64), ValueError, "block_rows"), (lambda: quantize_e4m3(x[0], 128), ValueError, "columns"),
            (lambda: quantize_e4m3(x[:, :40]), ValueError, "multiple of 16"), (lambda: quantize_e4m3(x.double()), TypeError, "float32"),
            (lambda: quantize_e4m3(x.float().requires_grad_()), RuntimeError, "not differentiable")):
        _refused(call, error, match)
    q, s = quantize_e4m3(torch.randn(6, 256, device=DEV))
    wq, ws = quantize_e4m3(torch.randn(3, 100, 256, device=DEV), 128)
    ends = torch.tensor([1, 2, 6], dtype=torch.int32, device=DEV)
    for call, error, match in (
            (lambda: linear_e4m3(q.float(), s, wq, ws, ends=ends), TypeError, "x must be float8"),
            (lambda: linear_e4m3(q, s, wq.bfloat16(), ws, ends=ends), TypeError, "weight must be float8"),
            (lambda: linear_e4m3(q, s, wq, ws), ValueError, r"weight must be \[N, K\]"),
            (lambda: linear_e4m3(q, s, wq[0], ws[0], ends=ends), ValueError, "experts, N, K"),
            (lambda: linear_e4m3(q[:, :128], s[:, :1], wq, ws, ends=ends), ValueError, "x must end in 256"),
            (lambda: linear_e4m3(q, s[:, :1], wq, ws, ends=ends), ValueError, "x_scale must be"),
            (lambda: linear_e4m3(q, s, wq, ws[:, :, :1], ends=ends), ValueError, "weight_scale must be"),
            (lambda: linear_e4m3(q, s.double(), wq, ws, ends=ends), TypeError, "x_scale must be float32"),
            (lambda: linear_e4m3(q, s, wq, ws, ends=ends[:2]), ValueError, "ends must be"),
            (lambda: linear_e4m3(q, s, wq, ws, ends=ends.long()), TypeError, "ends must be int32"),
            (lambda: linear_e4m3(q, s, wq, ws, ends=ends.cpu()), RuntimeError, "no CPU path"),
            (lambda: linear_e4m3(q, s, wq, ws, ends=ends, out_dtype=torch.float64), TypeError, "out_dtype"),
            (lambda: linear_e4m3(q[None], s[None], wq, ws, ends=ends), ValueError, "rows belong to experts"),
            (lambda: linear_e4m3(q, s.requires_grad_(), wq, ws, ends=ends), RuntimeError, "not differentiable")):
        _refused(call, error, match)


def test_tangents_traces_and_transforms_are_refused():
    from torch.fx.experimental.proxy_tensor import make_fx
    x, w = torch.randn(4, 64, device=DEV), torch.ones(64, device=DEV)
    q, s = quantize_e4m3(x)
    wq, ws = quantize_e4m3(x, 128)
    linear_e4m3(q, s, wq, ws)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, x)
        for call in (lambda: rms_norm(dual), lambda: rms_norm(x, w, residual=dual), lambda: rms_norm(x, forward_ad.make_dual(w, w)),
                     lambda: quantize_e4m3(dual), lambda: linear_e4m3(q, forward_ad.make_dual(s, s), wq, ws), lambda: clip_coefficient([dual], 1.0)):
            _refused(call, RuntimeError, "forward-mode")
    for call in (lambda a: rms_norm(a, w), lambda a: rms_norm(a, w, residual=a)[0], lambda a: quantize_e4m3(a)[1], lambda a: clip_coefficient([a], 1.0)[0]):
        _refused(lambda: torch.jit.trace(call, x), RuntimeError, "cannot be traced")
        _refused(lambda: make_fx(call)(x), RuntimeError, "cannot be traced")
    _refused(lambda: torch.func.grad(lambda a: rms_norm(a, w).sum())(x), RuntimeError, "functorch")
    _refused(lambda: torch.func.vmap(lambda a: rms_norm(a, w))(x[None]), RuntimeError, "storage")


def test_saved_tensor_hooks():
    x, r, w = (torch.randn(40, 96, device=DEV).bfloat16() for _ in range(3))
    leaves = [x.requires_grad_(), r.requires_grad_(), w[0].clone().requires_grad_()]

    def step(unpack):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            out = rms_norm(x, leaves[2], residual=r)
        return torch.autograd.grad([o.float().square().sum() for o in out], leaves)

    want = step(lambda t: t)
    assert all(torch.equal(a, b) for a, b in zip(step(lambda t: t.clone()), want))
    assert all(torch.equal(a, b) for a, b in zip(step(lambda t: torch.stack((t, t), -1)[..., 0]), want))
    for change in (lambda t: t.cpu(), lambda t: t.double(), lambda t: t[:1]):
        _refused(lambda: step(change), (RuntimeError, TypeError, ValueError), "")


def test_a_capture_beside_an_eager_graph_of_the_same_leaves_is_refused():
    x, w = torch.randn(40, 96, device=DEV).bfloat16().requires_grad_(), torch.ones(96, device=DEV).requires_grad_()
    y, h = rms_norm(x, w, residual=x)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        with pytest.raises(RuntimeError, match="before the capture"):
            rms_norm(x, w, residual=x)
    del y, h
    with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
        sum(rms_norm(x, w, residual=x)).sum().backward()


class Block(torch.nn.Module):
    """A pre-norm residual block, the head's norm with its residual, and the loss."""

    def __init__(self, D, vocab):
        super().__init__()
        self.layer = MoELayer(D, 2 * D, 4, pre_norm="rms", aux_loss_coeff=0.01)
        self.norm = RMSNorm(D)
        self.head = torch.nn.Parameter(torch.randn(vocab, D) * D ** -0.5)

    def forward(self, x, target):
        y, losses = self.layer(x)
        out, _ = self.norm(y, residual=x)
        return linear_cross_entropy(out, self.head, target) + losses["aux_loss"]


@pytest.mark.parametrize("in_place", [True, False])
def test_a_captured_training_step_replays_to_the_eager_bits(in_place):
    D, vocab, steps = 256, 1000, 3
    xs = [torch.randn(300, D, device=DEV).bfloat16() for _ in range(steps)]
    targets = [torch.randint(0, vocab, (300,), device=DEV) for _ in range(steps)]

    def build():
        torch.manual_seed(0)
        model = Block(D, vocab).to(DEV).bfloat16()
        return model, AdamW(model.parameters(), lr=1e-3, state_bits=32)

    def step(model, opt, x, target):
        loss = model(x, target)
        loss.backward()
        if in_place:
            norm = clip_grad_norm(model.parameters(), 0.05)
            opt.step()
        else:
            norm, coefficient = clip_coefficient([p.grad for p in model.parameters()], 0.05)
            opt.step(grad_scale=coefficient)
        opt.zero_grad(set_to_none=False)
        return loss.detach(), norm

    model, opt = build()
    eager = [tuple(float(v) for v in step(model, opt, x, t)) for x, t in zip(xs, targets)]
    want = [p.detach().clone() for p in model.parameters()]
    model, opt = build()
    x, target = xs[0].clone(), targets[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = tuple(float(v) for v in step(model, opt, x, target))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        loss, norm = step(model, opt, x, target)
    got = [first]
    for k in range(1, steps):
        x.copy_(xs[k])
        target.copy_(targets[k])
        graph.replay()
        got.append((float(loss), float(norm)))
    assert got == eager and all(n > 0.05 for _, n in got)
    assert all(torch.equal(p, q) for p, q in zip(model.parameters(), want))


def test_calls_on_two_streams_at_once():
    x, w = torch.randn(2000, 1024, device=DEV).bfloat16(), torch.ones(1024, device=DEV)
    wq, ws = quantize_e4m3(torch.randn(6, 1000, 1024, device=DEV) * 0.03, 128)
    grads = [torch.randn(300000, device=DEV), torch.randn(77, device=DEV).bfloat16()]
    ends = torch.tensor([100, 100, 900, 901, 1500, 1990], dtype=torch.int32, device=DEV)

    def chain(k):
        q, s, h = rms_norm(x[k:], w, residual=x[k:], quantize=True)
        few = linear_e4m3(q[:40], s[:40], wq, ws, ends=(ends // 50).int())
        return [q.view(torch.uint8), s, h, linear_e4m3(q, s, wq, ws, ends=ends.clamp(max=2000 - k)), few, *clip_coefficient(grads, 1.0 + k)]

    want = [chain(k) for k in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for k, side in enumerate(streams):
            with torch.cuda.stream(side):
                got.append(chain(k))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, v in zip(got, want) for a, b in zip(g, v))
    ops.check_status()


def test_a_first_call_cannot_be_captured(monkeypatch):
    x, s = torch.zeros(4, 128, device=DEV).to(torch.float8_e4m3fn), torch.ones(4, 1, device=DEV)
    linear_e4m3(x, s, x, s[:1])
    monkeypatch.setattr(ops, "has_status", lambda device: False)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(RuntimeError, match="first call"):
            linear_e4m3(x, s, x, s[:1])


def test_a_call_that_could_not_report_cannot_be_captured(monkeypatch):
    """The status word alone, as other calls make it, is not enough: without the host word bad ends in a replay would never be reported."""
    q, s = torch.zeros(4, 128, device=DEV).to(torch.float8_e4m3fn), torch.ones(4, 1, device=DEV)
    hidden, target = torch.randn(4, 64, device=DEV).bfloat16(), torch.zeros(4, dtype=torch.int64, device=DEV)

    def calls():
        return (lambda: linear_e4m3(q, s, q, s[:1])), (lambda: linear_cross_entropy(hidden, hidden, target))

    for call in calls():
        call()
    ops.check_status()
    monkeypatch.setattr(ops, "_reported", {})
    for call in calls():
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            with pytest.raises(RuntimeError, match="first call"):
                call()
    x, xs = torch.zeros(50, 128, device=DEV).to(torch.float8_e4m3fn), torch.ones(50, 1, device=DEV)
    w, ws, ends = torch.stack([x, x]), torch.ones(2, 1, 1, device=DEV), torch.tensor([20, 50], dtype=torch.int32, device=DEV)
    linear_e4m3(x, xs, w, ws, ends=ends)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        linear_e4m3(x, xs, w, ws, ends=ends)
    ends.fill_(51)   # past the rows: moved into place, and reported
    graph.replay()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="104"):
        linear_e4m3(x, xs, w, ws)
    ops.check_status()


def test_compiled_functions_call_them_eagerly():
    x, w = torch.randn(40, 128, device=DEV).bfloat16().requires_grad_(), torch.ones(128, device=DEV).requires_grad_()
    wq, ws = quantize_e4m3(torch.randn(64, 128, device=DEV), 128)

    def call(a):
        y, h = rms_norm(a, w, residual=a)
        with torch.no_grad():
            q, s = rms_norm(a, w, quantize=True)
            out = linear_e4m3(q, s, wq, ws)
        return (y + h).sum() + out.sum()

    got, want = torch.compile(call, backend="eager")(x), call(x)
    assert torch.equal(got, want)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, [x, w]), torch.autograd.grad(want, [x, w])))
