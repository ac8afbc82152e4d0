"""GPU: the norm of all gradients and clipping by it against sums in 64 bits.

Eight squares are added in fp32 (8 half steps of 2^-24, relative, since all are positive), those sums in fp64; the root halves that, and the
result is rounded once: 5 half steps for the norm, and two more for the coefficient."""

import os

import pytest
import torch

from flashfusedmoe_b200 import AdamW, MoELayer, clip_coefficient, clip_grad_norm, linear_cross_entropy, rms_norm

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
INF = float("inf")


def _grads(sizes, dtype, scale=1.0):
    return [(torch.randn(n, device="cuda") * scale * (1 + i)).to(dtype) for i, n in enumerate(sizes)]


def _norm(grads, kind=2.0):
    if kind == INF:
        return max(float(g.abs().max()) for g in grads if g.numel())
    return float(torch.stack([g.double().square().sum() for g in grads]).sum().sqrt())


def _near(got, want, halves):
    assert got.dtype == torch.float32 and got.dim() == 0 and got.is_cuda
    assert abs(float(got) - want) <= halves * 2.0 ** -24 * want, (float(got), want)


def _params(grads):
    params = [torch.nn.Parameter(torch.zeros(g.shape, dtype=g.dtype, device=g.device)) for g in grads]
    for p, g in zip(params, grads):
        p.grad = g
    return params


SIZES = [[1], [7], [16384], [5, 0, 4097, 33], [1000003], [3] * 700, [100] * 33 + [70000], [2 ** 22 + 5, 1, 12345]]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("kind", [2.0, INF])
def test_norm_and_coefficient(sizes, dtype, kind):
    grads = _grads(sizes, DTYPES[dtype], 0.01)
    want = _norm(grads, kind)
    for limit in (0.0, want / 3, want * 2, INF):
        norm, coefficient = clip_coefficient(grads, limit, kind)
        _near(norm, want, 5 if kind == 2.0 else 0)
        _near(coefficient, min(1.0, limit / (want + 1e-6)), 7)
    assert float(clip_coefficient(grads, want * 2, kind)[1]) == 1.0


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("sizes", SIZES)
def test_clipping_in_place(sizes, dtype):
    grads = _grads(sizes, DTYPES[dtype], 0.01)
    params, before = _params(grads), [g.clone() for g in grads]
    norm, coefficient = clip_coefficient(grads, 0.3 * _norm(grads))
    versions = [g._version for g in grads]
    assert torch.equal(clip_grad_norm(params, 0.3 * _norm(grads)), norm)
    # one product in fp32, rounded once
    assert all(torch.equal(p.grad, (b.float() * coefficient).to(b.dtype)) for p, b in zip(params, before))
    assert all(g._version > v for g, v in zip(grads, versions) if g.numel())
    after = [g.clone() for g in grads]
    clip_grad_norm(params, 1e9)
    assert all(torch.equal(a, g) for a, g in zip(after, grads))


def test_mixed_types_shapes_and_orders():
    base = torch.randn(64, 96, device="cuda")
    grads = [base[:, :50], base.new_empty(1, 8).bfloat16().normal_(), torch.randn(3, 5, 7, device="cuda").half().permute(2, 0, 1),
             torch.randn(40, 40, device="cuda")[::2], torch.randn((), device="cuda"), torch.randn(33, device="cuda").bfloat16()[1:]]
    before, untouched = [g.clone() for g in grads], base[:, 50:].clone()
    params = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
    for p, g in zip(params, grads):
        p.grad = g
    norm, coefficient = clip_coefficient([p.grad for p in params], 1.0)
    _near(norm, _norm(before), 5)
    clip_grad_norm(iter(params), 1.0)
    assert all(torch.equal(p.grad, (b.float() * coefficient).to(b.dtype)) for p, b in zip(params, before))
    assert torch.equal(base[:, 50:], untouched)


def test_columns_of_one_buffer():
    base = torch.randn(64, 96, device="cuda")
    before, params = base.clone(), _params([base[:, :50], base[:, 50:]])
    norm, coefficient = clip_coefficient([p.grad for p in params], 1.0)
    _near(norm, _norm([before]), 5)
    clip_grad_norm(params, 1.0)
    assert torch.equal(base, before * coefficient)


@pytest.mark.parametrize("dtype,scale", [("fp32", 1e25), ("bf16", 1e30), ("fp32", 1e-25), ("bf16", 1e-38), ("fp16", 6e-8), ("fp32", 1e-42)])
def test_values_whose_squares_leave_fp32(dtype, scale):
    grads = [(torch.randn(5000, device="cuda").double() * scale).to(DTYPES[dtype])]
    want = _norm(grads)
    norm, coefficient = clip_coefficient(grads, 0.5 * want)
    assert abs(float(norm) - want) <= 5 * 2.0 ** -24 * want + 2.0 ** -150
    mixed = [torch.full((9,), 1e-25, device="cuda"), torch.full((9,), 1e20, device="cuda"), torch.zeros(1000, device="cuda")]
    _near(clip_coefficient(mixed, 1.0)[0], _norm(mixed), 5)


@pytest.mark.parametrize("kind", [2.0, INF])
def test_values_that_are_not_finite(kind):
    for bad in (float("nan"), INF, -INF):
        grads = [torch.ones(5000, device="cuda"), torch.ones(3, device="cuda").bfloat16(), torch.ones(70000, device="cuda")]
        grads[0][4321] = bad
        params, theirs = _params([g.clone() for g in grads]), _params([g.clone() for g in grads])
        want = torch.nn.utils.clip_grad_norm_(theirs, 1.0, kind)
        norm, coefficient = clip_coefficient(grads, 1.0, kind)
        assert norm.isnan() == want.isnan() and norm.isinf() == want.isinf()
        assert bool(coefficient.isnan()) if bad != bad else float(coefficient) == 0.0
        with pytest.raises(RuntimeError, match="not finite"):
            clip_grad_norm(params, 1.0, kind, error_if_nonfinite=True)
        assert all(torch.equal(p.grad, g) or bad != bad for p, g in zip(params, grads))
        clip_grad_norm(params, 1.0, kind)
        for p, t in zip(params, theirs):
            assert torch.equal(p.grad.isnan(), t.grad.isnan()) and torch.equal(p.grad.nan_to_num(), t.grad.nan_to_num())


def test_as_torchs():
    grads = _grads([3000, 17, 40000], torch.float32)
    params, theirs = _params([g.clone() for g in grads]), _params([g.clone() for g in grads])
    want = torch.nn.utils.clip_grad_norm_(theirs, 2.5)
    _near(clip_grad_norm(params, 2.5), float(want), 30)
    # either norm is off by some half steps, and so are the coefficients
    assert all(torch.allclose(p.grad, t.grad, rtol=40 * 2.0 ** -24, atol=0) for p, t in zip(params, theirs))
    assert float(clip_grad_norm(params[0], 1e9)) > 0
    unused = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    assert float(clip_grad_norm([unused], 1.0)) == 0.0 and float(clip_grad_norm([], 1.0)) == 0.0


def test_refusals():
    g = torch.randn(100, device="cuda")
    with pytest.raises(ValueError, match="appears twice"):
        clip_grad_norm(_params([g, g]), 1.0)
    p = torch.nn.Parameter(torch.zeros(60, device="cuda"))
    p.grad = g[:60]
    q = torch.nn.Parameter(torch.zeros(50, device="cuda"))
    q.grad = g[50:]
    with pytest.raises(ValueError, match="appears twice"):
        clip_grad_norm([p, q], 1.0)
    p = torch.nn.Parameter(torch.zeros(4, 5, device="cuda"))
    p.grad = torch.randn(5, device="cuda").expand(4, 5)
    with pytest.raises(ValueError, match="expanded"):
        clip_grad_norm([p], 1.0)
    _near(clip_coefficient([p.grad], 1.0)[0], _norm([p.grad]), 5)
    with pytest.raises(TypeError, match="bfloat16, float16 or float32"):
        clip_coefficient([g.double()], 1.0)
    with pytest.raises(RuntimeError, match="no CPU path"):
        clip_coefficient([g, g.cpu()], 1.0)
    with pytest.raises(ValueError, match="dense"):
        clip_coefficient([g.to_sparse()], 1.0)


def test_captured_steps_do_not_share_anything():
    grads = _grads([30000, 77], torch.bfloat16)
    first, second = _params([g.clone() for g in grads]), _params([g.clone() * 2 for g in grads])
    graphs, norms = [], []
    for params in (first, second):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            norms.append(clip_grad_norm(params, 1.0))
    want = []
    for params, k in ((first, 1), (second, 2)):
        for p, g in zip(params, grads):
            p.grad.copy_(g * k)
        want.append(_norm([p.grad for p in params]))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for g, s in zip(graphs, streams):   # at the same time
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    for n, w in zip(norms, want):
        _near(n, w, 5)
    for params in (first, second):
        # every value is off by half a step of bfloat16
        assert abs(_norm([p.grad for p in params]) - 1.0) < 2.0 ** -8


def test_sharded_gradients_over_a_group_of_one():
    import torch.distributed as dist
    if dist.is_initialized():
        pytest.skip("a process group is there")
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT="29541")
    dist.init_process_group("nccl", rank=0, world_size=1, device_id=torch.device("cuda", 0))
    try:
        grads = _grads([3000, 17, 40000], torch.bfloat16)
        for kind in (2.0, INF):
            want = clip_coefficient(grads, 1.0, kind)
            got = clip_coefficient(grads[:1], 1.0, kind, sharded=grads[1:], group=dist.group.WORLD)
            # the sum of squares is added up in another order, in fp64
            _near(got[0], float(want[0]), 1)
            _near(got[1], float(want[1]), 1)
        params = _params([g.clone() for g in grads])
        _near(clip_grad_norm(params, 1.0, sharded=params[1:], group=dist.group.WORLD), _norm(grads), 5)
        none = [torch.nn.Parameter(torch.zeros(3, device="cuda"))]
        assert float(clip_grad_norm(none, 1.0, sharded=none, group=dist.group.WORLD)) == 0.0
    finally:
        dist.destroy_process_group()


def test_a_group_of_one_without_gradients_and_with_a_nan():
    import torch.distributed as dist
    if dist.is_initialized():
        pytest.skip("a process group is there")
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT="29543")
    dist.init_process_group("nccl", rank=0, world_size=1, device_id=torch.device("cuda", 0))
    try:
        group = dist.group.WORLD
        for kind in (2.0, INF):
            norm, coefficient = clip_coefficient([], 1.0, kind, group=group)
            assert float(norm) == 0.0 and float(coefficient) == 1.0
            assert float(clip_grad_norm([], 1.0, kind, group=group)) == 0.0
            bad = torch.ones(3000, device="cuda")
            bad[1234] = float("nan")
            norm, coefficient = clip_coefficient([torch.ones(5, device="cuda")], 1.0, kind, sharded=[-bad], group=group)
            assert bool(norm.isnan()) and bool(coefficient.isnan())
    finally:
        dist.destroy_process_group()


def test_a_training_step():
    """Norm, layer, loss, clipping and the optimizer's step as a user runs them: the coefficient handed to AdamW is clipping in place."""
    def build():
        torch.manual_seed(0)
        layer = MoELayer(256, 512, 4, pre_norm="rms", aux_loss_coeff=0.01).cuda().bfloat16()
        head = torch.nn.Parameter((torch.randn(1000, 256, device="cuda") * 0.05).bfloat16())
        final = torch.nn.Parameter(torch.ones(256, device="cuda").bfloat16())
        return layer, head, final

    x = torch.randn(512, 256, device="cuda").bfloat16()
    target = torch.randint(0, 1000, (512,), device="cuda")
    results = []
    for in_place in (True, False):
        layer, head, final = build()
        params = [*layer.parameters(), head, final]
        opt = AdamW(params, lr=1e-2)
        for _ in range(3):
            y, losses = layer(x)
            out, _ = rms_norm(y, final, residual=x)
            loss = linear_cross_entropy(out, head, target) + losses["aux_loss"]
            loss.backward()
            assert all(p.grad is not None and bool(p.grad.isfinite().all()) for p in params)
            if in_place:
                norm = clip_grad_norm(params, 0.05)
                assert float(norm) > 0.05
                opt.step()
            else:
                norm, coefficient = clip_coefficient([p.grad for p in params], 0.05)
                opt.step(grad_scale=coefficient)
            opt.zero_grad()
        results.append([p.detach().clone() for p in params])
    # scaled gradients are rounded to bfloat16 in place and are not with grad_scale: half a step of the update's operands, three steps of at
    # most lr (1 + a little) each, which Adam's sign-like first steps take for tiny gradients too
    for a, b in zip(*results):
        assert float((a.float() - b.float()).abs().max()) <= 2 * 3 * 1.1e-2


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("in_place", [True, False])
def test_the_optimizer_gets_the_clipped_gradients(dtype, in_place):
    """One step from nothing leaves (1 - beta) times the clipped gradient and its square in the moments. In place the gradient is rounded to its type
    first; then come roundings of fp32: the coefficient's product, 1 - beta, and the moment's product (for the square twice the first, and one more)."""
    grads = _grads([5000, 33, 128 * 70], DTYPES[dtype])
    params, limit = _params([g.clone() for g in grads]), 0.3 * _norm(grads)
    opt = AdamW(params, lr=1e-2)
    _, coefficient = clip_coefficient(grads, limit)
    assert abs(float(coefficient) - 0.3) < 1e-5
    if in_place:
        clip_grad_norm(params, limit)
        opt.step()
    else:
        opt.step(grad_scale=coefficient)
    info = torch.finfo(DTYPES[dtype])
    half, least = (info.eps / 2, info.tiny * info.eps) if in_place else (2.0 ** -24, 0.0)
    for p, g in zip(params, grads):
        want = g.double() * coefficient.double()
        m, v = (opt.state[p][name].double() for name in ("exp_avg", "exp_avg_sq"))
        off = (half + 3 * 2.0 ** -24) * (1 + 2.0 ** -10) * want.abs() + least
        assert bool(((m - 0.1 * want).abs() <= 0.1 * off).all())
        assert bool(((v - 0.001 * want.square()).abs() <= 0.001 * (2 * want.abs() * off + off * off + 5 * 2.0 ** -24 * want.square()) + 1e-44).all())
