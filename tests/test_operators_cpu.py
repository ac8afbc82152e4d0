"""CPU: the operators beside the layer refuse what they cannot run before anything reaches a device: tensors on the host, arguments
of the C entry points."""

import ctypes
import multiprocessing

import pytest
import torch

from flashfusedmoe_b200 import AdamW, LayerNorm, MoELayer, _lib, adamw_step, layer_norm, linear_cross_entropy

BAD, UNSUPPORTED, WORKSPACE = -1, -2, -4
BF16, FP16, FP32 = 0, 1, 2


def test_tensors_on_the_host_are_refused():
    x = torch.randn(4, 64).bfloat16()
    for call in (lambda: layer_norm(x), lambda: LayerNorm(64)(x), lambda: linear_cross_entropy(x, x, torch.zeros(4, dtype=torch.int64)),
                 lambda: adamw_step([x], [x], [x.float()], [x.float()], [torch.zeros((), dtype=torch.int32)], lr=1e-3)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    p = torch.nn.Parameter(torch.ones(8))
    p.grad = torch.ones(8)
    with pytest.raises(RuntimeError, match="no CPU path"):
        AdamW([p]).step()


def test_layer_norm_module_is_torchs():
    ours, theirs = LayerNorm(48, eps=1e-6), torch.nn.LayerNorm(48, eps=1e-6)
    assert ours.state_dict().keys() == theirs.state_dict().keys()
    theirs.load_state_dict(ours.state_dict())
    assert torch.equal(ours.weight, theirs.weight) and torch.equal(ours.bias, theirs.bias)
    assert list(LayerNorm(8, elementwise_affine=False).parameters()) == [] and LayerNorm(8, bias=False).bias is None
    for shape in ((3, 4), (), 0):
        with pytest.raises(ValueError, match="one dimension"):
            LayerNorm(shape)
    with pytest.raises(ValueError, match="must end in"):
        LayerNorm(8)(torch.zeros(2, 9))


def test_layers_have_a_norm_only_where_asked():
    names = [n for n, _ in MoELayer(32, 64, 4).named_parameters()]
    assert [n for n, _ in MoELayer(32, 64, 4, pre_norm=True).named_parameters() if n not in names] == ["norm.weight", "norm.bias"]
    assert MoELayer(32, 64, 4, pre_norm=True, norm_eps=1e-3).norm.eps == 1e-3


def test_optimizer_arguments():
    p = [torch.nn.Parameter(torch.ones(2))]
    for options in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1e-8), dict(weight_decay=-0.1)):
        with pytest.raises(ValueError):
            AdamW(p, **options)
    assert AdamW(p).step(closure=lambda: 3.0) == 3.0   # nothing has a gradient


def test_state_dicts_of_other_steps_are_refused():
    p = [torch.nn.Parameter(torch.ones(2))]
    for other in (torch.optim.AdamW(p, amsgrad=True), torch.optim.AdamW(p, maximize=True), torch.optim.Adam(p, weight_decay=0.1)):
        with pytest.raises(ValueError, match="another step"):
            AdamW(p).load_state_dict(other.state_dict())
    for same in (torch.optim.AdamW(p, lr=0.5), torch.optim.Adam(p, lr=0.5)):
        mine = AdamW(p)
        mine.load_state_dict(same.state_dict())
        assert mine.param_groups[0]["lr"] == 0.5 and mine.param_groups[0]["state_bits"] == 32


def test_layer_norm_entry_points():
    lib, a = _lib.load(), 256

    def forward(x=a, x_type=BF16, rows=4, stride=64, D=64, w=a, w_type=BF16, b=a, b_type=BF16, eps=1e-5, y=a, mean=a, rstd=a):
        return lib.ffm_layer_norm_forward(x, x_type, rows, stride, D, w, w_type, b, b_type, eps, y, mean, rstd, 0)

    for wrong in (dict(x=0), dict(y=0), dict(x_type=3), dict(x_type=-1), dict(w_type=7), dict(b_type=7), dict(rows=-1), dict(D=0), dict(stride=63),
                  dict(eps=-1.0), dict(eps=float("nan")), dict(mean=0), dict(rstd=0)):
        assert forward(**wrong) == BAD, wrong
    assert forward(D=32769, stride=32769) == UNSUPPORTED and forward(D=16385, stride=16385, x_type=FP32) == UNSUPPORTED
    assert forward(rows=0, x=0, y=0) == 0

    need = lib.ffm_layer_norm_workspace_bytes(1000, 64, BF16)
    assert need > 0 and lib.ffm_layer_norm_workspace_bytes(1000, 0, BF16) == 0 and lib.ffm_layer_norm_workspace_bytes(1000, 64, 9) == 0

    def backward(dy=a, x=a, rows=1000, D=64, mean=a, dx=a, dw=a, db=a, workspace=a, size=need, w_type=BF16, b_type=BF16):
        return lib.ffm_layer_norm_backward(dy, x, BF16, rows, D, D, a, w_type, mean, a, dx, dw, db, b_type, workspace, size, 0)

    for wrong in (dict(dy=0), dict(x=0), dict(mean=0), dict(rows=-1), dict(w_type=5), dict(b_type=5)):
        assert backward(**wrong) == BAD, wrong
    assert backward(size=need - 1) == WORKSPACE and backward(workspace=0) == WORKSPACE
    assert backward(rows=0, dw=0, db=0, workspace=0, size=0) == 0 and backward(dx=0, dw=0, db=0, workspace=0, size=0) == 0


class AdamWTensor(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int64) for n in ("param", "grad", "exp_avg", "exp_avg_sq", "master", "exp_avg_scale", "exp_avg_sq_scale", "step",
                                              "elements", "param_type", "grad_type")]


class AdamWArgs(ctypes.Structure):
    _fields_ = [(n, ctypes.c_double) for n in ("lr", "beta1", "beta2", "eps", "weight_decay")] + \
        [(n, ctypes.c_int64) for n in ("lr_device", "grad_scale", "bits", "seed", "ticket", "launched")]


def test_adamw_entry_point():
    lib = _lib.load()

    def call(count=1, tensor=(), **args):
        t = AdamWTensor(*[256] * 8, 100, BF16, BF16)
        h = AdamWArgs(1e-3, 0.9, 0.99, 1e-8, 0.0, 0, 0, 32, 0, 256, 0)
        for k, v in dict(tensor).items():
            setattr(t, k, v)
        for k, v in args.items():
            setattr(h, k, v)
        return lib.ffm_adamw_step(ctypes.addressof(t), count, ctypes.addressof(h), 0)

    assert call(count=0) == 0 and call(count=-1) == BAD and lib.ffm_adamw_step(0, 1, 0, 0) == BAD
    for wrong in ("param", "grad", "exp_avg", "exp_avg_sq", "step"):
        assert call(tensor={wrong: 0}) == BAD, wrong
    for wrong in ("exp_avg_scale", "exp_avg_sq_scale"):
        assert call(tensor={wrong: 0}, bits=8) == BAD, wrong
    for wrong in (dict(bits=16), dict(ticket=0), dict(beta1=1.0), dict(beta2=-0.1), dict(eps=-1.0), dict(beta1=float("nan"))):
        assert call(**wrong) == BAD, wrong
    for wrong in (dict(elements=-1), dict(param_type=3), dict(grad_type=-1)):
        assert call(tensor=wrong) == BAD, wrong


class LossArgs(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int64) for n in ("N", "D", "V", "ignore_index", "mean", "d_weight_f32", "piece_rows")] + [("z", ctypes.c_double)] + \
        [(n, ctypes.c_int64) for n in ("hidden", "weight", "targets", "row_grad", "nll", "loss", "d_hidden", "d_weight", "workspace",
                                       "workspace_bytes", "status", "status_host", "launched")]


def _loss(**values):
    fields = dict(N=10, D=64, V=100, ignore_index=-100, mean=1, piece_rows=256, hidden=256, weight=256, targets=256, nll=256, loss=256, d_hidden=256,
                  d_weight=256, workspace=256, workspace_bytes=1 << 40, status=256)
    fields.update(values)
    return LossArgs(**fields)


def _run_loss(lib, **values):
    block = _loss(**values)
    return lib.ffm_linear_cross_entropy(ctypes.addressof(block), 0)


def _loss_workspace(lib, **values):
    block = _loss(**values)
    return lib.ffm_linear_cross_entropy_workspace_bytes(ctypes.addressof(block))


def test_linear_cross_entropy_entry_points():
    lib = _lib.load()

    def call(**values):
        return _run_loss(lib, **values)

    for wrong in (dict(hidden=0), dict(weight=0), dict(targets=0), dict(nll=0), dict(status=0), dict(loss=0), dict(row_grad=256), dict(N=-1), dict(D=0),
                  dict(V=0), dict(piece_rows=0), dict(V=1 << 31)):
        assert call(**wrong) == BAD, wrong
    assert lib.ffm_linear_cross_entropy(0, 0) == BAD
    assert call(D=60) == UNSUPPORTED
    for off in ("hidden", "weight", "d_hidden", "d_weight", "workspace"):
        assert call(**{off: 260}) == UNSUPPORTED, off
    need = _loss_workspace(lib)
    assert call(workspace=0) == WORKSPACE and call(workspace_bytes=need - 1) == WORKSPACE

    def size(**values):
        return _loss_workspace(lib, N=100000, V=50257, **values)

    # two bytes an entry for a piece of the rows with gradients, eight bytes for 128 entries without
    assert size(piece_rows=256) < size(piece_rows=512) < 512 * 50257 * 3 + 50257 * 64 * 4 + (1 << 20)
    assert size(d_hidden=0, d_weight=0) < 100000 * 50257 // 8
    assert lib.ffm_linear_cross_entropy_workspace_bytes(0) == 0

    assert _scale(lib, [(256, BF16, 8)], factor=0) == BAD and _scale(lib, [(0, BF16, 8)]) == BAD and _scale(lib, [(256, 4, 8)]) == BAD
    assert _scale(lib, [(256, BF16, -8)]) == BAD and _scale(lib, [(256, BF16, 8)] * 9) == BAD and lib.ffm_scale_many(1, 0, 0, 0, 256, 0) == BAD
    assert _scale(lib, [(256, BF16, 7)]) == UNSUPPORTED and _scale(lib, [(256, BF16, 8), (260, BF16, 8)]) == UNSUPPORTED
    assert _scale(lib, []) == 0 and _scale(lib, [(0, BF16, 0)]) == 0


def _scale(lib, tensors, factor=256):
    columns = [(ctypes.c_int64 * max(1, len(tensors)))(*[t[i] for t in tensors]) for i in range(3)]
    return lib.ffm_scale_many(len(tensors), *[ctypes.addressof(c) for c in columns], factor, 0)


def _without_a_device():
    """With fitting arguments a call gets as far as a launch or a tensor map, which fails: an error code, no exception, no abort."""
    lib, a = _lib.load(), 256
    assert lib.ffm_layer_norm_forward(a, BF16, 4, 64, 64, a, FP32, 0, 0, 1e-5, a, a, a, 0) < 0
    assert lib.ffm_layer_norm_backward(a, a, FP16, 100000, 64, 64, a, FP16, a, a, a, a, a, FP16, a, 1 << 30, 0) < 0
    t, h = AdamWTensor(*[256] * 8, 100, BF16, BF16), AdamWArgs(1e-3, 0.9, 0.99, 1e-8, 0.0, 0, 0, 8, 0, 256, 0)
    assert lib.ffm_adamw_step(ctypes.addressof(t), 1, ctypes.addressof(h), 0) < 0
    for values in ({}, dict(d_hidden=0, d_weight=0), dict(mean=0, loss=0), dict(N=5, d_hidden=0, d_weight=0)):
        assert _run_loss(lib, **values) < 0
    assert _scale(lib, [(a, FP32, 8)]) < 0


def test_calls_without_a_device_return_an_error(monkeypatch):
    monkeypatch.setenv("CUDA_VISIBLE_DEVICES", "")
    child = multiprocessing.get_context("spawn").Process(target=_without_a_device)
    child.start()
    child.join()
    assert child.exitcode == 0
