"""CPU: the RMS norm, the 8-bit products and gradient clipping refuse what they cannot run before anything reaches a device: tensors on the
host, arguments of the C entry points."""

import ctypes
import datetime
import multiprocessing
import os
import shutil
import subprocess

import pytest
import torch

from flashfusedmoe_b200 import MoELayer, RMSNorm, _lib, clip, clip_coefficient, clip_grad_norm, linear_e4m3, quantize_e4m3, rms_norm

BAD, UNSUPPORTED, WORKSPACE = -1, -2, -4
BF16, FP16, FP32 = 0, 1, 2


def test_tensors_on_the_host_are_refused():
    x = torch.randn(4, 64).bfloat16()
    p = torch.nn.Parameter(torch.ones(8))
    p.grad = torch.ones(8)
    q, s = x.to(torch.float8_e4m3fn), torch.ones(4, 1)
    for call in (lambda: rms_norm(x), lambda: RMSNorm(64)(x), lambda: rms_norm(x, residual=x, quantize=True), lambda: quantize_e4m3(x),
                 lambda: quantize_e4m3(x, 128), lambda: linear_e4m3(q, s, q, torch.ones(1, 1)), lambda: clip_coefficient([p.grad], 1.0),
                 lambda: clip_grad_norm([p], 1.0), lambda: clip_grad_norm([p], 1.0, error_if_nonfinite=True)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_module_is_torchs():
    ours, theirs = RMSNorm(48, eps=1e-5), torch.nn.RMSNorm(48, eps=1e-5)
    assert ours.state_dict().keys() == theirs.state_dict().keys()
    theirs.load_state_dict(ours.state_dict())
    assert torch.equal(ours.weight, theirs.weight) and list(RMSNorm(8, elementwise_affine=False).parameters()) == []
    assert not bool(RMSNorm(8, weight_offset=1.0).weight.any())
    for shape in ((3, 4), (), 0):
        with pytest.raises(ValueError, match="one dimension"):
            RMSNorm(shape)
    with pytest.raises(ValueError, match="must end in"):
        RMSNorm(8)(torch.zeros(2, 9))


def test_layers_have_the_norm_that_was_asked_for():
    names = [n for n, _ in MoELayer(32, 64, 4).named_parameters()]
    layer = MoELayer(32, 64, 4, pre_norm="rms", norm_eps=1e-3)
    assert [n for n, _ in layer.named_parameters() if n not in names] == ["norm.weight"] and layer.norm.eps == 1e-3
    assert isinstance(MoELayer(32, 64, 4, pre_norm="layer").norm, type(MoELayer(32, 64, 4, pre_norm=True).norm))
    with pytest.raises(ValueError, match="Unknown norm"):
        MoELayer(32, 64, 4, pre_norm="batch")


def test_what_stands_for_no_norm():
    for none in (False, None, 0, ""):
        assert not any(n.startswith("norm") for n, _ in MoELayer(32, 64, 4, pre_norm=none).named_parameters())
    assert [n for n, _ in MoELayer(32, 64, 4, pre_norm=1).named_parameters() if n.startswith("norm")] == ["norm.weight", "norm.bias"]


def test_clipping_arguments():
    p = torch.nn.Parameter(torch.ones(2))
    for call in (clip_coefficient, clip_grad_norm):
        with pytest.raises(ValueError, match="norm_type"):
            call([p], 1.0, 1.0)
        for wrong in (-1.0, float("nan")):
            with pytest.raises(ValueError, match="max_norm"):
                call([p], wrong)
    with pytest.raises(ValueError, match="no gradients"):
        clip_coefficient([], 1.0)
    assert float(clip_grad_norm([], 1.0)) == 0.0 and float(clip_grad_norm(p, 1.0)) == 0.0   # nothing has a gradient
    with pytest.raises(ValueError, match="sharded"):
        clip_grad_norm([p], 1.0, sharded=[torch.nn.Parameter(torch.ones(2))], group=object())


def test_sharded_parameters_are_checked_without_a_group_too(monkeypatch):
    p, other = (torch.nn.Parameter(torch.ones(2)) for _ in range(2))
    for error_if_nonfinite in (False, True):
        with pytest.raises(ValueError, match="sharded"):
            clip_grad_norm([p], 1.0, error_if_nonfinite=error_if_nonfinite, sharded=[other])
    assert float(clip_grad_norm([p], 1.0, sharded=p)) == 0.0   # one tensor stands for a list of it
    monkeypatch.setattr(_lib, "native", _OneRank)
    norm, _ = clip_coefficient([torch.tensor([3.0])], 1.0, sharded=torch.tensor(4.0))
    assert float(norm) == 5.0


class RmsArgs(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int64) for n in ("rows", "D", "x_type", "w_type", "x_stride", "residual_stride")] + \
        [(n, ctypes.c_double) for n in ("eps", "offset")] + \
        [(n, ctypes.c_int64) for n in ("x", "residual", "weight", "h", "y", "y_scale", "rstd", "dy", "dh", "dx", "dweight", "workspace",
                                       "workspace_bytes")]


def _rms(function, **values):
    fields = dict(rows=4, D=64, x_stride=64, residual_stride=64, eps=1e-6, x=256, residual=256, weight=256, h=256, y=256, rstd=256, dy=256, dh=256,
                  dx=256, dweight=256, workspace=256, workspace_bytes=1 << 40)
    fields.update(values)
    block = RmsArgs(**fields)
    return function(ctypes.addressof(block), 0)


def test_rms_norm_entry_points():
    lib = _lib.load()
    forward, backward = lib.ffm_rms_norm_forward, lib.ffm_rms_norm_backward
    for call in (forward, backward):
        assert call(0, 0) == BAD
        for wrong in (dict(x=0), dict(x_type=3), dict(x_type=-1), dict(w_type=7), dict(rows=-1), dict(D=0), dict(x_stride=63), dict(eps=-1.0),
                      dict(eps=float("nan")), dict(offset=float("nan")), dict(offset=float("inf"))):
            assert _rms(call, **wrong) == BAD, wrong
        assert _rms(call, D=32769, x_stride=32769, residual_stride=32769) == UNSUPPORTED
        assert _rms(call, D=16385, x_stride=16385, residual_stride=16385, x_type=FP32, w_type=FP32) == UNSUPPORTED
    for wrong in (dict(y=0), dict(h=0), dict(residual_stride=63)):
        assert _rms(forward, **wrong) == BAD, wrong
    assert _rms(forward, rows=0, x=0, y=0) == 0
    # 8 bits: rows of 16 values on 16 bytes
    assert _rms(forward, y_scale=256, D=60) == UNSUPPORTED
    for off in ("x", "residual", "h", "weight"):
        assert _rms(forward, y_scale=256, **{off: 258}) == UNSUPPORTED, off
    assert _rms(forward, y_scale=256, y=260) == UNSUPPORTED and _rms(forward, y_scale=256, x_stride=68) == UNSUPPORTED
    for wrong in (dict(dy=0), dict(rstd=0), dict(weight=0)):
        assert _rms(backward, **wrong) == BAD, wrong
    need = lib.ffm_rms_norm_workspace_bytes(4, 64, BF16)
    assert need > 0 and lib.ffm_rms_norm_workspace_bytes(4, 0, BF16) == 0 and lib.ffm_rms_norm_workspace_bytes(4, 64, 9) == 0
    assert _rms(backward, workspace=0) == WORKSPACE and _rms(backward, workspace_bytes=need - 1) == WORKSPACE
    assert _rms(backward, dx=0, dweight=0) == 0 and _rms(backward, rows=0, dweight=0) == 0


class LinearArgs(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int64) for n in ("rows", "N", "K", "experts", "x_stride", "out_type", "x", "x_scale", "w", "w_scale", "ends", "out",
                                              "status", "status_host")]


def _linear(lib, **values):
    fields = dict(rows=10, N=100, K=64, experts=3, x_stride=64, x=256, x_scale=256, w=256, w_scale=256, ends=256, out=256, status=256)
    fields.update(values)
    block = LinearArgs(**fields)
    return lib.ffm_linear_blocks_e4m3(ctypes.addressof(block), 0)


def test_e4m3_entry_points():
    lib, a = _lib.load(), 256

    def quantize(x=a, x_type=BF16, matrices=1, rows=4, stride=64, K=64, block_rows=1, q=a, scale=a):
        return lib.ffm_quantize_blocks_e4m3(x, x_type, matrices, rows, stride, K, block_rows, q, scale, 0)

    for wrong in (dict(x=0), dict(q=0), dict(scale=0), dict(x_type=3), dict(matrices=-1), dict(rows=-1), dict(K=0), dict(block_rows=2), dict(stride=63),
                  dict(matrices=2)):
        assert quantize(**wrong) == BAD, wrong
    for wrong in (dict(K=60), dict(x=264), dict(q=260), dict(stride=68), dict(block_rows=128, stride=128)):
        assert quantize(**wrong) == UNSUPPORTED, wrong
    assert quantize(rows=0, x=0) == 0 and quantize(matrices=0, block_rows=128, x=0) == 0

    assert lib.ffm_linear_blocks_e4m3(0, 0) == BAD
    for wrong in (dict(rows=-1), dict(N=0), dict(K=0), dict(experts=0), dict(out_type=3), dict(x_stride=63), dict(x=0), dict(x_scale=0), dict(w=0),
                  dict(w_scale=0), dict(out=0), dict(status=0), dict(ends=0)):
        assert _linear(lib, **wrong) == BAD, wrong
    for wrong in (dict(K=56), dict(x_stride=72), dict(experts=1025), dict(rows=1 << 31)):
        assert _linear(lib, **wrong) == UNSUPPORTED, wrong
    assert _linear(lib, rows=0, x=0, out=0) == 0


class ClipTensor(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int64) for n in ("x", "type", "elements")]


class NormArgs(ctypes.Structure):
    _fields_ = [("kind", ctypes.c_int64), ("max_norm", ctypes.c_double)] + \
        [(n, ctypes.c_int64) for n in ("other", "total", "norm", "coefficient", "workspace", "workspace_bytes", "ticket", "launched")]


def _norm(lib, tensor=(), count=1, **values):
    fields = dict(max_norm=1.0, norm=256, coefficient=256, workspace=256, workspace_bytes=1 << 30, ticket=256)
    fields.update(values)
    t = ClipTensor(**dict(dict(x=256, type=BF16, elements=10), **dict(tensor)))
    block = NormArgs(**fields)
    return lib.ffm_grad_norm(ctypes.addressof(t), count, ctypes.addressof(block), 0)


def test_clipping_entry_points():
    lib = _lib.load()
    for wrong in (dict(count=-1), dict(kind=2), dict(max_norm=-1.0), dict(max_norm=float("nan")), dict(ticket=0), dict(tensor=dict(x=0)),
                  dict(tensor=dict(type=3)), dict(tensor=dict(elements=-1))):
        assert _norm(lib, **wrong) == BAD, wrong
    assert lib.ffm_grad_norm(0, 1, 0, 0) == BAD
    need = lib.ffm_grad_norm_workspace_bytes(1)
    assert lib.ffm_grad_norm_workspace_bytes(513) == 2 * need and lib.ffm_grad_norm_workspace_bytes(-1) == 0 < lib.ffm_grad_norm_workspace_bytes(0)
    assert _norm(lib, workspace=0) == WORKSPACE and _norm(lib, workspace_bytes=need - 1) == WORKSPACE
    t = ClipTensor(256, BF16, 10)
    assert lib.ffm_scale_tensors(ctypes.addressof(t), 1, 0, 0, 0) == BAD and lib.ffm_scale_tensors(0, 1, 256, 0, 0) == BAD
    assert lib.ffm_scale_tensors(0, 0, 0, 0, 0) == 0


def _without_a_device():
    """With fitting arguments a call gets as far as a launch or a tensor map, which fails: an error code, no exception, no abort."""
    lib, a = _lib.load(), 256
    for rows in (4, 100000):
        assert _rms(lib.ffm_rms_norm_forward, rows=rows) < 0 and _rms(lib.ffm_rms_norm_backward, rows=rows) < 0
        assert _rms(lib.ffm_rms_norm_forward, rows=rows, y_scale=256) < 0
    assert lib.ffm_quantize_blocks_e4m3(a, BF16, 1, 4, 64, 64, 1, a, a, 0) < 0 and lib.ffm_quantize_blocks_e4m3(a, FP32, 2, 4, 64, 64, 128, a, a, 0) < 0
    for values in ({}, dict(rows=100000), dict(ends=0, experts=1), dict(N=101, rows=5000)):
        assert _linear(lib, **values) < 0
    t = ClipTensor(256, BF16, 10)
    assert _norm(lib) < 0 and lib.ffm_scale_tensors(ctypes.addressof(t), 1, 256, 0, 0) < 0


def test_calls_without_a_device_return_an_error(monkeypatch):
    monkeypatch.setenv("CUDA_VISIBLE_DEVICES", "")
    child = multiprocessing.get_context("spawn").Process(target=_without_a_device)
    child.start()
    child.join()
    assert child.exitcode == 0


class _OneRank:
    """A stand-in for the library's norm of a rank's own gradients, on host tensors: what a group adds up is tested without a GPU."""

    def gradient_norm(self, grads, like, max_norm, largest, other):
        if largest:
            total = torch.stack([g.abs().max() for g in grads]).max().double() if grads else torch.zeros((), dtype=torch.float64)
            total = total if other is None else torch.maximum(total, other[0])
        else:
            total = sum((g.double().square().sum() for g in grads), torch.zeros((), dtype=torch.float64)) + (0 if other is None else other[0])
        norm = total if largest else total.sqrt()
        return total.view(1), norm.float(), (max_norm / (norm + 1e-6)).clamp(max=1.0).float()

    def scale_gradients(self, grads, factor):
        for g in grads:
            g.mul_(factor)


def _rank(rank, port, out):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    torch.distributed.init_process_group("gloo", rank=rank, world_size=2)
    _lib._native = _OneRank()
    _lib.native = lambda: _lib._native
    group = torch.distributed.group.WORLD
    dense, expert, other = (torch.nn.Parameter(torch.zeros(3)) for _ in range(3))
    dense.grad = torch.tensor([1.0, 2.0, 2.0])                   # the same on both ranks: counted once
    expert.grad = torch.tensor([4.0, 0.0, 0.0]) * (1 + rank)     # 16 and 64
    for kind, want in ((2.0, 89.0 ** 0.5), (float("inf"), 8.0)):
        norm, coefficient = clip_coefficient([dense.grad], 1.0, kind, sharded=[expert.grad], group=group)
        assert abs(float(norm) - want) < 1e-5 and abs(float(coefficient) - 1 / want) < 1e-5
    if rank == 1:
        expert.grad = None   # its experts had no rows: it takes part all the same
    norm = clip_grad_norm([dense, expert, other], 1.0, sharded=[expert], group=group)
    assert abs(float(norm) - 5.0) < 1e-5 and torch.allclose(dense.grad, torch.tensor([0.2, 0.4, 0.4]))
    assert rank == 1 or torch.allclose(expert.grad, torch.tensor([0.8, 0.0, 0.0]))
    out.put(rank)
    torch.distributed.destroy_process_group()


def test_sharded_gradients_are_added_up_over_the_group():
    context = multiprocessing.get_context("spawn")
    out, port = context.Queue(), 29600 + os.getpid() % 300
    ranks = [context.Process(target=_rank, args=(r, port, out)) for r in range(2)]
    for r in ranks:
        r.start()
    for r in ranks:
        r.join(120)
    assert [r.exitcode for r in ranks] == [0, 0] and sorted(out.get() for _ in ranks) == [0, 1]


def _rank_with_nan(rank, port, out):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    torch.distributed.init_process_group("gloo", rank=rank, world_size=2)
    _lib._native = _OneRank()
    _lib.native = lambda: _lib._native
    group = torch.distributed.group.WORLD
    for kind in (2.0, float("inf")):
        for bad in (0, 1):
            for value in (float("nan"), float("inf")):
                dense = torch.tensor([1.0])
                expert = torch.tensor([3.0, -value if rank == bad else 2.0])   # a negative NaN, where there is a sign
                norm, coefficient = clip_coefficient([dense], 1.0, kind, sharded=[expert], group=group)
                assert bool(norm.isnan() if value != value else norm.isinf()), (kind, bad, value, norm)
                assert bool(coefficient.isnan()) if value != value else float(coefficient) == 0.0
                p, q = torch.nn.Parameter(torch.zeros(1)), torch.nn.Parameter(torch.zeros(2))
                p.grad, q.grad = dense, expert
                try:
                    clip_grad_norm([p, q], 1.0, kind, error_if_nonfinite=True, sharded=[q], group=group)
                except RuntimeError as e:
                    assert "not finite" in str(e)
                else:
                    raise AssertionError("no error")
    out.put(rank)
    torch.distributed.destroy_process_group()


def test_a_nan_of_one_rank_reaches_all():
    context = multiprocessing.get_context("spawn")
    out, port = context.Queue(), 29900 + os.getpid() % 90
    ranks = [context.Process(target=_rank_with_nan, args=(r, port, out)) for r in range(2)]
    for r in ranks:
        r.start()
    for r in ranks:
        r.join(120)
    assert [r.exitcode for r in ranks] == [0, 0] and sorted(out.get() for _ in ranks) == [0, 1]


def _rank_without_any(rank, port, out):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    torch.distributed.init_process_group("gloo", rank=rank, world_size=2, timeout=datetime.timedelta(seconds=30))
    _lib._native = _OneRank()
    _lib.native = lambda: _lib._native
    clip._nothing = lambda: torch.empty(0)   # the device's
    group = torch.distributed.group.WORLD
    p = torch.nn.Parameter(torch.zeros(2))
    p.grad = torch.tensor([3.0, 4.0])
    mine = [p] if rank == 0 else []
    for kind, want in ((2.0, 5.0), (float("inf"), 4.0)):
        norm, coefficient = clip_coefficient([], 1.0, kind, sharded=[q.grad for q in mine], group=group)
        assert abs(float(norm) - want) < 1e-5 and abs(float(coefficient) - 1 / want) < 1e-5
    assert abs(float(clip_grad_norm(mine, 10.0, sharded=mine, group=group)) - 5.0) < 1e-5
    out.put(rank)
    torch.distributed.destroy_process_group()


def test_a_rank_without_gradients_takes_part():
    context = multiprocessing.get_context("spawn")
    out, port = context.Queue(), 29990 + os.getpid() % 90
    ranks = [context.Process(target=_rank_without_any, args=(r, port, out)) for r in range(2)]
    for r in ranks:
        r.start()
    for r in ranks:
        r.join(120)
    assert [r.exitcode for r in ranks] == [0, 0] and sorted(out.get() for _ in ranks) == [0, 1]


_FIRST_CALLS = r"""
#include <atomic>
#include <chrono>
#include <cstdio>
#include <thread>
#include <vector>
#include "ffm_gemm_common.cuh"

// in place of the runtime's: slow, as a first call is
extern "C" cudaError_t cudaGetDriverEntryPoint(const char*, void** f, unsigned long long, cudaDriverEntryPointQueryResult* result) {
  std::this_thread::sleep_for(std::chrono::milliseconds(200));
  *f = reinterpret_cast<void*>(64);
  *result = cudaDriverEntryPointSuccess;
  return cudaSuccess;
}

int main() {
  std::atomic<int> missing{0};
  std::vector<std::thread> threads;
  for (int i = 0; i < 8; ++i) threads.emplace_back([&] { missing += ffm::get_encode_fn() == nullptr; });
  for (auto& t : threads) t.join();
  std::printf("%d", missing.load());
  return 0;
}
"""


@pytest.mark.skipif(shutil.which("nvcc") is None, reason="needs nvcc")
def test_first_calls_of_several_threads_find_the_driver(tmp_path):
    source, program = tmp_path / "first.cu", tmp_path / "first"
    source.write_text(_FIRST_CALLS)
    csrc = os.path.join(os.path.dirname(_lib.__file__), "csrc")
    subprocess.run(["nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-cudart", "shared", "-I", csrc, str(source), "-o", str(program),
                    "-lpthread"], check=True, capture_output=True)
    assert subprocess.run([str(program)], check=True, capture_output=True, text=True).stdout == "0"
