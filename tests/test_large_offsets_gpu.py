"""Tensors of more than 2^31 values: offsets that do not fit in 32 bits, looked at where they are largest."""

import pytest
import torch

import test_adamw_gpu as adamw
import test_layer_norm_gpu as norm
import test_linear_cross_entropy_gpu as entropy

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def room():
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("width", [8192, 8191])
def test_layer_norm_rows(width):
    """Rows that start anywhere and rows on 16 bytes. All rows but the last ones are zero: their y is the bias, and nothing of dw."""
    rows = (1 << 31) // width + 700
    x, w, b, dy = norm.inputs(64, width, torch.bfloat16, 3)
    big, grad = torch.zeros(rows, width, dtype=torch.bfloat16, device="cuda"), torch.zeros(rows, width, dtype=torch.bfloat16, device="cuda")
    big[-64:], grad[-64:] = x, dy
    out, bound = norm.reference(x, w, b, 1e-5, dy)
    y, (dx, dw, db) = norm.run(big, w, b, grad)
    for got, name in ((y[-64:], "y"), (dx[-64:], "dx"), (dw, "dw"), (db, "db")):
        norm.check(got, out, bound, name)
    assert torch.equal(y[0], b) and torch.equal(y[rows - 65], b) and not dx[:64].any() and not dx[-128:-64].any()


def test_a_row_longer_than_32_bits_say_is_refused():
    from flashfusedmoe_b200 import layer_norm
    with pytest.raises(ValueError, match="4294967304 values"):
        layer_norm(torch.empty(1, (1 << 32) + 8, dtype=torch.bfloat16, device="cuda"))


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_values(bits):
    from flashfusedmoe_b200 import adamw_step
    n = (1 << 31) + 4096 * 3 + 77
    t = adamw.Tensors([5000], torch.bfloat16, bits, seed=9)
    tail, start = 5000, (n - 5000) // 128 * 128
    n = start + tail
    def wide(values, dtype):
        big = torch.zeros(n, dtype=torch.uint8, device="cuda").view(dtype) if dtype == torch.float8_e4m3fn else torch.zeros(n, dtype=dtype, device="cuda")
        (big.view(torch.uint8) if dtype == torch.float8_e4m3fn else big)[start:] = values.view(torch.uint8) if dtype == torch.float8_e4m3fn else values
        return big
    p, g = wide(t.params[0], torch.bfloat16), wide(t.grads[0], torch.bfloat16)
    m, v = wide(t.m[0], t.m[0].dtype), wide(t.v[0], t.v[0].dtype)
    scales = {}
    if bits == 8:
        for name, s in (("exp_avg_scales", t.m_scale[0]), ("exp_avg_sq_scales", t.v_scale[0])):
            big = torch.zeros((n + 127) // 128, dtype=torch.uint8, device="cuda")
            big[start // 128:] = s
            scales[name] = [big]
    found, before = t.exact(), [t.steps[0].item()]
    adamw_step([p], [g], [m], [v], t.steps, **scales, **adamw.HYPER)
    t.params, t.m, t.v = [p[start:].clone()], [m.view(m.dtype)[start:].clone()], [v[start:].clone()]
    if bits == 8:
        t.m_scale, t.v_scale = [scales["exp_avg_scales"][0][start // 128:]], [scales["exp_avg_sq_scales"][0][start // 128:]]
    t.check(found, before)
    assert not p[:start].any()


def test_a_weight_of_the_vocabulary():
    """V D and N V beyond 2^31: the rows' entries in one piece against pieces of 256 rows, and rows against 64 bits."""
    h, w, t = entropy.inputs(8192, 64, 300000, seed=1)
    loss, dh, dw = entropy.run(h, w, t, _piece_rows=8192)
    other = entropy.run(h, w, t, _piece_rows=256)
    assert torch.equal(loss, other[0])
    # the contraction over the vocabulary is split differently: each sum is off by (V / 16 + 20) 2^-22 of the terms' magnitudes,
    # which are at most 2 / 8192 in all times the largest weight, and half a unit of bf16
    off = (dh.double() - other[1].double()).abs()
    assert (off <= 2.0 ** -7 * dh.double().abs() + 2 * (300000 / 16 + 20) * 2.0 ** -22 * 2 / 8192 * w.double().abs().max()).all()
    # one sum in fp32 of 8192 terms against 32 sums of 256: each off by less than 2^-13 of the terms' magnitudes, which here is a
    # few times the result; then half a unit of bf16 each
    off = (dw.double() - other[2].double()).abs()
    assert (off <= 2.0 ** -7 * dw.double().abs() + 2.0 ** -11 * dw.double().abs().amax(1, keepdim=True)).all()
    del dw, other
    d = 8192
    h, w, t = entropy.inputs(40, d, (1 << 31) // d + 999, seed=2)
    t[:20] = w.shape[0] - 1 - torch.arange(20, device="cuda")
    from flashfusedmoe_b200 import linear_cross_entropy
    out, bound = entropy.reference(h[:10], w, t[:10], reduction="sum")
    with torch.no_grad():
        nll = linear_cross_entropy(h, w, t, reduction="none")
        few = linear_cross_entropy(h[:10], w, t[:10], reduction="none")
    entropy.check(nll[:10], out, bound, "nll")
    entropy.check(few, out, bound, "nll")
    loss, dh, dw = entropy.run(h[:10], w, t[:10], reduction="sum")
    entropy.check(loss, out, bound, "loss")
    entropy.check(dh, out, bound, "dh")
    entropy.check(dw[-64:], {"dw": out["dw"][-64:]}, {"dw": bound["dw"][-64:]}, "dw")
