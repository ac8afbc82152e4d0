"""Linear cross entropy at values where a maximum, a rounding or a difference can lose the result.

Logits that have to be exact are built from operands whose products and sums are. u = 2^-24."""

import pytest
import torch

from test_linear_cross_entropy_gpu import IGNORE, U, check, inputs, reference, run


# rows: the few-rows kernel with one and two groups of rows, tiles with a block a row, tiles with a warp a row
@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 3, 12, 40, 1500])
@pytest.mark.parametrize("v", [400, 5003])
def test_a_nan_in_the_vocabulary_reaches_every_row(n, v):
    """An entry that is no row's target: its logit is in every row's sum."""
    from flashfusedmoe_b200 import linear_cross_entropy
    h, w, t = inputs(n, 64, v, seed=n)
    bad = w.clone()
    bad[v // 2, 5] = float("nan")
    t[t == v // 2] = 0
    t[1::5] = IGNORE
    counts = t != IGNORE
    with torch.no_grad():
        nll = linear_cross_entropy(h, bad, t, reduction="none", z_loss_coeff=1e-4)
        assert nll[counts].isnan().all() and not nll[~counts].any()
        for reduction in ("mean", "sum"):
            assert linear_cross_entropy(h, bad, t, reduction=reduction).isnan()
    for reduction in ("mean", "none"):
        loss, dh, dw = run(h, bad, t, None if reduction == "mean" else torch.ones(n, device="cuda"), reduction=reduction)
        assert (loss if reduction == "mean" else loss[counts]).isnan().all()
        assert dh[counts].isnan().all() and dw.isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [3, 12, 40, 1500])
def test_an_infinity_in_the_vocabulary(n):
    """A logit of -infinity adds nothing to its row, one of +infinity leaves no finite sum."""
    from flashfusedmoe_b200 import linear_cross_entropy
    h, w, t = inputs(n, 64, 401, seed=n)
    t = t.clamp(max=399)
    bad = w.clone()
    bad[400] = 0.0
    bad[400, 2] = float("inf")
    h[:, 2] = torch.where(torch.arange(n, device="cuda") % 3 == 0, 1.0, -1.0)
    h[h == 0] = 1.0
    out, bound = reference(h, w[:400], t, 1e-4)
    with torch.no_grad():
        nll = linear_cross_entropy(h, bad, t, reduction="none", z_loss_coeff=1e-4)
    low = h[:, 2] < 0
    check(nll[low], {"nll": out["nll"][low]}, {"nll": bound["nll"][low]}, "nll")
    assert not nll[~low].isfinite().any()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 100, 1500])
@pytest.mark.parametrize("size", [0.0, 28.0, 500.0, -500.0])
def test_certain_rows_of_large_logits(rows, size):
    """Two entries, size and size - 10: the loss log(1 + e^-10), and 1 - p, do not depend on size, which fp32 holds in steps of 2^-15 at
    500. The sum is about 1 and is off by its roundings: three additions, the exponentials' and the logarithm's are less than 16 u in all."""
    from flashfusedmoe_b200 import linear_cross_entropy
    h = torch.zeros(rows, 8, device="cuda").bfloat16()
    h[:, 0] = 1.0
    h[:, 1] = 1.0
    w = torch.zeros(2, 8, device="cuda").bfloat16()
    w[:, 0] = size
    w[1, 1] = -10.0
    t = torch.zeros(rows, dtype=torch.int64, device="cuda")
    q = torch.exp(torch.tensor(-10.0, dtype=torch.float64, device="cuda"))
    with torch.no_grad():
        nll = linear_cross_entropy(h, w, t, reduction="none")
    assert ((nll.double() - torch.log1p(q)).abs() <= 16 * U).all()
    loss, dh, dw = run(h, w, t)
    assert (loss.double() - torch.log1p(q)).abs() <= 16 * U
    # dl = -(1 - p), 1 - p, each rounded to bf16, and so is their product with the rows' mean of 1 (times 1 / rows and rows times)
    share = q / (1 + q)
    for entry, sign in ((0, -1.0), (1, 1.0)):
        got = dw[entry, 0].double() * sign
        assert (got - share).abs() <= share * (2 * 2.0 ** -8 + 2.0 ** -10) + 16 * U


@pytest.mark.gpu
def test_gradients_of_entries_far_below_the_largest():
    """One entry dominates its piece of 128, others lie 1 to 26 nats below it, exactly. An exponential is held in fp16 as 2^15 of itself: 11 bits down to
    2^-29 (20 nats), steps of 2^-39 below. Beside that, dl is rounded once, to bf16 (2^-8), and everything in fp32 adds less than 2^-16:
    arguments of up to 38 in the exponential's base 2, rounded, are 38 u ln 2 of it. The products are with one row of ones."""
    below = torch.arange(1, 27, dtype=torch.float64, device="cuda")
    h = torch.zeros(1, 8, device="cuda").bfloat16()
    h[0, 0] = 1.0
    w = torch.zeros(300, 8, device="cuda").bfloat16()
    w[:, 0] = -100.0
    w[7, 0] = 0.0
    w[20:46, 0] = -below.bfloat16()
    t = torch.tensor([7], device="cuda")
    lse = torch.log1p(torch.exp(-below).sum())
    p = torch.exp(-below - lse)
    _, dh, dw = run(h, w, t)
    got = dw[20:46, 0].double()
    limit = p * (2.0 ** -11 + 2.0 ** -8 + 2.0 ** -16) + torch.where(below > 20, 2.0 ** -40, 0.0)
    assert ((got - p).abs() <= limit).all(), ((got - p).abs() / limit).tolist()
    assert (got > 0).all()
