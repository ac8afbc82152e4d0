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
