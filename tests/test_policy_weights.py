"""Weights of the policy loss that are no finite numbers."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [5, 3000])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_a_weight_that_is_not_finite_shows(bad, reduction, rows):
    """inf / inf is no number, nor is anything that a NaN is part of; a finite weight over an infinite sum is zero."""
    from mccl_b200.ops.loss import fused_policy_loss
    torch.manual_seed(0)
    z = torch.randn(rows, 300, device="cuda", dtype=torch.float32, requires_grad=True)
    tokens = torch.randint(0, 300, (rows,), device="cuda")
    old = torch.log_softmax(z.detach(), 1).gather(1, tokens[:, None])[:, 0]
    adv, w = torch.randn(rows, device="cuda") + 3 * torch.sign(torch.randn(rows, device="cuda")), torch.rand(rows, device="cuda") + 0.5
    w[2] = bad
    loss, _ = fused_policy_loss(z, tokens, old, adv, weights=w, reduction=reduction)
    (g,) = torch.autograd.grad(loss, z)
    over = w.double().sum() if reduction == "mean" else 1.0
    terms = -adv.double() * w.double()                       # the ratio is one
    want = terms.sum() / over
    assert torch.isnan(want) == torch.isnan(loss) and (torch.isnan(want) or want == loss.double())
    assert not torch.isfinite(g[2]).any()
    others = torch.arange(rows, device="cuda") != 2
    if bad != bad and reduction == "mean":                   # every row over a sum that is no number
        assert torch.isnan(g).all()
    elif reduction == "mean":
        assert (g[others] == 0).all()
    else:
        assert torch.isfinite(g[others]).all() and (g[others] != 0).any(1).all()
