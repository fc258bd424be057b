"""Gradients of ``fused_dropout`` that are to be differentiated again."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("unit", ["element", "channel", "sample"])
@pytest.mark.parametrize("create_graph", [False, True])
def test_what_the_relu_stops_is_zero_whatever_it_was(unit, create_graph):
    """As without a graph of the gradient: zero, where a product with the mask would be NaN."""
    from pointelligence_b200.layers.dropout import fused_dropout

    x = torch.randn(60, 16, device=DEV).requires_grad_()
    res = torch.randn(60, 16, device=DEV).requires_grad_()
    y = fused_dropout(x, 0.5, rng=(3, 4), unit=unit, lengths=torch.tensor([40, 20], device=DEV), residual=res, relu=True)
    go = torch.where(y.detach() > 0, torch.ones_like(y), torch.tensor(float("inf"), device=DEV))
    go[y.detach() <= 0] = torch.where(torch.rand_like(go) < 0.5, go, torch.full_like(go, float("nan")))[y.detach() <= 0]
    dx, dres = torch.autograd.grad(y, (x, res), go, create_graph=create_graph)
    assert torch.equal(dres.detach(), (y.detach() > 0).float())
    kept = fused_dropout(torch.ones_like(x), 0.5, rng=(3, 4), unit=unit, lengths=torch.tensor([40, 20], device=DEV)).detach()
    assert torch.equal(dx.detach(), kept * (y.detach() > 0))
