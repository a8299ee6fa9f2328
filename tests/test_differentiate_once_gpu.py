"""Gradients taken with ``create_graph=True`` and constant incoming gradients: the same bits, and an error where they are differentiated."""

import pytest
import torch

import dist_moe_b200 as dm

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("residual", [None, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("transposed", [False, True])
def test_norm(residual, transposed):
    x = torch.randn(5, 256, device=DEV).bfloat16()
    x = (x.t().contiguous().t() if transposed else x).requires_grad_()
    w = torch.randn(256, device=DEV, requires_grad=True)
    r = None if residual is None else torch.randn(5, 256, device=DEV).to(residual)
    y, total = dm.add_rms_norm(x, w, residual_TD=r)
    first = torch.autograd.grad(y.sum(), (x, w), retain_graph=True)
    again = torch.autograd.grad(y.sum(), (x, w), create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    for g, ask in ((again[0], x), (again[0], w), (again[1], x)):  # the gain's gradient does not depend on the gain
        with pytest.raises(RuntimeError, match="differentiate twice"):
            torch.autograd.grad(g.float().pow(2).sum() + x.sum() + w.sum(), ask, retain_graph=True)


def test_selection():
    logits = torch.randn(5, 16, device=DEV, requires_grad=True)
    scores = dm.select_experts(logits, 4)[1]
    first, = torch.autograd.grad(scores.sum(), logits, retain_graph=True)
    again, = torch.autograd.grad(scores.sum(), logits, create_graph=True)
    assert torch.equal(first, again)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        (again.pow(2).sum() + logits.sum()).backward()
