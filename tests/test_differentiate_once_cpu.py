"""Gradients of the norm and of the selection asked for with ``create_graph=True``: whatever the incoming gradients are, they are tied
to what they depend on by a node that raises.  The host side on the CPU, its launches replaced (the values do not matter)."""

import types

import pytest
import torch

from dist_moe_b200 import _native as nat
from dist_moe_b200 import _call, _norm, _selection


@pytest.fixture(autouse=True)
def no_device(monkeypatch):
    ok = lambda *a: 0  # noqa: E731
    monkeypatch.setattr(nat, "lib", types.SimpleNamespace(
        dm_add_rmsnorm_fwd=ok, dm_add_rmsnorm_bwd=ok, dm_add_rmsnorm_shares=lambda T, D: 2, dm_select_experts=ok, dm_select_experts_bwd=ok))
    monkeypatch.setattr(nat, "stream_ptr", lambda: 0)
    for module in (_norm, _selection):
        monkeypatch.setattr(module, "on_device", lambda device: _call._NOTHING)
    # the launches write nothing: zeros, so that nothing is NaN by chance
    monkeypatch.setattr(torch, "empty", lambda *a, **k: torch.zeros(*a, **k))
    monkeypatch.setattr(torch, "empty_like", lambda *a, **k: torch.zeros_like(*a, **k))


def _norm_case(residual, needs):
    leaves = dict(x=torch.ones(3, 8, dtype=torch.bfloat16), residual=torch.ones(3, 8, dtype=residual) if residual else None,
                  weight=torch.ones(8))
    for name in needs:
        leaves[name].requires_grad_()
    got = _norm._AddRmsNorm.apply(leaves["x"], leaves["residual"], leaves["weight"], 1e-6, 0.0)
    return (got if residual else (got,)), [leaves[n] for n in needs]


@pytest.mark.parametrize("residual", [None, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("needs", [("x",), ("weight",), ("x", "weight")])
@pytest.mark.parametrize("incoming", ["ones", "given", "differentiable"])
def test_norm(residual, needs, incoming):
    outputs, leaves = _norm_case(residual, needs)
    given = [torch.ones_like(o, requires_grad=incoming == "differentiable") for o in outputs]
    grads = torch.autograd.grad(outputs, leaves, given, create_graph=True) if incoming != "ones" else \
        torch.autograd.grad(sum(o.sum() for o in outputs), leaves, create_graph=True)
    if needs == ("weight",) and incoming != "differentiable":  # the gain's gradient does not depend on the gain
        assert not grads[0].requires_grad
        return
    assert all(g.requires_grad for g in grads)
    wanted = given if needs == ("weight",) else leaves
    # beside a path of its own: without the tie the second derivative would be left out in silence
    with pytest.raises(RuntimeError, match="differentiate twice"):
        torch.autograd.grad(sum(g.float().pow(2).sum() for g in grads) + sum(t.sum() for t in wanted), wanted)
    outputs, leaves = _norm_case(residual, needs)
    plain = torch.autograd.grad(sum(o.sum() for o in outputs), leaves)
    assert not any(g.requires_grad for g in plain)


def test_norm_by_the_sum_alone():
    """The sum is linear: its gradients are PyTorch's own operations, and are differentiated as such."""
    (_, total), (x, weight) = _norm_case(torch.float32, ("x", "weight"))
    gx, gw = torch.autograd.grad(total.sum(), (x, weight), create_graph=True)
    assert torch.equal(gx, torch.ones_like(x)) and not gw.any()
    assert torch.equal(torch.autograd.grad(gx.sum() + x.sum() + gw.sum(), x)[0], torch.ones_like(x))
    incoming = torch.ones(3, 8, requires_grad=True)
    (_, total), (x, weight) = _norm_case(torch.float32, ("x", "weight"))
    gx, = torch.autograd.grad(total, x, incoming, create_graph=True)
    assert torch.equal(torch.autograd.grad(gx, incoming, 3 * torch.ones_like(gx))[0], torch.full_like(incoming, 3.0))


def _select_case():
    logits = torch.ones(3, 8, requires_grad=True)
    options = (2, False, None, 1, 1, 2, False, 1.0, None, torch.int32, torch.float32)
    return _selection._SelectExperts.apply(logits, options)[1], logits


@pytest.mark.parametrize("incoming", ["ones", "given", "differentiable"])
def test_selection(incoming):
    scores, logits = _select_case()
    given = torch.ones_like(scores, requires_grad=incoming == "differentiable")
    grad, = torch.autograd.grad(scores, logits, given, create_graph=True) if incoming != "ones" else \
        torch.autograd.grad(scores.sum(), logits, create_graph=True)
    assert grad.requires_grad
    with pytest.raises(RuntimeError, match="differentiate twice"):
        torch.autograd.grad(grad.pow(2).sum() + logits.sum(), logits)
    scores, logits = _select_case()
    assert not torch.autograd.grad(scores.sum(), logits)[0].requires_grad


def test_gradients_may_be_accumulated_and_changed_in_place():
    outputs, leaves = _norm_case(torch.float32, ("x", "weight"))
    sum(o.sum() for o in outputs).backward(create_graph=True)
    with torch.no_grad():
        for t in leaves:
            t.grad.mul_(2).zero_()
            t.grad = None
