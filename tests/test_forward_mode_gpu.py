"""Tangents of forward-mode differentiation are refused, not dropped."""

import pytest
import torch
from torch.autograd import forward_ad

import dist_moe_b200 as dm

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _few():
    T, D, F, E, K = 3, 64, 32, 4, 2
    ctx = dm.create_context(group=None, device=DEV, config=dm.Config(
        max_num_local_input_tokens=T, hidden_dim=D, intermediate_dim=F, top_k=K, num_experts=E, max_moe_layers_per_activation_slot=1,
        inference=True))
    ids = torch.arange(K, device=DEV).expand(T, K).contiguous()
    tensors = [torch.randn(*s, device=DEV).bfloat16() for s in ((T, D), (T, K), (E, 2 * F, D), (E, D, F))]
    return ctx, tensors, lambda x, s, w13, w2: dm.routed_experts_few_tokens(x, ids, s, w13, w2, ctx)


def _cases():
    x, r, w = torch.randn(3, 64, device=DEV).bfloat16(), torch.randn(3, 64, device=DEV), torch.randn(64, device=DEV)
    yield "add_rms_norm", (x, r, w), lambda a, b, c: dm.add_rms_norm(a, c, residual_TD=b)
    yield "add_rms_norm", (x, w), lambda a, c: dm.add_rms_norm(a, c, quantize=True)[0]
    yield "select_experts", (torch.randn(3, 8, device=DEV), torch.randn(8, device=DEV)), lambda l, b: dm.select_experts(l, 2, bias_E=b)[1]
    ctx, tensors, call = _few()
    yield "few_tokens", tensors, call
    ctx.close()


def test_tangents_are_refused():
    for name, tensors, call in _cases():
        for i, t in enumerate(tensors):
            with forward_ad.dual_level():
                call(*tensors)  # a level alone does no harm
                mixed = list(tensors)
                mixed[i] = forward_ad.make_dual(t, torch.ones_like(t))
                with pytest.raises(RuntimeError, match=f"{name}.*forward-mode"):
                    call(*mixed)
                call(*(a.detach() for a in tensors))
            with pytest.raises(RuntimeError, match=f"{name}.*forward-mode"):
                torch.func.jvp(lambda a: call(*tensors[:i], a, *tensors[i + 1:]), (t,), (torch.ones_like(t),))
