"""The refusal of forward-mode tangents (CPU; the operators' own calls are tested on a device)."""

import pytest
import torch
from torch.autograd import forward_ad

import dist_moe_b200 as dm
from dist_moe_b200._call import refuse_tangents


def test_a_tangent_is_found():
    x = torch.randn(3)
    refuse_tangents("op", x, None)
    with forward_ad.dual_level():
        refuse_tangents("op", x, None)
        dual = forward_ad.make_dual(x, x)
        with pytest.raises(RuntimeError, match="op has no forward-mode derivative"):
            refuse_tangents("op", None, dual)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            refuse_tangents("op", dual)
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda a: refuse_tangents("op", a) or a, (x,), (x,))


class _OnDevice(torch.Tensor):
    """A CPU tensor that says it lies on a GPU: for the checks behind that of the device."""

    device = torch.device("cuda", 0)


@pytest.mark.parametrize("which", range(3))
def test_the_norm_and_the_selection_look_for_one(which):
    on = [torch.ones(2, 8, dtype=torch.bfloat16), torch.ones(8), torch.ones(2, 8)]
    calls = [lambda a, w, l: dm.add_rms_norm(a, w), lambda a, w, l: dm.add_rms_norm(a, w, residual_TD=a), lambda a, w, l: dm.select_experts(l, 2)]
    with forward_ad.dual_level():
        on[which] = forward_ad.make_dual(on[which], torch.ones_like(on[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            calls[which](*(t.as_subclass(_OnDevice) for t in on))
