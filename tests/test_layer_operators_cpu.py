"""What the operators around the routed experts refuse, before anything is launched (CPU)."""

import types

import pytest
import torch

import dist_moe_b200 as dm
from dist_moe_b200 import _native as nat

BF, F32 = torch.bfloat16, torch.float32


def _t(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("error,match,args,options", [
    (TypeError, "x_TD", (_t(2, 8, dtype=F32), _t(8)), {}),
    (TypeError, "weight_D", (_t(2, 8), _t(8, dtype=torch.float16)), {}),
    (TypeError, "residual_TD", (_t(2, 8), _t(8)), dict(residual_TD=_t(2, 8, dtype=torch.float64))),
    (ValueError, "shape", (_t(8), _t(8)), {}),
    (ValueError, "shape", (_t(2, 0), _t(0)), {}),
    (ValueError, "weight_D", (_t(2, 8), _t(9)), {}),
    (ValueError, "residual_TD", (_t(2, 8), _t(8)), dict(residual_TD=_t(3, 8))),
    (ValueError, "CUDA", (_t(2, 8), _t(8)), {}),
])
def test_add_rms_norm(error, match, args, options):
    with pytest.raises(error, match=match):
        dm.add_rms_norm(*args, **options)


class _OnDevice(torch.Tensor):
    """A CPU tensor that says it lies on a GPU: for the checks behind that of the device."""

    device = torch.device("cuda", 0)


@pytest.mark.parametrize("options", [dict(eps=v) for v in (0.0, -1e-6, 1e-46, float("inf"), float("nan"), "1")]
                         + [dict(gain_center=v) for v in (1e39, float("-inf"), float("nan"))])
def test_add_rms_norm_numbers_that_float32_does_not_hold(options):
    """An eps that vanishes in float32 would make NaN of a row of zeros."""
    with pytest.raises(ValueError, match=next(iter(options))):
        dm.add_rms_norm(_t(2, 8).as_subclass(_OnDevice), _t(8).as_subclass(_OnDevice), **options)


@pytest.mark.parametrize("error,match,options", [
    (TypeError, "logits_TE", dict(logits=_t(2, 8, dtype=torch.float16))),
    (ValueError, "logits_TE", dict(logits=_t(8))),
    (ValueError, "1024", dict(logits=_t(1, 1025))),
    (ValueError, "1024", dict(logits=_t(1, 0))),
    (TypeError, "top_k", dict(top_k=True)),
    (TypeError, "num_groups", dict(num_groups=2.0)),
    (ValueError, "top_k", dict(top_k=0)),
    (ValueError, "top_k", dict(top_k=9)),
    (ValueError, "top_k", dict(logits=_t(2, 64), top_k=33)),
    (ValueError, "num_groups", dict(num_groups=3)),
    (ValueError, "num_groups", dict(logits=_t(2, 64), num_groups=64)),
    (ValueError, "num_kept_groups", dict(num_groups=4, num_kept_groups=5)),
    (ValueError, "group_top", dict(num_groups=4, num_kept_groups=2, group_top=3)),
    (ValueError, "kept groups", dict(num_groups=4, num_kept_groups=1, top_k=3)),
    (ValueError, "score", dict(score="tanh")),
    (TypeError, "renormalize", dict(renormalize=1)),
    (ValueError, "scale", dict(scale=float("inf"))),
    (ValueError, "scale", dict(scale=float("nan"))),
    (ValueError, "scale", dict(scale=1e39)),
    (TypeError, "ids_dtype", dict(ids_dtype=torch.int16)),
    (TypeError, "scores_dtype", dict(scores_dtype=torch.float16)),
    (TypeError, "bias_E", dict(bias_E=_t(8))),
    (ValueError, "bias_E", dict(bias_E=_t(7, dtype=F32))),
    (ValueError, "no gradient", dict(bias_E=_t(8, dtype=F32).requires_grad_())),
    (TypeError, "token_mask_T", dict(token_mask_T=_t(2, dtype=torch.uint8))),
    (ValueError, "token_mask_T", dict(token_mask_T=_t(3, dtype=torch.bool))),
    (ValueError, "CUDA", {}),
])
def test_select_experts(error, match, options):
    options = dict(options)
    with pytest.raises(error, match=match):
        dm.select_experts(options.pop("logits", _t(2, 8, dtype=F32)), options.pop("top_k", 2), **options)


def test_quantised_rows():
    for packed, dim, error in ((_t(2, 48, dtype=torch.uint8), 32, TypeError), (None, 32, TypeError), (_t(2, 48), 32, TypeError)):
        with pytest.raises(error):
            dm.QuantizedRows(packed, dim)


def _context(*, closed=False, block_scaled=None, ep=1, workspace=True):
    """A context without a device: what the checks in front of a launch look at."""
    ctx = object.__new__(dm.Context)
    ctx.config = dm.Config(max_num_local_input_tokens=100, hidden_dim=64, intermediate_dim=32, top_k=2, num_experts=4,
                           max_moe_layers_per_activation_slot=1, inference=True, block_scaled=block_scaled)
    ctx._closed = closed
    ctx._state = types.SimpleNamespace(ep=ep, e_local=4, device=torch.device("cuda", 0), few_workspace=object() if workspace else None)
    return ctx


def _call(ctx, **changed):
    args = dict(x=_t(3, 64), ids=_t(3, 2, dtype=torch.int32), scores=_t(3, 2, dtype=F32), w13=_t(4, 64, 64), w2=_t(4, 64, 32)) | changed
    return dm.routed_experts_few_tokens(args["x"], args["ids"], args["scores"], args["w13"], args["w2"], ctx)


@pytest.mark.parametrize("error,match,context,changed", [
    (RuntimeError, "closed", dict(closed=True), {}),
    (ValueError, "BF16 contexts", dict(block_scaled=dm.BlockScaledConfig()), {}),
    (ValueError, "one rank", dict(ep=2), {}),
    (TypeError, "x_TD", {}, dict(x=_t(3, 64, dtype=F32))),
    (ValueError, "x_TD", {}, dict(x=_t(3, 32))),
    (ValueError, "local tokens", {}, dict(x=_t(0, 64))),
    (ValueError, "local tokens", {}, dict(x=_t(101, 64))),
    (TypeError, "topk_expert_ids", {}, dict(ids=_t(3, 2, dtype=torch.int16))),
    (TypeError, "topk_scores", {}, dict(scores=_t(3, 2, dtype=torch.float16))),
    (ValueError, "shape", {}, dict(ids=_t(3, 3, dtype=torch.int32))),
    (TypeError, "weights", {}, dict(w13=_t(4, 64, 64, dtype=F32))),
    (ValueError, "hidden", {}, dict(w13=_t(4, 64, 32))),
    (ValueError, "CUDA", {}, {}),
])
def test_routed_experts_few_tokens(error, match, context, changed):
    with pytest.raises(error, match=match):
        _call(_context(**context), **changed)
    with pytest.raises(TypeError, match="create_context"):
        _call(object())


def test_entry_points_return_codes():
    """Bad arguments come back as codes: nothing is launched, no device is needed."""
    lib, some = nat.lib, 4096  # an address that nothing reads
    assert lib.dm_add_rmsnorm_fwd(None, 8, None, 0, 0, None, 0, 0.0, 1e-6, 1, 8, None, None, None, None, 0, None) == -1
    assert lib.dm_add_rmsnorm_fwd(some, 8, some, 0, 8, some, 0, 0.0, 1e-6, 1, 8, None, some, None, None, 0, None) == -1
    assert lib.dm_add_rmsnorm_fwd(some, 40, None, 0, 0, some, 0, 0.0, 1e-6, 1, 40, None, some, None, some, 48, None) == -2
    assert lib.dm_add_rmsnorm_fwd(some, 8, None, 0, 0, some, 0, 0.0, 1e-6, 0, 8, None, some, None, None, 0, None) == 0
    assert lib.dm_add_rmsnorm_bwd(None, None, None, 0, 8, None, 0, 0.0, None, 1, 8, None, None, None, None, None) == -1
    assert lib.dm_add_rmsnorm_bwd(some, None, some, 0, 8, some, 0, 0.0, some, 1, 8, some, None, some, None, None) == -1
    assert lib.dm_dequant_mxfp8_rows(some, 48, 1, 31, some, None) == -1 and lib.dm_dequant_mxfp8_rows(some, 32, 1, 32, some, None) == -1
    select = lambda **c: lib.dm_select_experts(*({**dict(  # noqa: E731
        logits=some, bf16=0, stride=8, T=1, E=8, K=2, sigmoid=0, bias=None, groups=1, kept=1, top=2, norm=0, scale=1.0, mask=None, ids=some,
        i64=0, scores=some, sbf16=0, stream=None), **c}.values()))
    assert select(T=0) == 0 and select(logits=None) == -1 and select(K=9) == -1 and select(E=64, K=33) == -1 and select(groups=3) == -1
    assert select(groups=2, kept=3) == -1 and select(top=3) == -1 and select(E=1025, K=2) == -3 and select(stride=-1) == -1
    assert lib.dm_select_experts_bwd(None, 0, 8, 1, 8, 2, 0, 0, 1.0, some, 0, some, 0, some, None) == -1
    size = lib.dm_few_tokens_workspace_bytes
    assert size(65, 64, 32, 4, 2) == -3 and size(1, 64, 32, 1025, 2) == -3 and size(1, 64, 32, 64, 33) == -3
    assert size(1, 64, 12, 4, 2) == -2 and size(1, 48, 16, 4, 2) == -2 and size(0, 64, 32, 4, 2) == -1 and size(64, 64, 32, 4, 2) > 0
    few = lambda x=some, ws=some, n=1 << 40, T=1, out=some: lib.dm_few_tokens(  # noqa: E731
        x, some, 0, some, 0, some, some, out, T, 64, 32, 4, 2, 0, 1.0, 0.0, ws, n, 0, None, None)
    assert few(x=None) == -1 and few(x=some + 8) == -1 and few(out=some + 2) == -1 and few(n=16) == -1 and few(T=65) == -3 and few(ws=None) == -1
