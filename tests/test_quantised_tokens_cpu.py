"""Quantised tokens of a call on two ranks: what is checked before anything is launched, and what is handed on (CPU, fake tensors)."""

import types

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import dist_moe_b200 as dm
from dist_moe_b200 import _blockscaled, _call

T, D, F, E, K, RANKS = 5, 64, 32, 4, 2, 2


def _context(**more):
    ctx = object.__new__(dm.Context)
    ctx.config = dm.Config(**{**dict(max_num_local_input_tokens=8, hidden_dim=D, intermediate_dim=F, top_k=K, num_experts=E,
                                     max_moe_layers_per_activation_slot=1, inference=True, block_scaled=dm.BlockScaledConfig()), **more})
    ctx._closed = False
    ctx._state = types.SimpleNamespace(ep=RANKS, e_local=E // RANKS, device=torch.device("cuda", 0), config=ctx.config)
    return ctx


@pytest.fixture
def call(monkeypatch):
    handed = []
    monkeypatch.setattr(_call, "on_device", lambda device: _call._NOTHING)
    monkeypatch.setattr(_blockscaled, "run_block_scaled", lambda x, *a, **k: handed.append((x, k)))

    def run(ctx, rows=(T, 80), dim=D, gradient=False, **changed):
        with FakeTensorMode():
            on = dict(device="cuda:0")
            args = dict(ids=torch.empty(T, K, dtype=torch.int32, **on), scores=torch.empty(T, K, **on),
                        w13=torch.empty(E // RANKS, 2 * F, D, dtype=torch.bfloat16, **on),
                        w2=torch.empty(E // RANKS, D, F, dtype=torch.bfloat16, **on)) | changed
            if gradient:
                args["scores"].requires_grad_()
            tokens = dm.QuantizedRows(torch.empty(*rows, dtype=torch.uint8, **on), dim)
            dm.routed_experts(tokens, args["ids"], args["scores"], args["w13"], args["w2"], ctx)
        return tokens, handed

    return run


def test_rows_are_handed_on_as_they_are(call):
    tokens, handed = call(_context())
    (x, options), = handed
    assert x is tokens and options["save_for_backward"] is False


@pytest.mark.parametrize("error,match,context,changed", [
    (ValueError, "hidden dimension", {}, dict(rows=(T, 48), dim=32)),
    (ValueError, "tokens", {}, dict(rows=(9, 80))),
    (ValueError, "shape", {}, dict(rows=(T - 1, 80))),
    (ValueError, "local experts", {}, dict(w13=torch.empty(E, 2 * F, D, dtype=torch.bfloat16))),
    (ValueError, "MXFP8 context", dict(block_scaled=None), {}),
])
def test_refusals(call, error, match, context, changed):
    with pytest.raises(error, match=match):
        call(_context(**context), **changed)


def test_gradients_are_refused(call):
    with pytest.raises(RuntimeError, match="forward-only"):
        call(_context(inference=False), gradient=True)
