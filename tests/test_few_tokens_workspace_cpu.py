"""When a context takes the workspace of calls of few tokens (CPU)."""

import types

import pytest
import torch

import dist_moe_b200 as dm
from dist_moe_b200 import _few_tokens, _runtime


def _state(**more):
    cfg = dm.Config(max_num_local_input_tokens=100, hidden_dim=64, **{
        **dict(intermediate_dim=32, top_k=2, num_experts=4, max_moe_layers_per_activation_slot=1), **more})
    return types.SimpleNamespace(config=cfg, device=torch.device("cpu"), few_workspace=None, gather_flags=torch.ones(3),
                                 **{k: None for k in ("_native_layer",)})


@pytest.mark.parametrize("capturing", [False, True])
def test_taken_by_the_first_call_and_left_to_a_graph(capturing, monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    state = _state()
    ws = _few_tokens.workspace(state)
    assert ws.numel() == _few_tokens.workspace_bytes(state) > _few_tokens.COUNTER_BYTES and not ws[:_few_tokens.COUNTER_BYTES].any()
    assert (state.few_workspace is ws) == (not capturing)
    again = _few_tokens.workspace(state)
    assert (again is ws) == (not capturing) and not again[:_few_tokens.COUNTER_BYTES].any()


def test_counters_are_cleared_where_there_are_some():
    state = _state()
    _runtime.ContextState.clear_gather_flags(state)
    state.gather_flags.fill_(1)
    state.few_workspace = torch.ones(2 * _few_tokens.COUNTER_BYTES, dtype=torch.uint8)
    _runtime.ContextState.clear_gather_flags(state)
    assert not state.gather_flags.any() and not state.few_workspace[:_few_tokens.COUNTER_BYTES].any()
    assert state.few_workspace[_few_tokens.COUNTER_BYTES:].all()


def test_sizes_that_are_not_offered():
    assert _few_tokens.workspace_bytes(_state(intermediate_dim=60)) < 0 and _few_tokens.workspace_bytes(_state(num_experts=1025)) < 0


def test_a_first_call_in_inference_mode_leaves_counters_that_can_be_cleared_outside_it(monkeypatch):
    """An inference tensor may not be written outside of that mode, and the context clears its counters there."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    state = _state()
    with torch.inference_mode():
        _few_tokens.workspace(state)
    state.few_workspace.fill_(1)
    _runtime.ContextState.clear_gather_flags(state)
    assert not state.few_workspace[:_few_tokens.COUNTER_BYTES].any()
