"""The routed-expert layer for a decode step of few tokens: host side of ``dm_few_tokens`` (csrc/few_tokens.cu)."""

from __future__ import annotations

import torch

from . import _native as nat
from ._call import on_device

MAX_TOKENS = 64  # DM_FEW_TOKENS_MAX
COUNTER_BYTES = 8192  # DM_FEW_TOKENS_COUNTER_BYTES


def workspace_bytes(state) -> int:
    """Not positive where calls of few tokens are not offered for the context's sizes."""
    cfg = state.config
    return nat.lib.dm_few_tokens_workspace_bytes(min(MAX_TOKENS, cfg.max_num_local_input_tokens), cfg.hidden_dim, cfg.intermediate_dim,
                                                 cfg.num_experts, cfg.top_k)


def workspace(state) -> torch.Tensor:
    """The context's workspace, taken by its first call; the context clears its counters from then on.  A graph that is captured before
    has one of its own in its memory pool, cleared by every replay: an eager call may come in between."""
    ws = state.few_workspace
    if ws is None:
        with torch.inference_mode(False):  # the context clears it outside of that mode too
            ws = torch.empty(workspace_bytes(state), dtype=torch.uint8, device=state.device)
            ws[:COUNTER_BYTES].zero_()
        if not torch.cuda.is_current_stream_capturing():
            state.few_workspace = ws
    return ws


def checked_run(x, ids, scores, w13, w2, context) -> torch.Tensor:
    from .api import _few_tokens_arguments

    return run(*_few_tokens_arguments(x, ids, scores, w13, w2, context), context._state)


def run(x, ids, scores, w13, w2, state) -> torch.Tensor:
    if x.data_ptr() % 16:
        x = x.clone()
    w13_ptr, w2_ptr = w13.data_ptr(), w2.data_ptr()
    if w13_ptr % 16 or w2_ptr % 16:
        raise ValueError("w13_EFD and w2_EDF must start on a 16-byte boundary")
    with on_device(state.device):
        cfg, ws = state.config, state.few_workspace
        if ws is None:
            ws = workspace(state)
        out = torch.empty_like(x)
        nat.check(nat.lib.dm_few_tokens(
            x.data_ptr(), ids.data_ptr(), ids.dtype is torch.int64, scores.data_ptr(), scores.dtype is torch.bfloat16, w13_ptr,
            w2_ptr, out.data_ptr(), x.shape[0], cfg.hidden_dim, cfg.intermediate_dim, cfg.num_experts, cfg.top_k,
            cfg.activation == "swiglu_clamped", cfg.swiglu_alpha, cfg.swiglu_limit, ws.data_ptr(), ws.numel(), state.num_sms,
            state.status.data_ptr(), nat.stream_ptr()), "dm_few_tokens")
    return out
