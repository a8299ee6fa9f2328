"""The routed-expert layer for a decode step of few tokens: host side of ``dm_few_tokens`` (csrc/few_tokens.cu)."""

from __future__ import annotations

import torch

from . import _native as nat

MAX_TOKENS = 64  # DM_FEW_TOKENS_MAX
COUNTER_BYTES = 8192  # DM_FEW_TOKENS_COUNTER_BYTES


def workspace(state) -> torch.Tensor | None:
    """What a context keeps for calls of few tokens, None where they are not offered.  The context clears its counters."""
    cfg = state.config
    if state.ep != 1 or state.block_scaled:
        return None
    nbytes = nat.lib.dm_few_tokens_workspace_bytes(min(MAX_TOKENS, cfg.max_num_local_input_tokens), cfg.hidden_dim,
                                                   cfg.intermediate_dim, cfg.num_experts, cfg.top_k)
    return torch.empty(nbytes, dtype=torch.uint8, device=state.device) if nbytes > 0 else None


def run(x, ids, scores, w13, w2, state) -> torch.Tensor:
    cfg, ws = state.config, state.few_workspace
    out = torch.empty_like(x)
    nat.check(nat.lib.dm_few_tokens(
        x.data_ptr(), ids.data_ptr(), ids.dtype is torch.int64, scores.data_ptr(), scores.dtype is torch.bfloat16, w13.data_ptr(),
        w2.data_ptr(), out.data_ptr(), x.shape[0], cfg.hidden_dim, cfg.intermediate_dim, cfg.num_experts, cfg.top_k,
        cfg.activation == "swiglu_clamped", cfg.swiglu_alpha, cfg.swiglu_limit, ws.data_ptr(), ws.numel(), state.num_sms,
        state.status.data_ptr(), nat.stream_ptr()), "dm_few_tokens")
    return out
