"""Verification of drafted tokens from given random numbers, and drafting
from the tokens already there.

riallm decodes greedily, one token per forward (src/model.rs:1223-1270; its
temperature and top_p are accepted and unused).
"""
from __future__ import annotations

from typing import Dict, List, Optional, Sequence, Tuple, Union

import torch

from . import ConfigError, Context, _act_dtype, lib

# Workspace bytes by call shape.
_workspace: Dict[Tuple[int, ...], int] = {}


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ConfigError("verify_draft: " + what)


def verify_draft(logits: torch.Tensor, draft_tokens: Optional[torch.Tensor], accept_u: Optional[torch.Tensor],
                 sample_u: torch.Tensor, temperature: Union[float, torch.Tensor] = 1.0,
                 draft_probs: Optional[torch.Tensor] = None,
                 ctx: Optional[Context] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Verifies n drafted tokens per sequence against the model's logits
    [B, n + 1, V] (float32 or bf16) and takes one more token.

    draft_tokens [B, n] int32 (one outside [0, V) ends its sequence's
    drafts), accept_u [B, n] and sample_u [B] float32 uniforms in [0, 1),
    temperature a number or float32 [B] (0: greedy), draft_probs the
    distributions [B, n, V] float32 that the drafts were drawn from (None:
    each was chosen outright). With n == 0, draft_tokens and accept_u may be
    None: one token per sequence is sampled.

    Returns (tokens int32 [B, n + 1]: the accepted drafts, the token taken
    after them, then -1; accepted int32 [B]). The definition is
    riallm_cuda_verify_draft's (include/riallm_cuda.h)."""
    _need(logits.is_cuda and logits.dim() == 3 and logits.is_contiguous() and logits.shape[1] > 0,
          "logits must be a contiguous CUDA tensor [B, n + 1, V]")
    B, n1, V = logits.shape
    n, dev = n1 - 1, logits.device

    def check(t, dtype, shape, name):
        _need(t.dtype is dtype and t.shape == shape and t.is_contiguous() and t.device == dev,
              f"{name} must be contiguous {dtype} {list(shape)} on the logits' device")

    if n or draft_tokens is not None:
        _need(draft_tokens is not None and accept_u is not None, "draft_tokens and accept_u are wanted")
        check(draft_tokens, torch.int32, (B, n), "draft_tokens")
        check(accept_u, torch.float32, (B, n), "accept_u")
    check(sample_u, torch.float32, (B,), "sample_u")
    if draft_probs is not None:
        check(draft_probs, torch.float32, (B, n, V), "draft_probs")
    if not isinstance(temperature, torch.Tensor):
        temperature = torch.full((B,), float(temperature), dtype=torch.float32, device=dev)
    check(temperature, torch.float32, (B,), "temperature")
    tokens = torch.empty((B, n1), dtype=torch.int32, device=dev)
    accepted = torch.empty((B,), dtype=torch.int32, device=dev)
    ctx = ctx or Context.get(dev.index)
    _need(ctx.device == dev.index, "the context is another device's")
    L = lib()
    key = (dev.index, B, n, V)
    size = _workspace.get(key)
    if size is None:
        if len(_workspace) > 4096:
            _workspace.clear()
        size = _workspace[key] = L.riallm_cuda_verify_draft_workspace(ctx.ptr, B, n, V)
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    ctx.check(L.riallm_cuda_verify_draft(
        ctx.ptr, logits.data_ptr(), _act_dtype(logits.dtype), draft_tokens.data_ptr() if n else None,
        draft_probs.data_ptr() if draft_probs is not None and n else None, temperature.data_ptr(),
        accept_u.data_ptr() if n else None, sample_u.data_ptr(), B, n, V, tokens.data_ptr(), accepted.data_ptr(),
        ws.data_ptr() if ws is not None else None, size, torch.cuda.current_stream(dev).cuda_stream))
    return tokens, accepted


def lookup_drafts(tokens: Sequence[int], n: int, match: int = 2) -> List[int]:
    """Up to n drafts for a sequence from its own tokens: what followed the
    latest earlier place of its last `match` tokens (of fewer, down to one,
    where there is none)."""
    tokens = list(tokens)
    for m in range(min(match, len(tokens) - 1), 0, -1):
        tail = tokens[-m:]
        for i in range(len(tokens) - m - 1, -1, -1):
            if tokens[i:i + m] == tail:
                return tokens[i + m:i + m + n]
    return []
