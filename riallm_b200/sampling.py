"""Verification of drafted tokens from given random numbers, and drafting
from the tokens already there.

riallm decodes greedily, one token per forward (src/model.rs:1223-1270; its
temperature and top_p are accepted and unused).
"""
from __future__ import annotations

import struct
from typing import Dict, List, Optional, Sequence, Tuple, Union

import torch

from . import ConfigError, Context, lib
from .paged import _context, _stream

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
_VERIFY = struct.Struct("@8P4i")  # riallm_verify_draft_args

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
    dev = logits.get_device()
    _need(dev >= 0 and logits.dim() == 3 and logits.is_contiguous() and logits.shape[1] > 0,
          "logits must be a contiguous CUDA tensor [B, n + 1, V]")
    dtype = _DTYPES.get(logits.dtype)
    _need(dtype is not None, "logits must be float32 or bf16")
    B, n1, V = logits.shape
    n, device, f32 = n1 - 1, logits.device, torch.float32

    if not isinstance(temperature, torch.Tensor):
        temperature = torch.full((B,), float(temperature), dtype=f32, device=device)
    rows, drafts = (B,), (B, n)
    # A step of a small model is a few launches long: what holds costs little,
    # and the message is worked out only for what does not.
    if not (sample_u.dtype is f32 and sample_u.shape == rows and sample_u.get_device() == dev
            and sample_u.is_contiguous()
            and temperature.dtype is f32 and temperature.shape == rows and temperature.get_device() == dev
            and temperature.is_contiguous()
            and (draft_tokens is accept_u is None and n == 0 or draft_tokens is not None and accept_u is not None
                 and draft_tokens.dtype is torch.int32 and draft_tokens.shape == drafts
                 and draft_tokens.get_device() == dev and draft_tokens.is_contiguous()
                 and accept_u.dtype is f32 and accept_u.shape == drafts and accept_u.get_device() == dev
                 and accept_u.is_contiguous())
            and (draft_probs is None or draft_probs.dtype is f32 and draft_probs.shape == (B, n, V)
                 and draft_probs.get_device() == dev and draft_probs.is_contiguous())):
        def check(t, dtype, shape, name):
            if not (t.dtype is dtype and t.shape == shape and t.get_device() == dev and t.is_contiguous()):
                raise ConfigError(f"verify_draft: {name} must be contiguous {dtype} {list(shape)} on the logits' "
                                  "device")

        if n or draft_tokens is not None:
            _need(draft_tokens is not None and accept_u is not None, "draft_tokens and accept_u are wanted")
            check(draft_tokens, torch.int32, drafts, "draft_tokens")
            check(accept_u, f32, drafts, "accept_u")
        check(sample_u, f32, rows, "sample_u")
        check(temperature, f32, rows, "temperature")
        if draft_probs is not None:
            check(draft_probs, f32, (B, n, V), "draft_probs")
    if n:
        tokens, accepted = draft_tokens.new_empty((B, n1)), draft_tokens.new_empty(B)
    else:
        tokens, accepted = (torch.empty(x, dtype=torch.int32, device=device) for x in ((B, n1), B))
    ctx = _context("verify_draft", ctx, dev)
    L = lib()
    key = (dev, B, n, V)
    size = _workspace.get(key)
    if size is None:
        if len(_workspace) > 4096:
            _workspace.clear()
        size = _workspace[key] = L.riallm_cuda_verify_draft_workspace(ctx.ptr, B, n, V)
    ws = sample_u.new_empty((size + 3) // 4)  # per call, in its stream's order
    try:
        args = _VERIFY.pack(logits.data_ptr(), draft_tokens.data_ptr() if n else 0,
                            draft_probs.data_ptr() if draft_probs is not None and n else 0, temperature.data_ptr(),
                            accept_u.data_ptr() if n else 0, sample_u.data_ptr(), tokens.data_ptr(),
                            accepted.data_ptr(), dtype, B, n, V)
    except struct.error:
        raise ConfigError("verify_draft: sizes must be 32-bit integers") from None
    status = L.riallm_cuda_verify_draft(ctx.ptr, args, ws.data_ptr(), size, _stream(dev))
    if status:
        ctx.check(status)
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
