"""Log probabilities of given tokens, entropies and top alternatives of logits
(starkv_token_logprobs in include/starkv.h)."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import LogprobsDesc, StarKVError
from .ops import _dt, _launch, _out

__all__ = ["TokenLogprobs", "token_logprobs", "MAX_TOP"]

MAX_TOP = 64                         # STARKV_MAX_TOP
MAX_ROWS = 1 << 30                   # of one call (fewer where rows are many: the library says)


class TokenLogprobs(NamedTuple):
    logprob: Optional[torch.Tensor]  # [...] fp32; None without tokens
    entropy: torch.Tensor            # [...] fp32, nats
    top_logprobs: torch.Tensor       # [..., top] fp32, descending
    top_ids: torch.Tensor            # [..., top] int64


def token_logprobs(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, top: int = 0) -> TokenLogprobs:
    """log_softmax(logits [..., V])[token] for ``tokens`` [...] (int64), each
    row's entropy, and its ``top`` most probable tokens with their log
    probabilities (equal logits by ascending index), in one pass over the
    logits (fp16, bf16 or fp32; rows at any alignment).  Logits of -inf are
    barred tokens.  A token outside [0, V) has the log probability NaN, and so
    has everything of a row without a finite logit or with a NaN or +inf."""
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise StarKVError(f"logits must be [..., V], got shape {tuple(logits.shape)}")
    dev, v, lead = logits.device, logits.shape[-1], logits.shape[:-1]
    if lead.numel() > MAX_ROWS:
        raise StarKVError(f"logits have more than {MAX_ROWS} rows: {tuple(logits.shape)}")
    if dev.type != "cuda":
        raise StarKVError("libstarkv operators take device tensors (there is no CPU path)")
    if not 0 <= top <= min(MAX_TOP, v):
        raise StarKVError(f"top must be 0 .. min({MAX_TOP}, V = {v}), got {top}")
    if v > 1 and logits.stride(-1) != 1:
        raise StarKVError("logits must have a contiguous last dim")
    rows = logits
    if rows.dim() != 2:
        try:
            rows = rows.view(-1, v) if rows.numel() else rows.reshape(0, v)
        except RuntimeError:
            raise StarKVError("logits rows must be addressable with one row stride") from None
    n = rows.shape[0]
    if tokens is not None:
        if tokens.shape != lead or tokens.dtype != torch.int64 or tokens.device != dev:
            raise StarKVError(f"tokens must be int64 {tuple(lead)} on {dev}, got {tokens.dtype} {tuple(tokens.shape)} "
                              f"on {tokens.device}")
        if not tokens.is_contiguous():
            tokens = tokens.contiguous()
    lp = _out(lead, dtype=torch.float32, device=dev) if tokens is not None else None
    ent = _out(lead, dtype=torch.float32, device=dev)
    tops = _out(*lead, top, dtype=torch.float32, device=dev)
    ids = _out(*lead, top, dtype=torch.int64, device=dev)
    d = LogprobsDesc(n, v, _dt(logits), top, rows.data_ptr(), rows.stride(0) if n > 1 else v,
                     None if tokens is None else tokens.data_ptr(), None if lp is None else lp.data_ptr(),
                     ent.data_ptr(), tops.data_ptr(), ids.data_ptr())
    _launch("starkv_token_logprobs", d, dev, workspace=True)
    return TokenLogprobs(lp, ent, tops, ids)
