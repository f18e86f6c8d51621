"""Log probabilities of given tokens, entropies and top alternatives of logits
(starkv_token_logprobs in include/starkv.h)."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import LogprobsDesc, StarKVError
from .ops import _launch, _out

__all__ = ["TokenLogprobs", "token_logprobs", "MAX_TOP"]

MAX_TOP = 64                         # STARKV_MAX_TOP
_TYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}
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
    shape, dev, dt = logits.shape, logits.device, _TYPES.get(logits.dtype)
    if not shape or shape[-1] < 1:
        raise StarKVError(f"logits must be [..., V], got shape {tuple(shape)}")
    v, lead, stride = shape[-1], shape[:-1], logits.stride()
    n = lead.numel()
    if n > MAX_ROWS:
        raise StarKVError(f"logits have more than {MAX_ROWS} rows: {tuple(shape)}")
    if dev.type != "cuda":
        raise StarKVError("libstarkv operators take device tensors (there is no CPU path)")
    if dt is None:
        raise StarKVError(f"unsupported dtype {logits.dtype}")
    if not 0 <= top <= MAX_TOP or top > v:
        raise StarKVError(f"top must be 0 .. min({MAX_TOP}, V = {v}), got {top}")
    if v > 1 and stride[-1] != 1:
        raise StarKVError("logits must have a contiguous last dim")
    if len(lead) == 1:
        step = stride[0]
    elif n < 2:
        step = v
    else:
        try:
            step = logits.view(-1, v).stride(0)
        except RuntimeError:
            raise StarKVError("logits rows must be addressable with one row stride") from None
    tp = lp = lpp = None
    size = lead or ((),)
    if tokens is not None:
        if tokens.shape != lead or tokens.dtype != torch.int64 or tokens.device != dev:
            raise StarKVError(f"tokens must be int64 {tuple(lead)} on {dev}, got {tokens.dtype} {tuple(tokens.shape)} "
                              f"on {tokens.device}")
        if not tokens.is_contiguous():
            tokens = tokens.contiguous()
        lp = _out(*size, dtype=torch.float32, device=dev)
        tp, lpp = tokens.data_ptr(), lp.data_ptr()
    ent = _out(*size, dtype=torch.float32, device=dev)
    tops = _out(*lead, top, dtype=torch.float32, device=dev)
    ids = _out(*lead, top, dtype=torch.int64, device=dev)
    d = LogprobsDesc(n, v, dt, top, logits.data_ptr(), step if n > 1 else v, tp, lpp, ent.data_ptr(), tops.data_ptr(),
                     ids.data_ptr())
    _launch("starkv_token_logprobs", d, dev, workspace=True)
    return TokenLogprobs(lp, ent, tops, ids)
