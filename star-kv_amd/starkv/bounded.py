"""Caches bounded by what their positions are worth: attention weights summed by position, the positions kept, and
their rows moved together (starkv_attention_scores, starkv_select_positions and starkv_keep_positions in
include/starkv.h)."""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from ._lib import KeepDesc, ScoresDesc, SelectDesc, StarKVError
from .ops import KLatentSpec, _check_scores, _dt, _flag_ptr, _launch, _out, _require_cuda, _vspec

__all__ = ["attention_scores", "select_positions", "keep_positions"]

_TYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}


def attention_scores(logits: torch.Tensor, scores: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Each position's attention weights summed over the heads: softmax over
    the last dim of ``logits`` [B, H, S] (fp16, bf16 or fp32), added over H in
    fp32.  ``scores`` [B, >= S] fp32: they are added onto it, in place; else a
    new tensor [B, S] is returned.  A row of nothing but -inf adds nothing, a
    row with a NaN or +inf adds NaN everywhere."""
    _require_cuda(logits, scores)
    if logits.dim() != 3 or min(logits.shape) < 1:
        raise StarKVError(f"logits must be [B, H, S], none of them 0, got {tuple(logits.shape)}")
    B, H, S = logits.shape
    if logits.dtype not in _TYPES:
        raise StarKVError(f"unsupported dtype {logits.dtype}")
    if S > 1 and logits.stride(2) != 1:
        raise StarKVError("logits must have a contiguous last dim")
    add = scores is not None
    if add:
        _check_scores(scores, B, S, logits.device)
    else:
        scores = _out(B, S, dtype=torch.float32, device=logits.device)
    d = ScoresDesc(B, H, S, _TYPES[logits.dtype], logits.data_ptr(), logits.stride(0), logits.stride(1), add,
                   scores.data_ptr(), scores.stride(0))
    _launch("starkv_attention_scores", d, logits.device, workspace=True)
    return scores


def select_positions(scores: torch.Tensor, keep: int, length: Optional[int] = None, sinks: int = 0,
                     recent: int = 0) -> torch.Tensor:
    """The ``keep`` of the first ``length`` positions of ``scores`` [B, S]
    (fp32; length defaults to S) that a bounded cache keeps, int32 [B, keep] in
    ascending order: the first ``sinks``, the last ``recent``, and of those
    between the ones with the largest scores (equal ones: the lowest
    positions; NaN counts as -inf)."""
    _require_cuda(scores)
    if scores.dim() != 2 or scores.dtype != torch.float32 or (scores.shape[1] > 1 and scores.stride(1) != 1):
        raise StarKVError(f"scores must be float32 [B, S] with a contiguous last dim, got {scores.dtype} "
                          f"{tuple(scores.shape)}")
    B, S = scores.shape
    n = S if length is None else int(length)
    if not (0 <= n <= S and min(sinks, recent) >= 0 and sinks + recent <= keep <= n):
        raise StarKVError(f"need 0 <= sinks + recent <= keep <= length <= {S}, got sinks {sinks}, recent {recent}, "
                          f"keep {keep}, length {n}")
    out = _out(B, keep, dtype=torch.int32, device=scores.device)
    d = SelectDesc(B, n, keep, sinks, recent, scores.data_ptr(), scores.stride(0), out.data_ptr(), keep)
    _launch("starkv_select_positions", d, scores.device, workspace=n > 28672)
    return out


def keep_positions(k: KLatentSpec, v, positions: torch.Tensor, length: int, scores: Optional[torch.Tensor] = None,
                   error_flag: Optional[torch.Tensor] = None) -> None:
    """Move rows ``positions`` [B, keep] (int32, as ``select_positions`` gives
    them: ascending, positions[b, i] in i .. length - 1) of the latent caches
    ``k`` and ``v`` (any format; a VLatentSpec or a dense tensor) to rows 0 ..
    keep - 1, in place; rows from keep on stay as they are.  ``scores`` [B, >=
    length] move along, zeros behind.  A position that breaks the rule leaves
    its row as it is and sets ``error_flag`` (int32 device tensor) to 1.  Rows
    that share memory (an expanded head or batch) and tensors that end before
    the rows are refused.  Keys are cached before rotation: a moved row takes
    the angle of its new place, and the next token's position is ``keep``."""
    vs = _vspec(v)
    _require_cuda(positions, scores, error_flag, *k.tensors, *vs.tensors)
    if positions.dim() != 2 or positions.dtype != torch.int32 or (positions.shape[1] > 1 and positions.stride(1) != 1):
        raise StarKVError(f"positions must be int32 [B, keep] with a contiguous last dim, got {positions.dtype} "
                          f"{tuple(positions.shape)}")
    B, keep = positions.shape
    length = int(length)
    if B < 1 or not 0 <= keep <= length:
        raise StarKVError(f"need at least one sequence and 0 <= keep <= length, got positions {tuple(positions.shape)}, "
                          f"length {length}")
    if vs.data.shape[0] != B or k.data.shape[0] != B or (length and not (k.holds(B, length) and vs.holds(B, length))):
        raise StarKVError(f"the caches must hold {B} sequences of at least {length} positions, and their scales too: K "
                          f"{tuple(k.data.shape)}, V {tuple(vs.data.shape)}")
    device = vs.data.device
    moved = [positions, k.data, k.scale, k.data2, k.scale2, error_flag, *vs.tensors]
    if any(t is not None and t.device != device for t in moved):
        raise StarKVError(f"positions, the error flag, latents and scales must lie on {device} as the V latent does")
    if scores is not None:
        _check_scores(scores, B, length, device)
    dense = k.data.dtype in (torch.float16, torch.bfloat16)
    arrays: list = []
    d = KeepDesc()
    d.batch, d.length, d.keep = B, length, keep
    d.dtype = _dt(k.data) if dense else _lib.F16
    d.positions, d.positions_stride_b = positions.data_ptr(), positions.stride(0)
    d.k, d.v = k.c_struct(arrays), vs.c_struct()
    if scores is not None:
        d.scores, d.scores_stride_b = scores.data_ptr(), scores.stride(0)
    d.error_flag = _flag_ptr(error_flag)
    _launch("starkv_keep_positions", d, device)
