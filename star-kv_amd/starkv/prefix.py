"""Decode of a batch whose sequences share a prefix: a system prompt, or the prompt of several samples
(starkv_prefix_pack and starkv_prefix_decode in include/starkv.h)."""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from . import _lib
from ._lib import FMT_DENSE, DecodeDesc, PrefixDecodeDesc, PrefixPackDesc, StarKVError, int_array
from .ops import (HEAD_DIM, KLatentSpec, _check_scores, _decode_desc, _dt, _launch, _out, _q3,
                  _require_cuda, _vspec)
from .rope import RopeConfig, rope_table

__all__ = ["SharedPrefix", "prefix_decode_attention"]


class SharedPrefix:
    """The latents of positions [0, length) of one sequence (``row`` of the
    batch that ``k`` and ``v`` describe), laid out once for
    ``prefix_decode_attention`` in memory of their own: the caches that they
    come from may be overwritten afterwards.  ``k``: a dense KLatentSpec (with
    B_k); ``v``: a dense V latent [B, >= length, Rv].  ``LatentCache.share``
    makes one from a cache of any format."""

    def __init__(self, k: KLatentSpec, v, length: Optional[int] = None, rope: RopeConfig = RopeConfig(), row: int = 0):
        vs = _vspec(v)
        _require_cuda(*k.tensors, *vs.tensors)
        if k.fmt != FMT_DENSE or vs.fmt != FMT_DENSE:
            raise StarKVError("a shared prefix takes dense latents (LatentCache.share dequantises)")
        n = int(vs.data.shape[1] if length is None else length)
        if not 1 <= n <= vs.data.shape[1] or not 0 <= row < vs.data.shape[0]:
            raise StarKVError(f"row {row} of the V latent {tuple(vs.data.shape)} does not hold {n} positions")
        if not k.holds(row + 1, n):
            raise StarKVError(f"row {row} of the K latent {tuple(k.data.shape)} does not hold {n} positions")
        if not k.holds_bk():
            raise StarKVError(f"B_k {tuple(k.bk.shape)} does not hold {k.ranks} rows of {HEAD_DIM} contiguous elements")
        if k.data.dtype != vs.data.dtype or k.bk.dtype != k.data.dtype:
            raise StarKVError(f"K latents, B_k and V latents must share a type, got {k.data.dtype}, {k.bk.dtype}, "
                              f"{vs.data.dtype}")
        devices = {t.device for t in k.tensors + vs.tensors}
        if len(devices) > 1:
            raise StarKVError(f"K latents, B_k and V latents lie on different devices: {devices}")
        self.length, self.ranks, self.v_rank, self.rope = n, list(k.ranks), vs.rank, rope
        self.span = -(-n // 64) * 64               # positions of the rotation table that the kernels read
        self.dtype, self.device = k.data.dtype, vs.data.device
        rope_table(rope, self.span, self.device)   # here, not in a decode call that may be captured
        keep: list = []
        d = PrefixPackDesc()
        d.length, d.dtype = n, _dt(k.data)
        d.k, d.v = k.c_struct(keep), vs.c_struct()
        d.k.data = k.data.data_ptr() + row * k.stride_b * k.data.element_size()
        d.v.data = vs.data.data_ptr() + row * vs.data.stride(0) * vs.data.element_size()
        d.attention_scaling = rope.attention_scaling
        nb = _lib.lib().starkv_prefix_bytes(ctypes.byref(d))
        self.data = _out(max(nb, 1), dtype=torch.uint8, device=self.device)
        d.prefix, d.prefix_bytes = self.data.data_ptr(), nb
        _launch("starkv_prefix_pack", d, self.device)
        angle = rope.inv_freq().double() * n       # (an fp32 product is off by up to 2^-9 rad at 65000 positions)
        self._cos = (ctypes.c_float * 64)(*angle.cos().tolist())
        self._sin = (ctypes.c_float * 64)(*angle.sin().tolist())
        self._rank = int_array(self.ranks)


def prefix_decode_attention(q: torch.Tensor, prefix: SharedPrefix, k: Optional[KLatentSpec], xv,
                            uv_weight: torch.Tensor, seq_len: Optional[int] = None,
                            mask: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                            out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                            last_pos: Optional[torch.Tensor] = None,
                            scores: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``decode_attention`` of sequences that all follow ``prefix``: attention
    over its positions, computed for the batch together, and over each sequence's
    own latents (``k``, ``xv``, ``seq_len``, ``mask`` and ``last_pos`` as
    there; ``k`` and ``xv`` None, or ``seq_len`` 0: none yet).  B_k is the
    layer's, as the prefix was packed with it.  A sequence whose mask leaves
    none of its own positions (-inf, or a value as low as a type's lowest)
    attends to the prefix alone.  Masked positions of dense K latents may hold
    NaN and infinities (to finite logits a finite mask is added as it is); V
    latents, and the scales of quantised ones, have to be finite in all
    ``seq_len`` positions (their weight there is 0, and 0 times NaN is NaN).

    Positions are those of the sequences' own caches: ``q`` [B, Hq, 128] is
    rotated at its position behind the sequence's own first one, own key s at
    s, and the prefix lies before them.  ``scores``: fp32 [B, >= seq_len], onto
    which the weights of own positions are added, summed over the heads (the
    prefix's weights are in the softmax but not in the sums)."""
    q = _q3(q)
    B = q.shape[0]
    if (k is None) != (xv is None):
        raise StarKVError("own latents are k and xv together")
    n, v = 0, None
    if k is not None:
        v = _vspec(xv)
        n = int(v.data.shape[1] if seq_len is None else seq_len)
    elif seq_len or mask is not None or last_pos is not None:
        raise StarKVError("seq_len, mask and last_pos describe own latents: k and xv")
    if n < 0:
        raise StarKVError(f"seq_len must not be negative, got {n}")
    _require_cuda(q, uv_weight, scores)
    device = q.device
    if q.dtype != prefix.dtype or uv_weight.dtype != prefix.dtype:
        raise StarKVError(f"q and uv_weight must be {prefix.dtype} as the prefix is, got {q.dtype} and {uv_weight.dtype}")
    if device != prefix.device or uv_weight.device != device:
        raise StarKVError(f"the prefix lies on {prefix.device}, q on {device}, uv_weight on {uv_weight.device}")
    if n:
        if k.ranks != prefix.ranks or v.rank != prefix.v_rank:
            raise StarKVError(f"own latents have K ranks {k.ranks} and V rank {v.rank}, the prefix {prefix.ranks} and "
                              f"{prefix.v_rank}")
        if not v.holds(B, n):
            raise StarKVError(f"the V latent {tuple(v.data.shape)} does not hold {B} sequences of {n} positions")
        if not k.holds(B, n):
            raise StarKVError(f"the K latent {tuple(k.data.shape)} does not hold {B} sequences of {n} positions")
        if any(t is not None and t.device != device for t in (mask, last_pos, *k.tensors, *v.tensors)):
            raise StarKVError(f"own latents, mask and last_pos must lie on {device} as q does")
        if k.fmt == FMT_DENSE and k.data.dtype != prefix.dtype or v.fmt == FMT_DENSE and v.data.dtype != prefix.dtype:
            raise StarKVError(f"dense own latents must be {prefix.dtype}, got {k.data.dtype} and {v.data.dtype}")
    if out is not None and (out.shape != (B, q.shape[1], HEAD_DIM) or out.device != device):
        raise StarKVError(f"out must be {(B, q.shape[1], HEAD_DIM)} on {device}, got {tuple(out.shape)} on {out.device}")
    if scores is not None:
        _check_scores(scores, B, n, device)
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return prefix_decode_attention(q, prefix, k, xv, uv_weight, seq_len, mask, scale, out, out_dtype, last_pos, scores)
    if n:
        own, out, keep = _decode_desc(q, k, v, uv_weight, prefix.rope, n, mask, scale, out, out_dtype, last_pos)
    else:
        own, out, keep = _prefix_only(q, prefix, uv_weight, scale, out, out_dtype)
    if own.rope_max_positions < prefix.span:
        table, own.rope_max_positions = rope_table(prefix.rope, prefix.span, device)
        own.rope_table = table.data_ptr()
    d = PrefixDecodeDesc(own, len(prefix.ranks), prefix.v_rank, prefix.length, prefix._rank, prefix.data.data_ptr(),
                         prefix.data.numel(), prefix._cos, prefix._sin)
    if scores is not None and n:
        d.scores, d.scores_stride_b = scores.data_ptr(), scores.stride(0)
    _launch("starkv_prefix_decode", d, device, workspace=True)
    return out


def _prefix_only(q, prefix: SharedPrefix, uv_weight, scale, out, out_dtype):
    """The descriptor of a call without own positions."""
    B, Hq, _ = q.shape
    if uv_weight.shape != (len(prefix.ranks) * HEAD_DIM, prefix.v_rank) or uv_weight.stride(1) != 1:
        raise StarKVError("uv_weight must be [Hkv*128, Rv] with a contiguous last dim")
    if out is None:
        out = _out(B, Hq, HEAD_DIM, dtype=out_dtype or q.dtype, device=q.device)
    if out.dtype not in (q.dtype, torch.float32) or out.stride(-1) != 1:
        raise StarKVError("out must be [B, Hq, 128] of q's dtype or float32")
    d = DecodeDesc()
    d.batch, d.n_q_heads, d.head_dim, d.seq_len, d.dtype = B, Hq, HEAD_DIM, 0, _dt(q)
    d.q, d.q_stride_b, d.q_stride_h = q.data_ptr(), q.stride(0), q.stride(1)
    d.uv, d.uv_row_stride = uv_weight.data_ptr(), uv_weight.stride(0)
    d.scale = float(scale if scale is not None else 1.0 / math.sqrt(HEAD_DIM))
    d.out, d.out_stride_b, d.out_stride_h = out.data_ptr(), out.stride(0), out.stride(1)
    d.out_dtype = _lib.F32 if out.dtype == torch.float32 else 0
    return d, out, ()
