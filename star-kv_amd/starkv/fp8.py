"""Projections in 8-bit floating point (e4m3) with a scale for each block of
128 (the formats and formulas are in include/starkv.h, starkv_fp8_quantize and
starkv_fp8_gemm).

A quantised tensor is a pair: the e4m3 values [..., k] (``torch.float8_e4m3fn``)
and the scales, [..., ceil(k / 128)] of activation rows and [ceil(n / 128),
ceil(k / 128)] of a weight [n, k].  Scales are powers of two
(``torch.float8_e8m0fnu``: the matrix instructions apply them) or
``torch.float32`` (checkpoints that come with such).  Like the other operators
these serve inference: their outputs carry no gradient.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib, ops
from ._lib import Fp8GemmDesc, Fp8QuantizeDesc, StarKVError
from .ops import _launch, _out, _poison

__all__ = ["fp8_quantize", "fp8_quantize_weight", "fp8_matmul", "fp8_linear"]

BLOCK = 128
E4M3_MAX = 448.0
MAX_DIM = 1 << 30                    # rows and columns of one call
_ACT = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_OUT = {**_ACT, torch.float32: _lib.F32}
_SCALE = {torch.float8_e8m0fnu: _lib.E8M0, torch.float32: _lib.F32}


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _e4m3_rows(rows: int, k: int, device) -> torch.Tensor:
    """[rows, k] e4m3 whose rows lie whole 16-byte pieces apart, as the kernels read them."""
    return torch.empty(rows, -(-k // 16) * 16, dtype=torch.float8_e4m3fn, device=device)[:, :k]


def _rows2d(t: torch.Tensor, name: str) -> Tuple[int, int, int]:
    """(rows, width, row stride) of t as [rows, width]; one row has any stride, 16 * ceil(width / 16) is given."""
    shape, stride = t.shape, t.stride()
    if len(shape) == 2:
        m, w = shape
    else:
        w = shape[-1] if shape else 0
        m = shape[:-1].numel()
    if w < 1:
        raise StarKVError(f"{name} must have rows of at least one value, got shape {tuple(shape)}")
    if w > 1 and stride[-1] != 1:
        raise StarKVError(f"{name} must have a contiguous last dim")
    if len(shape) != 2 and m > 1:
        try:
            t = t.view(-1, w)
        except RuntimeError:
            raise StarKVError(f"{name} rows must be addressable with one row stride") from None
        stride = t.stride()
    if m > MAX_DIM or w > MAX_DIM:
        raise StarKVError(f"{name} has more than {MAX_DIM} rows or columns: {tuple(shape)}")
    return m, w, (stride[0] if m > 1 else -(-w // 16) * 16)


def _on(device, *ts: Optional[torch.Tensor]) -> None:
    if device.type != "cuda":
        raise StarKVError("libstarkv operators take device tensors (there is no CPU path)")
    for t in ts:
        if t is not None and t.device != device:
            raise StarKVError(f"a {t.dtype} {tuple(t.shape)} is on {t.device}, the activations on {device}")


def _scale_code(dtype) -> int:
    code = _SCALE.get(dtype)
    if code is None:
        raise StarKVError(f"scales are float8_e8m0fnu or float32, got {dtype}")
    return code


def fp8_quantize(x: torch.Tensor, scale_dtype: torch.dtype = torch.float8_e8m0fnu) -> Tuple[torch.Tensor, torch.Tensor]:
    """Activations x [..., k] (fp16 / bf16) as e4m3 with one scale for each
    row's block of 128 columns (starkv_fp8_quantize).  Returns (values [..., k],
    scales [..., ceil(k / 128)]); the rows of the values lie whole 16-byte
    pieces apart, the scales block by block."""
    dt = _ACT.get(x.dtype)
    if dt is None:
        raise StarKVError(f"activations are float16 or bfloat16, got {x.dtype}")
    sd = _scale_code(scale_dtype)
    m, k, xs = _rows2d(x, "x")
    dev = x.device
    _on(dev)
    kb, lead, pitch = -(-k // BLOCK), x.shape[:-1], -(-k // 16) * 16
    q = _out(*lead, pitch, dtype=torch.float8_e4m3fn, device=dev)
    # the scales of a block of columns together: [ceil(k / 128)][rows]
    if x.dim() == 2:
        strides = (1, m)
    else:
        strides, s = [m], 1
        for n in reversed(lead):
            strides.insert(0, s)
            s *= n
    scale = torch.empty_strided((*lead, kb), strides, dtype=scale_dtype, device=dev)
    if ops.POISON:
        _poison(scale.movedim(-1, 0))
    _launch("starkv_fp8_quantize", Fp8QuantizeDesc(m, k, dt, x.data_ptr(), xs, q.data_ptr(), pitch, scale.data_ptr(),
                                                   sd, 1, m), dev)
    return (q if pitch == k else q[..., :k]), scale


@torch.no_grad()
def fp8_quantize_weight(w: torch.Tensor, scale_dtype: torch.dtype = torch.float8_e8m0fnu,
                        norm_weight: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """An nn.Linear weight [n, k] (any float type, any device) as e4m3 with one
    scale for each block of 128 x 128: (values [n, k], scales [ceil(n / 128),
    ceil(k / 128)]), by the same rule as ``fp8_quantize``.  ``norm_weight`` [k]:
    the weight of an RMSNorm applied to the input first, folded in for
    ``fp8_linear(..., rms_eps=...)``.  Run once when a model is loaded (torch
    operations, none of them recorded for gradients)."""
    _scale_code(scale_dtype)
    if w.dim() != 2 or not w.numel():
        raise StarKVError(f"a weight is [n, k], got shape {tuple(w.shape)}")
    n, k = w.shape
    f = w.float()
    if norm_weight is not None:
        if norm_weight.shape != (k,):
            raise StarKVError("norm_weight must be [k]")
        f = f * norm_weight.float()
    nb, kb = _blocks(n), _blocks(k)
    b = torch.nn.functional.pad(f, (0, kb * BLOCK - k, 0, nb * BLOCK - n)).view(nb, BLOCK, kb, BLOCK)
    a = b.abs().amax(dim=(1, 3))                                   # a NaN stays one
    good = torch.isfinite(a)
    nan = torch.full_like(a, float("nan"))
    if scale_dtype == torch.float8_e8m0fnu:
        mant, e = torch.frexp(torch.where(good, a, 1.0))
        e = torch.where(a > 0, (e - 9 + (mant > 0.875).int()).clamp_min(-126), 0).int()
        inv = torch.where(good, ((127 - e) << 23).view(torch.float32), nan)
        scale = torch.where(good, e + 127, 255).to(torch.uint8).view(torch.float8_e8m0fnu)
    else:
        most, a1 = torch.full_like(a, E4M3_MAX), a.clamp_min(2.0 ** -100)
        inv = torch.where(good, most / a1, nan)
        scale = torch.where(good, torch.where(a > 0, a1 / most, 1.0), nan)
    out = _e4m3_rows(n, k, w.device)
    out.copy_((b * inv[:, None, :, None]).view(nb * BLOCK, kb * BLOCK)[:n, :k])
    return out, scale


def _product(name, x, x_scale, weight, weight_scale, residual, silu_mul, rms_eps, out, out_dtype):
    dev = x.device
    _on(dev, weight, weight_scale, x_scale, residual, out)
    if weight.dtype != torch.float8_e4m3fn or weight.dim() != 2:
        raise StarKVError(f"{name}: weight must be a float8_e4m3fn [n, k], got {weight.dtype} {tuple(weight.shape)}")
    sd = _scale_code(weight_scale.dtype)
    n, k, ws = _rows2d(weight, "weight")
    m, xw, xs = _rows2d(x, "x")
    if xw != k:
        raise StarKVError(f"{name}: x has {xw} columns, the weight {k}")
    kb = (k + BLOCK - 1) // BLOCK
    if weight_scale.shape != ((n + BLOCK - 1) // BLOCK, kb):
        raise StarKVError(f"{name}: weight_scale must be [{_blocks(n)}, {kb}], got {tuple(weight_scale.shape)}")
    n_out = n
    if silu_mul:
        n_out = n // 2
        if n % (2 * BLOCK):
            raise StarKVError(f"{name}: the gate and the up half of a merged weight are whole blocks of {BLOCK} rows "
                              f"each, got n = {n}")
        if residual is not None:
            raise StarKVError(f"{name}: silu_mul takes no residual")
    lead = x.shape[:-1]
    shape = (*lead, n_out)
    if out is None:
        out, os_ = _out(*shape, dtype=out_dtype, device=dev), n_out
    else:
        if out.shape != shape or (out_dtype is not None and out.dtype != out_dtype):
            raise StarKVError(f"{name}: out must be {shape} of {out_dtype}, got {tuple(out.shape)} of {out.dtype}")
        os_ = _rows2d(out, "out")[2]
    od = _OUT.get(out.dtype)
    if od is None:
        raise StarKVError(f"{name}: outputs are float16, bfloat16 or float32, got {out.dtype}")
    rp, rs = None, 0
    if residual is not None:
        if residual.shape != shape or residual.dtype != out.dtype:
            raise StarKVError(f"{name}: residual must be {shape} of {out.dtype}")
        rp, rs = residual.data_ptr(), _rows2d(residual, "residual")[2]
    if x_scale is None:
        xd, xp, xsr, xsb = _ACT[x.dtype], None, 0, 0
    else:
        if x_scale.shape != (*lead, kb) or x_scale.dtype != weight_scale.dtype:
            raise StarKVError(f"{name}: x_scale must be {(*lead, kb)} of {weight_scale.dtype} like weight_scale")
        sr = x_scale
        if len(lead) != 1:
            try:
                sr = sr.view(-1, kb) if m else sr.reshape(0, kb)
            except RuntimeError:
                raise StarKVError(f"{name}: x_scale rows must be addressable with one row stride") from None
        xd, xp, (xsr, xsb) = _lib.E4M3, sr.data_ptr(), sr.stride()
    wsr, wsb = weight_scale.stride()
    d = Fp8GemmDesc(m, n, k, xd, od, x.data_ptr(), xs, xp, xsr, xsb, weight.data_ptr(), ws, weight_scale.data_ptr(),
                    wsr, wsb, sd, rp, rs, 1 if silu_mul else 0, 0 if rms_eps is None else 1, rms_eps or 0.0,
                    out.data_ptr(), os_)
    # e4m3 activations need no workspace
    _launch("starkv_fp8_gemm", d, dev, workspace=x_scale is None)
    return out


def fp8_matmul(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
               residual: Optional[torch.Tensor] = None, silu_mul: bool = False, out: Optional[torch.Tensor] = None,
               out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x W^T of quantised activations (``fp8_quantize``: e4m3 x [..., k] with
    x_scale [..., ceil(k / 128)], rows whole 16-byte pieces apart) and a
    quantised weight [n, k], summed in fp32 and rounded once (to bfloat16
    unless ``out_dtype`` or ``out`` says otherwise).  For 16-bit results the
    matrix instruction keeps 13 bits or more below the largest of each eight
    products (1.5e-5 of the results in the norm); ``out_dtype=torch.float32``
    adds exact products, at half the rate.  The scales of both are of one type.  ``residual`` [..., n] is added (``out`` may be it); with
    ``silu_mul`` the weight holds gate rows then up rows and the result is
    SiLU(x Wg^T) * (x Wu^T) [..., n / 2], each half whole blocks of 128 rows."""
    if x.dtype != torch.float8_e4m3fn:
        raise StarKVError(f"fp8_matmul: x must be float8_e4m3fn, got {x.dtype} (fp8_linear quantises)")
    if out is None and out_dtype is None:
        out_dtype = torch.bfloat16
    return _product("fp8_matmul", x, x_scale, weight, weight_scale, residual, silu_mul, None, out, out_dtype)


def fp8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
               residual: Optional[torch.Tensor] = None, silu_mul: bool = False, rms_eps: Optional[float] = None,
               out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``fp8_matmul`` of fp16 / bf16 activations x [..., k], quantised on the
    way as ``fp8_quantize(x, weight_scale.dtype)`` would.  ``rms_eps``: x is the raw input
    of an RMSNorm whose weight is folded into ``weight``
    (``fp8_quantize_weight(w, norm_weight=...)``); each row of the product is
    scaled by rsqrt(mean(x^2) + rms_eps).  The result has x's type unless
    ``out_dtype`` or ``out`` says otherwise."""
    if x.dtype not in _ACT:
        raise StarKVError(f"fp8_linear: activations are float16 or bfloat16, got {x.dtype}")
    if out is None and out_dtype is None:
        out_dtype = x.dtype
    return _product("fp8_linear", x, None, weight, weight_scale, residual, silu_mul, rms_eps, out, out_dtype)
