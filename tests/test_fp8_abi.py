"""CPU checks of the 8-bit projections' and the log probabilities' C ABI: struct
layout, refusals (validation runs before any HIP call), workspace sizes; and of
the weight quantiser, which runs on any device."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

from starkv import _lib as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK, NULL, SHAPE, DTYPE, ALIGN, WORKSPACE, LIMIT = 0, -1, -2, -3, -4, -6, -7
FAKE = 0x7F0000000000          # 256-byte aligned stand-in for a device address

_STRUCTS = {"starkv_fp8_quantize_desc": L.Fp8QuantizeDesc, "starkv_fp8_gemm_desc": L.Fp8GemmDesc,
            "starkv_logprobs_desc": L.LogprobsDesc}


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
def test_struct_layouts_match_the_c_compiler(tmp_path):
    body = "".join(f'printf("{c} sizeof %zu\\n", sizeof({c}));'
                   + "".join(f'printf("{c} {f[0]} %zu\\n", offsetof({c}, {f[0]}));' for f in py._fields_)
                   for c, py in _STRUCTS.items())
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "starkv.h"\nint main(void) {' + body
                   + 'printf("codes e4m3 %d\\ncodes e8m0 %d\\ncodes top %d\\n", STARKV_E4M3, STARKV_E8M0, STARKV_MAX_TOP); return 0; }')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    from starkv import logprobs
    codes = {"e4m3": L.E4M3, "e8m0": L.E8M0, "top": logprobs.MAX_TOP}
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        c, f, v = line.split()
        got = codes[f] if c == "codes" else ctypes.sizeof(_STRUCTS[c]) if f == "sizeof" else getattr(_STRUCTS[c], f).offset
        assert got == int(v), line


def _set(d, **kw):
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _quant(**kw):
    return _set(L.Fp8QuantizeDesc(8, 1000, L.F16, FAKE, 1000, FAKE, 1008, FAKE, L.E8M0, 1, 8), **kw)


@pytest.mark.parametrize("kw,code", [
    (dict(rows=-1), SHAPE), (dict(k=0), SHAPE), (dict(dtype=L.F32), DTYPE), (dict(scale_dtype=L.F16), DTYPE),
    (dict(x=None), NULL), (dict(q=None), NULL), (dict(scale=None), NULL), (dict(x_stride=999), SHAPE),
    (dict(q_stride=992), SHAPE), (dict(q_stride=1012), ALIGN), (dict(q=FAKE + 8), ALIGN), (dict(x=FAKE + 1), ALIGN),
    (dict(scale_dtype=L.F32, scale=FAKE + 2), ALIGN), (dict(scale_stride_b=-1), SHAPE), (dict(rows=0, x=None), OK),
])
def test_quantize_refuses(kw, code):
    assert L.lib().starkv_fp8_quantize(ctypes.byref(_quant(**kw)), None) == code
    assert L.lib().starkv_fp8_quantize(None, None) == NULL


def _gemm(**kw):
    d = L.Fp8GemmDesc(8, 512, 1000, L.F16, L.F16, FAKE, 1000, None, 0, 0, FAKE, 1008, FAKE, 8, 1, L.E8M0, None, 0, 0, 0,
                      0.0, FAKE, 512)
    return _set(d, **kw)


@pytest.mark.parametrize("kw,code", [
    (dict(m=-1), SHAPE), (dict(n=0), SHAPE), (dict(k=0), SHAPE), (dict(dtype=L.F32), DTYPE), (dict(out_dtype=L.I8), DTYPE),
    (dict(scale_dtype=L.F16), DTYPE), (dict(x=None), NULL), (dict(w=None), NULL), (dict(w_scale=None), NULL),
    (dict(out=None), NULL), (dict(dtype=L.E4M3, x_stride=1008), NULL), (dict(x_stride=999), SHAPE),
    (dict(w_stride=992), SHAPE), (dict(w_stride=1004), ALIGN), (dict(w=FAKE + 8), ALIGN), (dict(out_stride=511), SHAPE),
    (dict(out=FAKE + 1), ALIGN), (dict(x=FAKE + 1), ALIGN), (dict(silu_mul=1, n=384), SHAPE),
    (dict(silu_mul=1, residual=FAKE, residual_stride=512), SHAPE), (dict(residual=FAKE, residual_stride=511), SHAPE),
    (dict(rms=1, rms_eps=-1.0), SHAPE), (dict(rms=1, rms_eps=float("nan")), SHAPE),
    (dict(rms=1, dtype=L.E4M3, x_stride=1008, x_scale=FAKE), SHAPE), (dict(w_scale_stride_r=-1), SHAPE),
    (dict(dtype=L.E4M3, x_scale=FAKE, x_stride=1000), ALIGN), (dict(scale_dtype=L.F32, w_scale=FAKE + 2), ALIGN),
    (dict(m=100), WORKSPACE), (dict(), WORKSPACE), (dict(m=1 << 30, n=1 << 30, dtype=L.E4M3, x_stride=1008, x_scale=FAKE), LIMIT), (dict(m=0, x=None), OK),
])
def test_gemm_refuses(kw, code):
    assert L.lib().starkv_fp8_gemm(ctypes.byref(_gemm(**kw)), None, 0, None) == code


def test_gemm_workspace():
    size = lambda **kw: L.lib().starkv_fp8_gemm_workspace_bytes(ctypes.byref(_gemm(**kw)))
    assert size(m=0) == 0 and size(k=0) == 0 and size(dtype=L.E4M3) == 0 and size(dtype=L.E4M3, m=16) == 0
    # quantised rows, their scales, and partial sums where k is split
    assert size(m=17) >= 17 * 1008 + 17 * 8 and size(m=3) >= 3 * 1008 + 3 * 8
    assert size(m=8192, n=22016) >= 8192 * 1008
    assert L.lib().starkv_fp8_gemm(ctypes.byref(_gemm(m=17)), FAKE, size(m=17) - 1, None) == WORKSPACE
    assert L.lib().starkv_fp8_gemm(ctypes.byref(_gemm(m=17)), FAKE + 64, size(m=17), None) == ALIGN


def _lp(**kw):
    return _set(L.LogprobsDesc(4, 1000, L.F16, 5, FAKE, 1000, FAKE, FAKE, FAKE, FAKE, FAKE), **kw)


@pytest.mark.parametrize("kw,code", [
    (dict(rows=-1), SHAPE), (dict(vocab=0), SHAPE), (dict(top=-1), SHAPE), (dict(vocab=4), SHAPE), (dict(top=65), LIMIT),
    (dict(vocab=(1 << 24) + 1), LIMIT), (dict(dtype=L.I8), DTYPE), (dict(logits=None), NULL), (dict(logprob=None), NULL),
    (dict(top_id=None), NULL), (dict(top_logprob=None), NULL), (dict(stride=999), SHAPE), (dict(logits=FAKE + 1), ALIGN),
    (dict(dtype=L.F32, logits=FAKE + 2), ALIGN), (dict(tokens=FAKE + 4), ALIGN), (dict(top_id=FAKE + 4), ALIGN),
    (dict(entropy=FAKE + 2), ALIGN), (dict(rows=0, logits=None), OK),
])
def test_logprobs_refuses(kw, code):
    assert L.lib().starkv_token_logprobs(ctypes.byref(_lp(**kw)), None, 0, None) == code


def test_operators_refuse_host_tensors():
    import starkv
    x = torch.zeros(2, 128, dtype=torch.float16)
    w, s = starkv.fp8_quantize_weight(torch.ones(128, 128))
    for f in (lambda: starkv.fp8_quantize(x), lambda: starkv.fp8_linear(x, w, s),
              lambda: starkv.fp8_matmul(x.to(torch.float8_e4m3fn), s, w, s),
              lambda: starkv.token_logprobs(x, torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(starkv.StarKVError):
            f()


@pytest.mark.parametrize("kind", ["e8m0", "f32"])
@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (130, 300), (257, 1000)])
def test_quantize_weight(n, k, kind):
    """Blocks of 128 x 128: the scale by its rule, each value within half an e4m3 step of its quotient, rows 16-byte
    pieces apart."""
    from starkv import fp8_quantize_weight
    g = torch.Generator().manual_seed(n + k)
    w = torch.randn(n, k, generator=g) * torch.exp2(torch.randint(-6, 6, (n, 1), generator=g).float())
    q, s = fp8_quantize_weight(w, torch.float8_e8m0fnu if kind == "e8m0" else torch.float32)
    assert q.shape == (n, k) and q.stride(0) % 16 == 0 and s.shape == (-(-n // 128), -(-k // 128))
    sd = s.double()
    for i in range(s.shape[0]):
        for b in range(s.shape[1]):
            blk = w[128 * i:128 * i + 128, 128 * b:128 * b + 128].double()
            a, v = float(blk.abs().max()), float(sd[i, b])
            if kind == "e8m0":
                assert a <= 448 * v and a > 224 * v
            else:
                assert v == float(torch.tensor(a / 448.0, dtype=torch.float64).float())
            r, d = blk / v, q[128 * i:128 * i + 128, 128 * b:128 * b + 128].double()
            # half a step: 2^-4 of the value, at least 2^-10
            assert bool(((r - d).abs() <= (r.abs() * 2.0 ** -4).clamp_min(2.0 ** -10) * (1 + 2.0 ** -20)).all())


def test_quantize_weight_norm_zero_and_nan():
    from starkv import StarKVError, fp8_quantize_weight
    w = torch.zeros(256, 256)
    w[200, 200] = float("nan")
    q, s = fp8_quantize_weight(w)
    assert s[0].double().tolist() == [1.0, 1.0] and s[1, 0].double() == 1.0 and s[1, 1].float().isnan()
    assert q[:128].float().abs().sum() == 0 and q[128:, 128:].float().isnan().all()
    nw = torch.full((256,), 2.0)
    a = fp8_quantize_weight(torch.ones(128, 256), norm_weight=nw)
    b = fp8_quantize_weight(torch.full((128, 256), 2.0))
    assert torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and torch.equal(a[1].float(), b[1].float())
    for bad in (lambda: fp8_quantize_weight(w[0]), lambda: fp8_quantize_weight(w[:0]),
                lambda: fp8_quantize_weight(w, torch.float16), lambda: fp8_quantize_weight(w, norm_weight=nw[:3])):
        with pytest.raises(StarKVError):
            bad()


def test_dimensions_that_pass_32_bits_are_refused():
    """A row count that the C interface's int cannot hold is an error, not its low bits."""
    from starkv import StarKVError, fp8_quantize, token_logprobs
    many = torch.zeros(1, 1, dtype=torch.float16).expand(2 ** 32 + 5, 1)
    with pytest.raises(StarKVError, match="rows or columns"):
        fp8_quantize(many)
    with pytest.raises(StarKVError, match="rows"):
        token_logprobs(many)


def test_gemm_refuses_weight_scales_too_far_apart():
    """With SiLU-multiply a tile's up rows' scales are reached by a 32-bit offset from its gate rows'."""
    d = _set(_gemm(), m=512, n=4096, out_stride=4096, silu_mul=1, w_scale_stride_r=2 ** 29)
    assert L.lib().starkv_fp8_gemm(ctypes.byref(d), FAKE, 1 << 40, None) == LIMIT
