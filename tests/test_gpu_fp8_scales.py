"""GPU checks of 8-bit products by power-of-two scales whose product passes
fp32's range although no value of the operands or of the result does: with a
16-bit output the scales are applied exactly, whatever the number of rows."""
import pytest
import torch

from test_gpu_fp8 import BF16, E4M3, E8, F16, _flush, _rows8, check

pytestmark = pytest.mark.gpu


def _e8(t):
    return torch.exp2(t.float()).to(E8)


@pytest.mark.parametrize("out", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("epilogue", ["none", "residual", "silu_mul"])
@pytest.mark.parametrize("m", [1, 4, 16, 17, 40, 300])
def test_scale_products_past_fp32(m, epilogue, out):
    """Block 0: activations of zero with the scale 2^90 (rows of an outlier elsewhere) against weights of scale 2^60;
    block 1: scales 2^90 and 2^-97; block 2, short: 2^-60 and 2^53."""
    from starkv import fp8_matmul
    _flush(f"[scales] {m} {epilogue} {out}")
    n, k = 512, 300
    g = torch.Generator(device="cuda").manual_seed(m)
    x, w = _rows8(g, m, k), _rows8(g, n, k)
    x[:, :128] = torch.zeros(m, 128, device="cuda").to(E4M3)
    xs = _e8(torch.tensor([90, 90, -60]))[None].expand(m, 3).contiguous().cuda()
    ws = _e8(torch.tensor([60, -104, 46]))[None].expand(n // 128, 3).contiguous().cuda()
    res = torch.randn(m, n, generator=g, device="cuda").to(out) if epilogue == "residual" else None
    c = dict(m=m, n=n, k=k, x=x, xs=xs, w=w, ws=ws, out=out, res=res, epilogue=epilogue, dtype=E4M3, scale=E8)
    check(fp8_matmul(x, xs, w, ws, residual=res, silu_mul=epilogue == "silu_mul", out_dtype=out), c)
    if out == BF16 and epilogue == "none":
        # the least products there are, under a product of scales of 2^130
        x[:, 0] = torch.full((m,), 2.0 ** -9, device="cuda").to(E4M3)
        w[:, 0] = torch.full((n,), 2.0 ** -9, device="cuda").to(E4M3)
        xs[:, 0] = _e8(torch.tensor(70.0)).cuda()
        check(fp8_matmul(x, xs, w, ws), c)


@pytest.mark.parametrize("out", [F16, BF16, torch.float32], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("scale", [E8, torch.float32], ids=["e8m0", "f32"])
@pytest.mark.parametrize("m", [1, 4, 17, 40, 300])
def test_a_scale_that_is_not_a_number(m, scale, out):
    """A NaN scale over finite values, zeros among them: its row, or its weight block's columns, are NaN and nothing else."""
    from starkv import fp8_matmul
    g = torch.Generator(device="cuda").manual_seed(m)
    n, k = 512, 300
    x, w = _rows8(g, m, k), _rows8(g, n, k)
    x[:, 128:256] = torch.zeros(m, 128, device="cuda").to(E4M3)
    xs, ws = torch.full((m, 3), 2.0 ** -7, device="cuda"), torch.full((4, 3), 2.0 ** -9, device="cuda")
    clean = fp8_matmul(x, xs.to(scale), w, ws.to(scale), out_dtype=out)
    assert bool(torch.isfinite(clean).all())
    for b in range(3):
        bad = xs.clone()
        bad[m - 1, b] = float("nan")
        got = fp8_matmul(x, bad.to(scale), w, ws.to(scale), out_dtype=out)
        assert bool(got[m - 1].isnan().all()) and torch.equal(got[:m - 1], clean[:m - 1])
        bad = ws.clone()
        bad[2, b] = float("nan")
        got = fp8_matmul(x, xs.to(scale), w, bad.to(scale), out_dtype=out)
        assert bool(got[:, 256:384].isnan().all())
        assert torch.equal(got[:, :256], clean[:, :256]) and torch.equal(got[:, 384:], clean[:, 384:])


@pytest.mark.parametrize("out", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("m", [1, 4, 16, 17, 40, 300])
def test_the_least_and_largest_scales(m, out):
    """Scale bytes 0 (2^-127) and 254 (2^127) against ones that bring the product of scales back to 2^-16 and 2^-15."""
    from starkv import fp8_matmul
    g = torch.Generator(device="cuda").manual_seed(m)
    n, k = 256, 300
    x, w = _rows8(g, m, k), _rows8(g, n, k)
    byte = lambda rows, t: torch.tensor(t, dtype=torch.uint8)[None].expand(rows, 3).contiguous().cuda().view(E8)
    xs, ws = byte(m, [0, 239, 254]), byte(n // 128, [238, 0, 0])
    x[:, 256:] = torch.zeros(m, k - 256, device="cuda").to(E4M3)      # 2^127 2^-127 = 1: too large for fp16 but of zeros
    c = dict(m=m, n=n, k=k, x=x, xs=xs, w=w, ws=ws, out=out, res=None, epilogue="none", dtype=E4M3, scale=E8)
    check(fp8_matmul(x, xs, w, ws, out_dtype=out), c)
