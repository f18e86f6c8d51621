"""GPU checks of 8-bit projections of more rows than one launch has workgroups
of 256 threads for (2^24): the row factors of a folded norm."""
import pytest
import torch

from test_gpu_fp8 import E8, F16, F32, _flush, _rows8, _scales, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [E8, F32], ids=["e8m0", "f32"])
def test_rms_of_more_rows_than_a_launch_has_workgroups(scale):
    from starkv import fp8_linear
    m, n, k = (1 << 24) + 5, 16, 40
    _flush(f"[many rows] {m} {scale}")
    g = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn(m, k, generator=g, device="cuda", dtype=F16)
    w, ws = _rows8(g, n, k), _scales(g, (1, 1), scale, -9)
    x *= torch.exp2((torch.arange(m, device="cuda") % 7 - 3).half())[:, None]      # rows of other factors side by side
    out = fp8_linear(x, w, ws, rms_eps=1e-5)
    torch.cuda.synchronize()
    at = torch.tensor([0, 1, 2, (1 << 22) - 1, 1 << 22, (1 << 22) + 1, 3 << 22, (1 << 24) - 1, 1 << 24, m - 2, m - 1]).cuda()
    check(out[at], dict(m=len(at), n=n, k=k, x=x[at], w=w, ws=ws, dtype=F16, out=F16, scale=scale, res=None,
                        epilogue="none"), rms_eps=1e-5)
    # every row: as the same rows give in calls that one launch holds
    n = 1 << 21
    for i in (*range(0, m - n, n), m - n):
        assert torch.equal(out[i:i + n], fp8_linear(x[i:i + n], w, ws, rms_eps=1e-5))
