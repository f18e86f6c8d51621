"""CPU checks of the exact workspace sizes of the 8-bit products and the token log probabilities."""
import ctypes

import pytest

from starkv import _lib as L
from test_fp8_abi import _gemm, _lp


def _up(n, to):
    return -(-n // to) * to


@pytest.mark.parametrize("scale,size", [(L.E8M0, 1), (L.F32, 4)], ids=["e8m0", "f32"])
@pytest.mark.parametrize("m,n,k", [(1, 512, 1), (3, 512, 1000), (17, 512, 1000), (40, 256, 130), (8192, 22016, 4096)])
def test_gemm_workspace_is_the_quantised_rows(m, n, k, scale, size):
    """The rows (whole 16-byte pieces), their scales and the row factors, each in whole 256 bytes; nothing else,
    however k is split, and nothing at all for rows that are quantised already."""
    d = dict(m=m, n=n, k=k, x_stride=k, w_stride=_up(k, 16), out_stride=n, scale_dtype=scale)
    bytes_of = lambda **kw: L.lib().starkv_fp8_gemm_workspace_bytes(ctypes.byref(_gemm(**(d | kw))))
    want = _up(m * _up(k, 16), 256) + _up(m * -(-k // 128) * size, 256) + _up(4 * m, 256)
    for kw in (dict(), dict(rms=1, rms_eps=1e-5), dict(silu_mul=1), dict(dtype=L.BF16), dict(out_dtype=L.F32)):
        assert bytes_of(**kw) == want
    assert bytes_of(dtype=L.E4M3, x_stride=_up(k, 16)) == 0


def test_logprobs_workspace_is_the_pieces():
    """16 bytes of statistics and the keys for each piece of a row that is split; none where rows are whole."""
    size = lambda **kw: L.lib().starkv_token_logprobs_workspace_bytes(ctypes.byref(_lp(**kw)))
    assert size() == 0 and size(rows=100000) == 0 and size(rows=0) == 0 and size(vocab=0) == 0
    one = dict(rows=1, vocab=131072, dtype=L.F32)
    pieces = (size(**one, top=20) - size(**one, top=10)) // 80
    assert 1 < pieces <= 64
    for top in (0, 1, 20, 64):
        assert size(**one, top=top) == _up(16 * pieces, 256) + 8 * pieces * top
