"""LatentCache.bound keeps what the plain selection by the sums of the decode steps keeps."""
import pytest
import torch

import starkv
from starkv.cache import LatentCache
from test_gpu_bounded import DEV, select_oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["dense", "int8_g64", "reference"])
@pytest.mark.parametrize("length,keep,sinks,recent", [(60, 20, 2, 5), (60, 7, 2, 5), (60, 59, 0, 0), (60, 60, 4, 8), (9, 20, 4, 8)])
def test_bound_keeps_the_largest_sums(fmt, length, keep, sinks, recent):
    B, ranks, Rv = 2, [16, 24, 40], 96
    g = torch.Generator(device=DEV).manual_seed(length + keep)
    mk = lambda *s: torch.randn(*s, generator=g, device=DEV).half()
    bk, uv = mk(3, 40, 128) / 6, mk(384, Rv) / 9
    cache = LatentCache(B, ranks, Rv, 64, torch.float16, DEV, fmt)
    ks, vs, n = cache.append(mk(B, 3, length, 40), mk(B, length, Rv), bk)
    scores = torch.zeros(B, 64, device=DEV)
    for _ in range(3):
        starkv.decode_attention(mk(B, 6, 128), ks, vs, uv, seq_len=n, scores=scores)
    before = scores.clone()
    p = cache.bound(keep, scores, sinks=sinks, recent=recent)
    kept = min(keep, length)
    assert cache.length == kept
    assert torch.equal(p.cpu(), select_oracle(before.cpu(), kept, length, min(sinks, kept), min(recent, kept - min(sinks, kept))))
    assert torch.equal(scores[:, :kept], before.gather(1, p.long())) and (scores[:, kept:] == 0).all()
