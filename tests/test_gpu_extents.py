"""Calls whose scales, lower blocks, last rows or B_k end before what they describe are refused before anything runs."""
import pytest
import torch

from starkv import KLatentSpec, SharedPrefix, StarKVError, VLatentSpec, keep_positions, prefix_decode_attention
from starkv.cache import LatentCache

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
RANKS = [24, 5, 40]


def filled(fmt, n=20):
    g = torch.Generator(device=DEV).manual_seed(1)
    mk = lambda *s: torch.randn(*s, generator=g, device=DEV).half()
    c = LatentCache(2, RANKS, 300, n, torch.float16, DEV, fmt)
    bk = mk(3, 40, 128)
    k, v, _ = c.append(mk(2, 3, n, 40), mk(2, n, 300), bk)
    return c, k, v, bk, mk


def cut(spec, name):
    t = getattr(spec, name)
    if t is None:
        return False
    setattr(spec, name, t[:, :-1] if t.dim() == 3 and isinstance(spec, VLatentSpec) else t.reshape(-1)[:t.numel() // 2][None].expand(2, -1))
    return True


@pytest.mark.parametrize("fmt", ["dense", "int8_g64", "reference"])
def test_short_tensors_are_refused(fmt):
    for which in ("k", "v"):
        for name in ("data", "scale", "data2", "scale2", "zero"):
            c, k, v, bk, mk = filled(fmt)
            whole = c.share(bk)
            q, uv = mk(2, 6, 128), mk(384, 300)
            pos = torch.arange(5, dtype=torch.int32, device=DEV).expand(2, 5).contiguous()
            prefix_decode_attention(q, whole, k, v, uv)
            keep_positions(k, v, pos, 20)
            spec = k if which == "k" else v
            if not hasattr(spec, name) or not cut(spec, name):
                continue
            for call in (lambda: keep_positions(k, v, pos, 20), lambda: prefix_decode_attention(q, whole, k, v, uv, seq_len=20)):
                with pytest.raises(StarKVError):
                    call()
                    pytest.fail(f"{which}.{name}")


def test_short_b_k_and_last_rows_are_refused():
    k = torch.zeros(1, 2, 30, 16, device=DEV).half()
    bk = torch.zeros(2, 16, 128, device=DEV).half()
    v = torch.zeros(1, 30, 64, device=DEV).half()
    spec = lambda k, b, rank=16: KLatentSpec(k, [rank] * 2, [0, 480], [16, 16], 960, b, [0, 2048], 128)
    SharedPrefix(spec(k, bk), v)
    for s in (spec(k, bk.view(-1)[:-1]), spec(k, bk[:1]), spec(k, bk.transpose(1, 2)), spec(k.view(1, -1)[:, :-1], bk)):
        with pytest.raises(StarKVError):
            SharedPrefix(s, v)
