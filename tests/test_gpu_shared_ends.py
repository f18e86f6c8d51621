"""What ends with a shared prompt, and B_k as a prefix takes it."""
import pytest
import torch

from starkv import KLatentSpec, SharedPrefix, StarKVError, e2e
from starkv.cache import LatentCache

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_share_takes_b_k_by_rows():
    """B_k whose rows are not contiguous (a transposed view of k_u) is refused, as LatentCache.k_spec does."""
    g = torch.Generator(device=DEV).manual_seed(2)
    mk = lambda *s: torch.randn(*s, generator=g, device=DEV).half()
    ku = mk(4, 128, 128)                                         # [head, dim, rank] of rank 128: its transpose fits B_k's shape
    cache = LatentCache(1, [128] * 4, 64, 30, torch.float16, DEV, "dense")
    cache.append(mk(1, 4, 20, 128), mk(1, 20, 64), ku)
    with pytest.raises(StarKVError):
        cache.share(ku.transpose(1, 2))
    with pytest.raises(StarKVError):
        cache.share(ku[0])
    cache.share(ku.transpose(1, 2).contiguous())


def test_dropped_prompt_leaves_no_scores():
    model = e2e.build_model(batch=2, capacity=8, fmt="dense", n_layers=1, hidden=1024, heads=8, kv_heads=4, intermediate=1024,
                            vocab=100, ranks=[24, 40, 64, 32], v_rank=192)
    att, = e2e.attention_layers(model)
    att.scores = torch.zeros(2, 8, device=DEV)
    e2e.share_prompt(model, torch.arange(30, device=DEV)[None])
    e2e.decode_graphed(model, torch.ones(2, 1, dtype=torch.long, device=DEV), 3)
    assert (att.scores[:, :3] > 0).all()
    e2e.drop_prompt(model)
    assert att.prefix is None and att.cache.length == 0 and (att.scores == 0).all()
