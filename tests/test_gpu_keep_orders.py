"""Rows moved in place in every order of sequences, heads and positions that keeps them apart."""
import itertools

import pytest
import torch

from starkv import KLatentSpec, StarKVError, keep_positions
from test_gpu_bounded import DEV, kept

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("names", list(itertools.permutations(["sequence", "head", "position"])), ids=", ".join)
@pytest.mark.parametrize("pad", [0, 5])
def test_keep_in_every_order(names, pad):
    B, H, n, r = 3, 4, 50, 24
    dims = {"sequence": B, "position": n, "head": H}
    g = torch.Generator().manual_seed(7)
    x = torch.randn(*(dims[a] for a in names), r + pad, generator=g).half().to(DEV)
    x = x.permute(*(names.index(a) for a in ("sequence", "head", "position")), 3)  # [B, H, n, r + pad]
    ranks = [r, r - 7, r, 1]
    spec = KLatentSpec(x, ranks, [h * x.stride(1) for h in range(H)], [x.stride(2)] * H, x.stride(0), x, [0] * H, 128)
    v = torch.randn(B, n, 16, generator=g).half().to(DEV)
    pos = kept(B, n, 20).to(DEV)
    want = x.clone()
    for h, w in enumerate(ranks):
        want[:, h, :20, :w] = x[:, h, :, :w].gather(1, pos.long()[..., None].expand(B, 20, w))
    keep_positions(spec, v, pos, n)
    assert torch.equal(x, want)


@pytest.mark.parametrize("order", ["position, head, sequence", "head, position, sequence"])
def test_sequences_side_by_side_that_overlap_are_refused(order):
    """Rows one element longer than the step to the next sequence's."""
    B, H, n, r = 3, 2, 20, 8
    base = torch.zeros(n * H * B * r + 1, device=DEV).half()
    p, h = (H * B * r, B * r) if order[0] == "p" else (B * r, n * B * r)
    spec = KLatentSpec(base, [r + 1] * H, [0, h], [p] * H, r, base, [0] * H, 128)
    v = torch.zeros(B, n, 16, device=DEV).half()
    with pytest.raises(StarKVError):
        keep_positions(spec, v, kept(B, n, 5).to(DEV), n)
