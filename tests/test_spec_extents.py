"""KLatentSpec.holds and VLatentSpec.holds: what a specification's tensors hold, to their last element (CPU only)."""
import pytest
import torch

from starkv import KLatentSpec, VLatentSpec
from starkv.cache import LatentCache

RANKS = [24, 5, 40]


def cache(fmt, n=10):
    c = LatentCache(2, RANKS, 300, n, torch.float16, "cpu", fmt)
    return c.k_spec(torch.zeros(3, 40, 128).half()), c.v_spec


@pytest.mark.parametrize("fmt", ["dense", "int8_g64", "reference"])
def test_caches_hold_their_capacity(fmt):
    k, v = cache(fmt)
    assert k.holds(2, 10) and v.holds(2, 10) and k.holds(1, 1) and v.holds(1, 1) and k.holds_bk()
    assert not v.holds(2, 11) and not v.holds(3, 10) and not k.holds(3, 10)


@pytest.mark.parametrize("fmt", ["dense", "int8_g64", "reference"])
def test_every_tensor_of_k_counts(fmt):
    for name in ("data", "scale", "data2", "scale2"):
        k, _ = cache(fmt)
        t = getattr(k, name)
        if t is None:
            continue
        # the last element that a row, a scale needs is the last that is there: without it they are not held
        flat, need = t.reshape(-1), {"data": [k.head_offset, k.pos_stride, k.stride_b], "data2": [k.head_offset2, k.pos_stride2, k.stride2_b],
                                     "scale": [[2 * k.scale_stride_h], [1], k.scale_stride_b],
                                     "scale2": [[2 * k.scale2_stride_h], [1], k.scale2_stride_b]}[name]
        width = {"dense": RANKS, "int8_g64": RANKS, "reference": [16, 5, 16]}[fmt] if name == "data" else \
            [4, 0, 12] if name == "data2" else [1]
        end = max(o + 9 * p + w for o, p, w in zip(need[0], need[1], width) if w) + need[2]
        setattr(k, name, flat[:end])
        assert k.holds(2, 10), name
        setattr(k, name, flat[:end - 1])
        assert not k.holds(2, 10), name
        setattr(k, name, flat[:0])
        assert not k.holds(1, 1), name


def test_a_last_row_that_ends_before_its_rank():
    x = torch.zeros(2 * 4 * 8)
    spec = lambda t: KLatentSpec(t, [8], [0], [8], 32, x, [0], 128)
    assert spec(x).holds(2, 4) and not spec(x[:-1]).holds(2, 4) and not spec(x[:-7]).holds(2, 4) and spec(x[:-1]).holds(2, 3)


@pytest.mark.parametrize("fmt", ["dense", "int8_g64", "reference"])
def test_every_tensor_of_v_counts(fmt):
    for name in ("data", "scale", "data2", "scale2", "zero"):
        _, v = cache(fmt)
        t = getattr(v, name)
        if t is None:
            continue
        for dim in range(3):
            short = t.narrow(dim, 0, t.shape[dim] - 1)
            setattr(v, name, short)
            assert not v.holds(2, 10), (name, dim)
        setattr(v, name, t)
        assert v.holds(2, 10)


def test_v_of_one_block():
    int8 = VLatentSpec.int8(torch.zeros(2, 9, 33, dtype=torch.int8), torch.zeros(2, 9, 1).half())
    nibbles = VLatentSpec.int4_ref(torch.zeros(2, 9, 17, dtype=torch.uint8), torch.zeros(2, 9, 1).half(), 33)
    for v in (int8, nibbles):
        assert v.holds(2, 9) and not v.holds(2, 10)
        v.scale = v.scale[:, :8]
        assert not v.holds(2, 9)


def test_b_k():
    b = torch.zeros(3, 40, 128)
    spec = lambda t: KLatentSpec(t, RANKS, [0] * 3, [1] * 3, 1, t, [h * 40 * 128 for h in range(3)], 128)
    assert spec(b).holds_bk() and not spec(b.view(-1)[:-1]).holds_bk() and not spec(b[:2]).holds_bk()
    assert not spec(torch.zeros(3, 128, 40).transpose(1, 2)).holds_bk()
