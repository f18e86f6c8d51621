"""Own keys outside fp16's range behind a shared prefix, and what lies in masked places beside them."""
import math

import pytest
import torch

from test_gpu_prefix import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,kx,bx,qx", [(torch.float16, 15000.0, 8.0, 1e-5), (torch.float16, 1.0, 1.0, 1.0),
                                            (torch.float16, 15000.0, 1e-3, 0.06), (torch.bfloat16, 3e4, 1.0, 2e-5),
                                            (torch.bfloat16, 1e8, 1e3, 1e-11), (torch.bfloat16, 1e-5, 1.0, 1e5)])
@pytest.mark.parametrize("shape", [(3, 8, 4, 130, 70, 9, 61, 64), (2, 8, 8, 64, 1000, 3, 128, 33), (2, 64, 1, 70, 33, 127, 127, 40)],
                         ids=str)
def test_keys_of_large_and_small_magnitude(shape, dtype, kx, bx, qx):
    c = Case(*shape, dtype, seed=sum(shape), kx=kx, qx=qx, pad=1)
    for t in (c.k, c.pk):                                        # draws past 4.4 sigma of 15000 are no fp16 numbers
        t.clamp_(-torch.finfo(dtype).max, torch.finfo(dtype).max)
    c.bk = (c.bk.float() * bx).to(dtype)
    own = (c.k.float() @ c.bk.float()).abs().max()
    assert own > 65504 or kx * bx < 100
    c.check(c.run())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_rows_of_one_tile_keep_their_own_scale(dtype):
    """Keys of magnitudes 2^0 to 2^17 beside one another: the small ones, whose queries are as large, stay exact."""
    c = Case(2, 4, 4, 70, 96, 16, 64, 64, dtype, seed=83, kx=1.0, qx=1.0)
    big = torch.zeros(96, dtype=torch.bool)
    big[::5] = True
    c.k[:, :, big] = (c.k[:, :, big].float() * 2.0 ** 13).to(dtype)
    c.bk = (c.bk.float() * 2.0 ** 4).to(dtype)
    c.q = (c.q.float() * 2.0 ** -4).to(dtype)
    m = torch.zeros(2, 96).masked_fill(big, -math.inf)           # the large ones are taken out, the rest counts
    assert (c.k.float() @ c.bk.float()).abs().max() > 65504
    kept = Case(2, 4, 4, 70, 96, 16, 64, 64, dtype, seed=83)
    kept.k, kept.bk, kept.q = c.k.masked_fill(big[:, None], 0.0), c.bk, c.q
    kept.check(c.run(m), m)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("mdtype", [torch.float32, torch.float16, torch.bfloat16])
def test_padding_of_infinities_is_not_looked_at(mdtype, bad, dtype):
    """Own dense K latents that are no finite numbers in masked places, beside keys past 65504: as if they held zeros."""
    for low in (torch.finfo(mdtype).min, -math.inf):
        c = Case(3, 8, 4, 130, 40, 16, 32, 64, dtype, seed=53, kx=15000.0, qx=1e-5)
        for t in (c.k, c.pk):                                    # as above
            t.clamp_(-torch.finfo(dtype).max, torch.finfo(dtype).max)
        c.bk = (c.bk.float() * 8).to(dtype)
        keep = torch.tensor([40, 17, 0])
        mask = torch.zeros(3, 1, 40).masked_fill_(torch.arange(40) >= keep[:, None, None], low).to(mdtype)
        pad = (mask[:, 0] < 0)[:, None, :, None]
        c.k = c.k.masked_fill(pad, 0.0)
        want = c.run(mask)
        c.check(want, mask)
        c.k = c.k.masked_fill(pad, bad)
        assert torch.equal(c.run(mask), want)
        c.k[1, :, 3] = bad
        got = c.run(mask)
        assert torch.isnan(got[1]).all() and torch.equal(got[::2], want[::2])


def test_one_infinite_rank_in_a_masked_place():
    """A single infinite element gives infinite keys, which a finite mask does not take out."""
    c = Case(3, 8, 4, 130, 40, 16, 32, 64, torch.float16, seed=53)
    mask = torch.zeros(3, 1, 40)
    mask[:, :, 20:] = torch.finfo(torch.float32).min
    want = c.run(mask)
    c.k[:, :, 25, 2] = math.inf
    assert torch.equal(c.run(mask), want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_finite_value_padding_has_no_weight(dtype):
    """Own V rows in masked places may hold any finite number (their weight is 0, not their place in the product)."""
    c = Case(3, 8, 4, 130, 40, 16, 32, 64, dtype, seed=53)
    keep = torch.tensor([40, 17, 0])
    mask = torch.zeros(3, 1, 40).masked_fill_(torch.arange(40) >= keep[:, None, None], -math.inf)
    want = c.run(mask)
    c.v = c.v.masked_fill((mask[:, 0] < 0)[:, :, None], torch.finfo(dtype).max)
    assert torch.equal(c.run(mask), want)


def test_value_padding_that_is_no_number_shows_where_others_are_kept():
    """V rows have to be finite: a NaN one in a masked place makes its row NaN if the row keeps other own positions, as
    decode_attention has it, and is not read if it keeps none."""
    c = Case(3, 8, 4, 130, 40, 16, 32, 64, torch.float16, seed=53)
    keep = torch.tensor([40, 17, 0])
    mask = torch.zeros(3, 1, 40).masked_fill_(torch.arange(40) >= keep[:, None, None], -math.inf)
    want = c.run(mask)
    c.v = c.v.masked_fill((mask[:, 0] < 0)[:, :, None], math.nan)
    got = c.run(mask)
    assert torch.isnan(got[1]).all() and torch.equal(got[::2], want[::2])
