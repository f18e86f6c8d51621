"""Own latents that are no numbers behind a shared prefix: they show where they count, whatever else the row masks."""
import math

import pytest
import torch

from starkv import KLatentSpec, prefix_decode_attention
from test_gpu_prefix import DEV, Case

pytestmark = pytest.mark.gpu

LOW = [(-math.inf, torch.float32), (torch.finfo(torch.float32).min, torch.float32), (-1e30, torch.float32),
       (torch.finfo(torch.float16).min, torch.float16), (torch.finfo(torch.bfloat16).min, torch.bfloat16)]


def quantised(S, dtype, bad):
    """(arguments, K scales): three sequences of S own int8 rows; the scales of the second's rows `bad` are NaN."""
    c = Case(3, 8, 4, 70, S, 16, 32, 64, dtype, seed=51)
    c.ranks = [16] * 4
    scale = torch.full((3, 4, S, 1), 0.01, device=DEV).half()
    scale[1, :, bad] = math.nan
    x = torch.randint(-90, 90, (3, 4, S, 16), generator=torch.Generator().manual_seed(2)).to(torch.int8).to(DEV)
    k = KLatentSpec.from_reference_quant(x, scale, c.bk[:, :16].contiguous().to(DEV), 16)
    return (c.q.to(DEV), c.prefix(), k, c.v.to(DEV).contiguous(), c.uv.to(DEV)), scale


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("S,valid", [(5, 3), (40, 1), (700, 333)])
@pytest.mark.parametrize("low,mdtype", LOW, ids=str)
def test_quantised_rows_that_keep_nothing_but_nan(S, valid, low, mdtype, dtype):
    args, scale = quantised(S, dtype, slice(0, valid))
    mask = torch.zeros(3, 1, S, dtype=mdtype)
    mask[1, :, valid:] = low
    sums = torch.zeros(3, S, device=DEV)
    got = prefix_decode_attention(*args, mask=mask.to(DEV), scores=sums)
    scale[1] = 0.01
    clean_sums = torch.zeros(3, S, device=DEV)
    clean = prefix_decode_attention(*args, mask=mask.to(DEV), scores=clean_sums)
    assert torch.isnan(got[1]).all() and torch.isfinite(clean).all()
    assert torch.equal(got[::2], clean[::2])
    assert torch.isnan(sums[1]).all() and torch.equal(sums[::2], clean_sums[::2])


@pytest.mark.parametrize("S,last", [(5, 2), (64, 0), (700, 400)])
def test_quantised_rows_that_keep_nothing_but_nan_up_to_last_pos(S, last):
    args, scale = quantised(S, torch.float16, slice(0, last + 1))
    pos = torch.tensor([last], dtype=torch.int32, device=DEV)
    got = prefix_decode_attention(*args, last_pos=pos)
    scale[1] = 0.01
    clean = prefix_decode_attention(*args, last_pos=pos)
    assert torch.isnan(got[1]).all() and torch.isfinite(clean).all() and torch.equal(got[::2], clean[::2])


def test_quantised_rows_whose_nan_is_all_masked_are_the_prefix_alone():
    """As where nothing is masked finitely: no unmasked position of the row has a logit."""
    args, _ = quantised(40, torch.float16, slice(0, 40))
    alone = prefix_decode_attention(args[0], args[1], None, None, args[4])[1].float()
    for low, mdtype in LOW:
        mask = torch.zeros(3, 1, 40, dtype=mdtype)
        mask[1] = low
        got = prefix_decode_attention(*args, mask=mask.to(DEV))[1].float()
        # the prefix's sums in another split, fp32 (2^-16), before the output's rounding
        assert ((got - alone).abs() <= 2.0 ** -10 * alone.abs() + 2.0 ** -14).all()
