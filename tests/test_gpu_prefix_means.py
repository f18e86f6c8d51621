"""Means of a shared prefix's values that cancel, of values far below one: sums of splits keep their bits."""
import pytest
import torch

from starkv import prefix_decode_attention
from test_gpu_prefix import DEV, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,vx", [(torch.float16, 1.0), (torch.float16, 1e-3), (torch.float16, 1e-4), (torch.bfloat16, 1e-4)])
def test_nearly_uniform_weights_over_small_values(dtype, vx):
    """Values of N(0, vx^2), weights all nearly 2^-15: an output is vx / 181 of them, and a split's mean not much more.
    Roundings of weights add by their squares, as the values do: each of the three to fp16 that a weight may take is off by
    up to 2^-11 and by 2^-11 / sqrt(3) at most in the mean of squares, 2^-11 together.  The logits here are below 2^-3
    and off by 2^-9 of that.  fp32 sums of 2^15 terms in parts of 2^11: 2^-13 at most."""
    c = Case(2, 4, 2, 32768, 0, 8, 8, 64, dtype, seed=71, vx=vx, qx=0.002)
    got = prefix_decode_attention(c.q.to(DEV), c.prefix(), None, None, c.dev(c.uv), out_dtype=torch.float32)
    want, _, w = c.oracle()
    assert w.max() < 2.0 ** -14
    rel = (got.double().cpu() - want).norm() / want.norm()
    assert rel < 2.0 ** -11 + 2.0 ** -12 + 2.0 ** -13, rel


def test_columns_of_very_different_values():
    """A column of values 2^-30 of the largest column's, met by a U_v that reads it alone.  Its mean is 2^-38 of the row's
    largest, and the up-projection takes a row in two fp16 terms, the largest value at 2^14 or more: what they leave is
    below 2^-25 of that scale, 2^-39 of the largest.  The roundings of the weights, each 2^-11 at most, add to the error as
    the values themselves do, by their squares: four times 2^-11 of sqrt(sum w^2 v^2) for one column of one output."""
    P = 32768
    c = Case(1, 1, 1, P, 0, 8, 8, 2, torch.float16, seed=73, qx=0.002)
    g = torch.Generator().manual_seed(5)
    c.pv = torch.stack((torch.full((P,), 65504.0), torch.randn(P, generator=g) * 6e-5), -1).half()
    c.uv = torch.zeros(128, 2).half()
    c.uv[:, 1] = 1.0
    got = prefix_decode_attention(c.q.to(DEV), c.prefix(), None, None, c.uv.to(DEV), out_dtype=torch.float32)
    want, _, w = c.oracle()
    spread = (w[0, 0] * c.pv[:, 1].double()).norm()
    assert (got.double().cpu() - want).abs().max() <= 2.0 ** -39 * 65504 + 4 * 2.0 ** -11 * spread
