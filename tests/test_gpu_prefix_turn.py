"""The turn of queries past a long prefix, and the single rounding of its weights."""
import math

import pytest
import torch

from starkv import RopeConfig, prefix_decode_attention
from test_gpu_prefix import DEV, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("theta", [1e4, 5e5])
def test_turn_past_a_long_prefix(theta):
    """Query and first key in one frequency's plane, at a length where an fp32 product with that frequency is off most.
    The first key's logit is placed near 0, where it follows the angle most: A = 16 times an error of the angle.  Its own
    error: the key is exact (angle 0), the turned query's component is near 0 and keeps 2^-11 of itself.  Its weight is
    1 of 65000, so its value's share of the output is off by that error and two roundings to fp16 (2^-11 each)."""
    inv = RopeConfig(theta=theta).inv_freq()
    lengths = torch.arange(64500, 65500)
    off = (lengths[:, None].float() * inv).double() - lengths[:, None].double() * inv.double()
    at = int(off.abs().argmax())
    P, i = int(lengths[at // 64]), at % 64
    assert off.flatten()[at].abs() > 2.0 ** -10
    c = Case(1, 1, 1, P, 0, 1, 1, 1, torch.float16, seed=1, theta=theta)
    for t in (c.pk, c.bk, c.q, c.pv):
        t.zero_()
    c.pk[0, 0, 0], c.bk[0, 0, i], c.pv[0, 0] = 8.0, 1.0, 1.0
    turned = float(P * inv[i].double())                          # the direction that this turn takes to a right angle
    size = 16 * math.sqrt(128) / 8
    c.q[0, 0, i], c.q[0, 0, 64 + i] = size * math.sin(turned), size * math.cos(turned)
    c.uv = torch.ones(128, 1).half()
    want, _, w = c.oracle()
    assert abs(math.log(w[0, 0, 0].item() * P)) < 0.1
    got = prefix_decode_attention(c.q.to(DEV), c.prefix(), None, None, c.uv.to(DEV), out_dtype=torch.float32)
    rel = ((got.double().cpu() - want).abs() / want.abs()).max()
    assert rel < 3 * 2.0 ** -11, rel


@pytest.mark.parametrize("a,b,c3", [(-0.765625, -1.654296875, -0.70263671875), (2.966796875, 2.025390625, 2.990234375),
                                    (2.453125, 1.556640625, 2.48828125), (-0.9765625, -1.876953125, -0.96435546875)])
def test_weights_are_rounded_once(a, b, c3):
    """63 positions of one weight in a strip whose maximum is another's, below the next strip's: where values are all 1,
    the output is off by their rounding alone, 2^-11 at most (and fp32 sums).  (At these logits the roundings of the
    weight, the strip's factor and their product would fall the same way, 1.7 times 2^-11.)"""
    c = Case(1, 1, 1, 128, 0, 1, 1, 1, torch.float16, seed=1, theta=1e9)
    for t in (c.pk, c.bk, c.q):
        t.zero_()
    c.q[..., 63] = 8                                             # the slowest frequency: no turn to speak of
    c.bk[0, 0, 63] = 1
    c.pk[0, :64, 0] = b
    c.pk[0, 0, 0] = a
    c.pk[0, 64:, 0] = -80.0
    c.pk[0, 64, 0] = c3
    c.pv.fill_(1.0)
    c.uv = torch.ones(128, 1).half()
    got = prefix_decode_attention(c.q.to(DEV), c.prefix(), None, None, c.uv.to(DEV), out_dtype=torch.float32)
    assert (got.double() - 1).abs().max() <= 2.0 ** -11 + 2.0 ** -16
