"""GPU checks of starkv.token_logprobs on rows of large finite logits: masks of
a finite value other than the type's lowest, maxima of every magnitude, and
rows on both sides of +-2^20, where the kernel goes from sums in units of log 2
over the rounded maximum to sums over x - max.  Against log_softmax in 64 bits,
within test_gpu_logprobs.py's bound: neither way of summing has a term that
grows with |max| (x - max is rounded once, |d| u, which the bound holds; what
fl(max log2 e) is short of max log2 e is known exactly and taken back by one
exponential, 2 u, one product and one difference).

Each kind of row is given as one of many (a workgroup a row) and alone; the
longest alone are split over workgroups, pieces wholly of masked logits among
them."""
import math

import pytest
import torch

from test_gpu_logprobs import BF16, F16, F32, _flush, check

pytestmark = pytest.mark.gpu

MAGNITUDES = (1e6, 2.0 ** 20, 1e9, 3e9, 1e10, 1e11, 1e12, 1e18, 1e20, 1e25, 9e29, 1e30, 3e38)


def _kinds(V, a):
    """Rows with the magnitude a, by name."""
    g = torch.Generator().manual_seed(V)
    n = torch.randn(V, generator=g) * 3
    some = torch.rand(V, generator=g) < 0.9
    at = torch.arange(V)
    one = n.clone()
    one[V // 3] = a
    last = torch.full((V,), -a)
    last[V - 1] = 2.0
    return {
        "nine of ten masked": torch.where(some, -a, n),
        "all masked": torch.full((V,), -a),
        "the first three quarters masked": torch.where(at < 3 * V // 4, -a, n),
        "the last three quarters masked": torch.where(at >= V // 4, -a, n),
        "one allowed": last,
        "masked, some barred": torch.where(some, -a, -math.inf),
        "one large": one,
        "nine of ten large": torch.where(some, a, n),
        "all large": torch.full((V,), a),
        "large over masked": torch.where(some, -a, a),
        "the first quarter large": torch.where(at < V // 4, a, n),
    }


def _all(kinds, top, dtype):
    from starkv import token_logprobs
    V = next(iter(kinds.values())).shape[0]
    x = torch.stack(list(kinds.values())).to(dtype).cuda()
    tok = torch.arange(len(kinds), device="cuda") * 131 % V
    res = token_logprobs(x, tok, top=top)
    torch.cuda.synchronize()
    wrong = []
    for i, name in enumerate(kinds):
        one = token_logprobs(x[i:i + 1], tok[i:i + 1], top=top)
        for how, r in (("of many", type(res)(*(t[i:i + 1] for t in res))), ("alone", one)):
            try:
                check(x[i:i + 1], tok[i:i + 1], top, r)
            except AssertionError:
                wrong.append(f"{name}, {how}")
    assert not wrong, wrong


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("a", MAGNITUDES, ids=lambda a: f"{a:.3g}")
@pytest.mark.parametrize("V,top", [(40, 8), (5000, 5), (32000, 0), (131072, 20)])
def test_finite_masks_and_large_maxima(V, top, a, dtype):
    _flush(f"[magnitudes] V {V} top {top} {a:.3g} {dtype}")
    _all(_kinds(V, a), top, dtype)


@pytest.mark.parametrize("a", [1000.0, 30000.0, 65504.0])
@pytest.mark.parametrize("V,top", [(5000, 5), (131072, 20)])
def test_fp16_masks(V, top, a):
    _flush(f"[magnitudes] V {V} top {top} {a:.3g} fp16")
    _all(_kinds(V, a), top, F16)


@pytest.mark.parametrize("sign", [-1, 1], ids=["below", "above"])
@pytest.mark.parametrize("V,top", [(300, 7), (5000, 5), (131072, 20)])
def test_rows_across_the_limit(V, top, sign):
    """Logits within a few units of +-2^20, on one side, the other, and both: what either side adds counts."""
    _flush(f"[limit] V {V} top {top} {sign}")
    g = torch.Generator().manual_seed(V + sign)
    c = sign * 2.0 ** 20
    n = torch.randn(V, generator=g) * 2
    ramp = torch.linspace(-6, 6, V)
    _all({"both sides": c + n, "inside": c - sign * (n.abs() + 0.125), "outside": c + sign * (n.abs() + 0.125),
          "at it": torch.full((V,), c), "next to it, inside": torch.full((V,), c * (1 - 2.0 ** -24)),
          "next to it, outside": torch.full((V,), c * (1 + 2.0 ** -23)),
          "pieces on either side, ascending": c + ramp, "pieces on either side, descending": c - ramp,
          "a step across it": c + torch.where(torch.arange(V) < V // 2, -0.5, 0.5)}, top, F32)


def test_a_long_row_in_a_graph():
    """A masked row that is split over workgroups, captured once and replayed on other rows."""
    from starkv import token_logprobs
    kinds = [t.cuda()[None].contiguous() for t in _kinds(131072, 1e10).values()]
    tok = torch.tensor([5], device="cuda")
    x = kinds[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = token_logprobs(x, tok, top=9)
    for row in kinds:
        x.copy_(row)
        graph.replay()
        eager = token_logprobs(row, tok, top=9)
        torch.cuda.synchronize()
        check(row, tok, 9, r)
        assert all(torch.equal(a, b) for a, b in zip(r, eager))
