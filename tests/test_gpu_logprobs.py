"""GPU checks of starkv.token_logprobs against log_softmax in 64 bits.

Tolerance, in fp32 units u = 2^-24: with d = x - max and D = sum p |d|, each
term e^d of Z carries the rounding of its exponent (d log2 e: |d| u, and the
constant's error, less than |d| u) and the exponential's last bits (2 u); on
average over the terms that is (2 D + 2) u.  Sums run over at most V / 256
terms of a thread and 16 levels of merging, (V / 256 + 32) u.  ln Z, x - max
and their difference round once each.  So a log probability is off by at most
u (2 D + V / 256 + 40 + 2 |d| + 2 ln Z), the entropy, whose S / Z has those
errors relative to D, by (1 + D) times that."""
import math
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _flush(msg):
    print(msg, flush=True)
    sys.stdout.flush()


def check(x, tokens, top, res):
    """res against fp64 of the logits x [rows, V]."""
    xd = x.double().cpu()
    rows, V = xd.shape
    m = xd.amax(-1, keepdim=True)
    d = xd - m
    lnz = d.exp().sum(-1, keepdim=True).log()         # not logsumexp(x) - max: x may be 1e38
    lp = d - lnz
    p = lp.exp()
    ent = -torch.where(p == 0, 0.0, p * lp).sum(-1)      # NaN where the row has no distribution
    D = torch.where(p > 0, p * d.abs(), 0.0).sum(-1)        # (and 0 there)
    lnz = lnz.squeeze(-1)
    u = 2.0 ** -24
    base = u * (2 * D + V / 256 + 40 + 2 * lnz)
    ids = torch.sort(xd, dim=-1, descending=True, stable=True).indices[:, :top]
    got = [t.double().cpu() if t.is_floating_point() else t.cpu() for t in (res.entropy, res.top_logprobs, res.top_ids)]

    def near(a, b, lim):
        b = torch.where(b.abs() > torch.finfo(F32).max, b.float().double(), b)      # beyond fp32: infinity
        same = (a == b) | (a.isnan() & b.isnan())
        over = torch.where(same, 0.0, (a - b).abs() / lim)
        worst = float(over.max()) if over.numel() else 0.0
        assert worst <= 1.0, worst
        return worst
    w = [near(got[0], ent, (1 + D) * base)]
    assert torch.equal(got[2], ids)
    w.append(near(got[1], lp.gather(1, ids), base[:, None] + 2 * u * d.gather(1, ids).abs()))
    if tokens is not None:
        t = tokens.cpu()
        ok = (t >= 0) & (t < V)
        tc = t.clamp(0, V - 1)[:, None]
        want = torch.where(ok, lp.gather(1, tc).squeeze(1), math.nan)
        w.append(near(res.logprob.double().cpu(), want, base + 2 * u * torch.where(ok, d.gather(1, tc).squeeze(1).abs(), 0.0)))
    _flush(f"   worst error / bound: {', '.join('%.3f' % v for v in w)}")


@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,V,top", [(1, 1, 1), (3, 2, 2), (2, 7, 0), (5, 63, 5), (4, 64, 64), (3, 65, 64), (33, 1000, 5),
                                        (2, 1023, 20), (7, 4097, 33), (300, 3001, 8), (8, 32000, 5), (1, 131072, 20),
                                        (3, 100003, 64), (1, 300001, 1), (2000, 500, 3)])
def test_matches_log_softmax(rows, V, top, dtype):
    from starkv import token_logprobs
    _flush(f"[logprobs] {rows}x{V} top {top} {dtype}")
    g = torch.Generator(device="cuda").manual_seed(rows * 13 + V)
    x = (torch.randn(rows, V, generator=g, device="cuda") * 3).to(dtype)
    tok = torch.randint(0, V, (rows,), generator=g, device="cuda")
    res = token_logprobs(x, tok, top=top)
    torch.cuda.synchronize()
    assert res.logprob.dtype == F32 and res.top_ids.shape == (rows, top) and res.top_ids.dtype == torch.int64
    check(x, tok, top, res)
    again = token_logprobs(x, tok, top=top)
    assert all(torch.equal(a, b) for a, b in zip(res, again))


def _row_kinds(V, dtype):
    """Rows that go wrong easily, by name."""
    g = torch.Generator().manual_seed(V)
    n = torch.randn(V, generator=g) * 3
    inf = math.inf
    low = float(torch.finfo(dtype).min)
    k = {"normal": n}
    k["all equal"] = torch.full((V,), 1.5)
    k["ascending"] = torch.arange(V).float() / V * 20
    k["descending"] = -torch.arange(V).float() / V * 20
    k["few levels"] = torch.randint(0, 3, (V,), generator=g).float()
    t = torch.full((V,), -inf)
    t[[V // 3, V // 2, V - 1]] = torch.tensor([1.0, 2.0, 1.0])
    k["three allowed"] = t
    t = torch.full((V,), -inf)
    t[V - 2] = -5.0
    k["one allowed"] = t
    k["lowest mask"] = torch.where(torch.rand(V, generator=g) < 0.9, low, n)
    k["all lowest"] = torch.full((V,), low)
    k["none allowed"] = torch.full((V,), -inf)
    k["largest"] = torch.where(torch.rand(V, generator=g) < 0.5, float(torch.finfo(dtype).max), low)
    k["signed zeros"] = torch.where(torch.rand(V, generator=g) < 0.5, -0.0, 0.0)
    k["far below zero"] = n - 300
    t = n.clone()
    t[V // 2:] = -inf
    k["upper half barred"] = t
    # what one thread of a workgroup of 256, 512 or 1024 reads is large, the rest small
    for per in (256 * 8, 512 * 8, 1024 * 4):
        k[f"period {per}"] = torch.where(torch.arange(V) % per < 8, 5.0 + n.abs(), n - 20)
        k[f"not period {per}"] = torch.where(torch.arange(V) % per < 256 * 4, n - 20, 5.0 + n.abs())
    return k


@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("V,top", [(40, 8), (5000, 5), (32000, 64), (70001, 20)])
def test_hard_rows(V, top, dtype):
    from starkv import token_logprobs
    kinds = _row_kinds(V, dtype)
    _flush(f"[hard rows] V {V} top {top} {dtype}")
    x = torch.stack(list(kinds.values())).to(dtype).cuda()
    tok = torch.arange(len(kinds), device="cuda") * 7 % V
    res = token_logprobs(x, tok, top=top)
    torch.cuda.synchronize()
    for i, name in enumerate(kinds):
        _flush(f"   {name}")
        r = type(res)(res.logprob[i:i + 1], res.entropy[i:i + 1], res.top_logprobs[i:i + 1], res.top_ids[i:i + 1])
        check(x[i:i + 1], tok[i:i + 1], top, r)
        one = token_logprobs(x[i:i + 1], tok[i:i + 1], top=top)      # few rows: another launch shape
        check(x[i:i + 1], tok[i:i + 1], top, one)


@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("V", [9, 3000, 40000])
def test_nan_and_infinity(V, dtype):
    """A NaN or +inf makes its row NaN, and only its row; the alternatives put NaN first, as a descending sort does."""
    from starkv import token_logprobs
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(4, V, generator=g, device="cuda").to(dtype)
    clean = token_logprobs(x, torch.zeros(4, dtype=torch.int64, device="cuda"), top=4)
    x[1, V // 2] = math.nan
    x[1, V - 1] = math.nan
    x[2, 3] = math.inf
    res = token_logprobs(x, torch.zeros(4, dtype=torch.int64, device="cuda"), top=4)
    for r in (1, 2):
        assert res.logprob[r].isnan() and res.entropy[r].isnan() and res.top_logprobs[r].isnan().all()
    for r in (0, 3):
        assert all(torch.equal(a[r], b[r]) for a, b in zip(res, clean))
    assert res.top_ids[1, :2].tolist() == [V // 2, V - 1] and res.top_ids[2, 0] == 3
    want = torch.sort(x.float(), dim=-1, descending=True, stable=True).indices[:, :4]
    assert torch.equal(res.top_ids, want)


def test_tokens_outside_and_layouts():
    """Tokens outside [0, V) have no log probability; rows at any offset and stride; leading dims; no rows, no tokens."""
    from starkv import token_logprobs
    g = torch.Generator(device="cuda").manual_seed(2)
    wide = (torch.randn(6, 4100, generator=g, device="cuda") * 2)
    for dtype in (F16, BF16, F32):
        for lo, V in ((0, 4096), (1, 4001), (3, 130), (7, 4093)):
            x = wide.to(dtype)[:, lo:lo + V]
            tok = torch.tensor([0, V - 1, -100, V, 5, -1], device="cuda")
            check(x, tok, 6, token_logprobs(x, tok, top=6))
    x = wide.half()
    t3 = token_logprobs(x.view(2, 3, 4100), torch.zeros(2, 3, dtype=torch.int64, device="cuda"), top=2)
    flat = token_logprobs(x, torch.zeros(6, dtype=torch.int64, device="cuda"), top=2)
    assert t3.logprob.shape == (2, 3) and t3.top_ids.shape == (2, 3, 2)
    assert all(torch.equal(a.reshape(b.shape), b) for a, b in zip(t3, flat))
    none = token_logprobs(x, top=2)
    assert none.logprob is None and torch.equal(none.top_ids, flat.top_ids) and torch.equal(none.entropy, flat.entropy)
    empty = token_logprobs(x[:0], torch.zeros(0, dtype=torch.int64, device="cuda"), top=3)
    assert empty.logprob.shape == (0,) and empty.top_ids.shape == (0, 3)
    one = token_logprobs(x[0], torch.tensor(7, device="cuda"), top=1)
    assert one.logprob.shape == () and one.top_ids.shape == (1,)


def test_rows_beyond_are_left_alone():
    """Two launches on two streams and a captured one give what one stream gives."""
    from starkv import token_logprobs
    g = torch.Generator(device="cuda").manual_seed(4)
    xs = [torch.randn(r, V, generator=g, device="cuda").half() for r, V in ((1, 150000), (64, 9000))]
    toks = [torch.zeros(x.shape[0], dtype=torch.int64, device="cuda") for x in xs]
    want = [token_logprobs(x, t, top=9) for x, t in zip(xs, toks)]
    side = [torch.cuda.Stream() for _ in xs]
    got = []
    for s, x, t in zip(side, xs, toks):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(token_logprobs(x, t, top=9))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    for x, t in zip(xs, toks):
        xin = x.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r = token_logprobs(xin, t, top=9)
        for i in range(4):
            xin.copy_(x * (i - 1.5))
            graph.replay()
            e = token_logprobs(x * (i - 1.5), t, top=9)
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(r, e))


def test_offsets_past_32_bits():
    """More than 2^31 logits: rows on both sides of the border and the last one; and rows a long stride apart."""
    from starkv import token_logprobs
    V, rows = 32000, 70001
    x = torch.zeros(rows, V, dtype=BF16, device="cuda")
    at = torch.tensor([0, 67107, 67108, 67109, 70000])
    g = torch.Generator(device="cuda").manual_seed(2)
    x[at.cuda()] = (torch.randn(len(at), V, generator=g, device="cuda") * 3).bfloat16()
    tok = torch.randint(0, V, (rows,), generator=g, device="cuda")
    res = token_logprobs(x, tok, top=3)
    check(x[at.cuda()], tok[at.cuda()], 3, type(res)(*(t[at.cuda()] for t in res)))
    far = torch.as_strided(x, (2, V), (67109 * V, 1))
    check(far, tok[:2], 5, token_logprobs(far, tok[:2], top=5))


def test_refusals():
    from starkv import StarKVError, token_logprobs
    x = torch.zeros(2, 100, device="cuda")
    t = torch.zeros(2, dtype=torch.int64, device="cuda")
    for f in (lambda: token_logprobs(x, t, top=65), lambda: token_logprobs(x, t, top=-1),
              lambda: token_logprobs(x[:, :3], t, top=4), lambda: token_logprobs(x, t.int()),
              lambda: token_logprobs(x, t[:1]), lambda: token_logprobs(x.double(), t), lambda: token_logprobs(x.t(), t),
              lambda: token_logprobs(x, t.cpu()), lambda: token_logprobs(x[:, :0], t), lambda: token_logprobs(x.cpu(), t.cpu())):
        with pytest.raises(StarKVError):
            f()
