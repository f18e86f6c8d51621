"""Attention scores by position, selection and moved rows of bounded caches against plain fp64 / integer definitions."""
import math

import pytest
import torch

import starkv
from starkv import KLatentSpec, StarKVError, VLatentSpec, attention_scores, keep_positions, select_positions
from starkv.cache import LatentCache

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


# ---------------------------------------------------------------- scores
def scores_oracle(x):
    x = x.double()
    m = x.amax(-1, keepdim=True)
    w = torch.exp(x - torch.where(m > -math.inf, m, 0.0))
    t = w.sum(-1, keepdim=True)
    return (w / torch.where(t > 0, t, 1.0)).sum(1)


def score_bound(x):
    """fp32: a weight's exponent (x - m) log2 e carries two roundings (2^-24 each of up to R = max - min of what still
    counts, R <= 104: beyond exp(-104) a weight is below 2^-149), exp2 one unit in the last place, the product with
    1 / sum three roundings, sums over S and H by trees and short runs of at most 64 + H terms: all in all a relative
    (104 * 2 * ln 2 + 64 + H + 8) 2^-24 of the position's own sum; weights below 2^-126 may be flushed."""
    return (150 + 72 + x.shape[1]) * 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 1, 2), (2, 3, 31), (1, 5, 255), (3, 4, 257), (2, 8, 4095), (2, 33, 4097),
                                   (1, 64, 9001), (2, 100, 700), (1, 1024, 65)], ids=str)
def test_scores(shape, dtype):
    g = torch.Generator().manual_seed(sum(shape))
    x = (torch.randn(*shape, generator=g) * 3).to(dtype)
    got = attention_scores(x.to(DEV))
    want = scores_oracle(x)
    assert got.dtype == torch.float32 and got.shape == want.shape
    assert ((got.double().cpu() - want).abs() <= want * score_bound(x) + shape[1] * 2.0 ** -126).all()
    onto = torch.rand(shape[0], shape[2] + 3, generator=g).to(DEV)
    before = onto.clone()
    assert attention_scores(x.to(DEV), onto) is onto
    assert torch.equal(onto[:, shape[2]:], before[:, shape[2]:])
    assert torch.equal(onto[:, :shape[2]], before[:, :shape[2]] + got)


def test_scores_masks_infinities_nan():
    x = torch.randn(2, 4, 300)
    x[0, :, 100:] = -math.inf
    x[1, 2] = -math.inf                                # nothing left
    x[1, 3] = torch.finfo(torch.float32).min           # nothing but the type's lowest: a uniform row
    got = attention_scores(x.to(DEV)).cpu()
    want = scores_oracle(x)
    assert ((got.double() - want).abs() <= want * score_bound(x)).all()
    assert (got[0, 100:] == 0).all()
    x = torch.full((1, 3, 70), -math.inf)
    assert (attention_scores(x.to(DEV)) == 0).all()
    x[0, 1, 5] = 2.0
    got = attention_scores(x.to(DEV)).cpu()
    assert got[0, 5] == 1 and got.sum() == 1
    for bad in (math.nan, math.inf):
        x = torch.randn(2, 3, 5000)
        x[1, 1, 4500] = bad
        got = attention_scores(x.to(DEV)).cpu()
        assert torch.isnan(got[1]).all() and torch.isfinite(got[0]).all()


def test_scores_strides():
    base = torch.randn(3, 9, 1030).half().to(DEV)
    x = base[:, 1:8:2, 3:1000]
    assert torch.equal(attention_scores(x), attention_scores(x.contiguous()))
    wide = torch.randn(1, 4, 50).to(DEV).expand(3, 4, 50)
    got = attention_scores(wide)
    assert torch.equal(got[0], got[2])


def test_scores_large_magnitudes():
    x = torch.tensor([[[1e30, 1e30, -1e30, 0.0], [-3e38, -3e38, -3e38, -3e38]]])
    got = attention_scores(x.to(DEV)).cpu()
    assert torch.equal(got, torch.tensor([[0.75, 0.75, 0.25, 0.25]]))


@pytest.mark.parametrize("fmt", ["dense", "int8_g64", "reference"])
@pytest.mark.parametrize("Hq,Hkv,S", [(4, 4, 33), (16, 4, 700), (40, 8, 129)])
def test_decode_scores(fmt, Hq, Hkv, S):
    """decode_attention(scores=): the output of decode alone, and the weights of its logits.  The logits are taken from
    k_logits, whose keys are rounded like decode's; both are within d = 4 2^-11 |scale q| |k| of the true ones (see
    tests/test_gpu_prefix.py), so weights agree within exp(4 d)."""
    B, Rv = 3, 64
    ranks = [16 + 8 * (h % 4) for h in range(Hkv)]
    g = torch.Generator(device=DEV).manual_seed(S)
    mk = lambda *s: torch.randn(*s, generator=g, device=DEV).half()
    cache = LatentCache(B, ranks, Rv, S + 5, torch.float16, DEV, fmt)
    bk = mk(Hkv, 40, 128) / 6
    ks, vs, n = cache.append(mk(B, Hkv, S, 40), mk(B, S, Rv), bk)
    q, uv = mk(B, Hq, 128), mk(Hkv * 128, Rv) / 8
    want_out = starkv.decode_attention(q, ks, vs, uv, seq_len=n)
    sc = torch.full((B, S + 5), 0.5, device=DEV)
    out = starkv.decode_attention(q, ks, vs, uv, seq_len=n, scores=sc)
    assert torch.equal(out, want_out)
    logits = starkv.k_logits(q, ks, n, scale=128 ** -0.5)
    want = scores_oracle(logits.cpu())
    keys = [x.double() @ bk[h, :r].double() for h, (x, r) in enumerate(zip(cache.dequant_k(), ranks))]
    d = 4 * 2.0 ** -11 / math.sqrt(128) * q.double().norm(dim=-1).max() * max(k.norm(dim=-1).max() for k in keys)
    err = (sc[:, :S].double().cpu() - 0.5 - want).abs()
    assert (err <= want * torch.expm1(4 * d).cpu() + 2.0 ** -18).all()
    assert (sc[:, S:] == 0.5).all()
    assert abs(sc[:, :S].double().sum().item() - B * (Hq + 0.5 * S)) < 1e-2 * B * Hq


# ---------------------------------------------------------------- selection
def select_oracle(x, keep, n, sinks, recent):
    out = []
    for row in x[:, :n].tolist():
        key = lambda p: (math.inf if p < sinks or p >= n - recent else 0, row[p] if row[p] == row[p] else -math.inf, -p)
        order = sorted(range(n), key=key, reverse=True)[:keep]
        out.append(sorted(order))
    return torch.tensor(out, dtype=torch.int32).reshape(x.shape[0], keep)


@pytest.mark.parametrize("B,n,keep,sinks,recent", [
    (1, 1, 1, 0, 0), (1, 1, 0, 0, 0), (2, 5, 3, 1, 1), (3, 64, 64, 4, 8), (2, 100, 1, 0, 0), (2, 100, 99, 0, 0),
    (1, 4096, 1000, 4, 100), (2, 4097, 2000, 0, 0), (1, 5000, 4999, 1, 0), (4, 9001, 1234, 7, 301),
    (1, 20000, 5000, 4, 64), (2, 33000, 100, 3, 90), (1, 70001, 35000, 4, 1000), (3, 300, 12, 5, 7)])
@pytest.mark.parametrize("kind", ["spread", "ties", "zeros", "special"])
def test_select(B, n, keep, sinks, recent, kind):
    g = torch.Generator().manual_seed(n + keep)
    x = torch.exp(2 * torch.randn(B, n + 2, generator=g))
    if kind == "ties":
        x = torch.randint(0, 4, (B, n + 2), generator=g).float()
    elif kind == "zeros":
        x = torch.where(torch.rand(B, n + 2, generator=g) < 0.5, 0.0, -0.0)
    elif kind == "special":
        pick = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-45, -1e-45, 3e38, -1.0, 1.0])
        x = pick[torch.randint(0, 10, (B, n + 2), generator=g)]
    got = select_positions(x.to(DEV), keep, n, sinks, recent)
    assert got.dtype == torch.int32
    assert torch.equal(got.cpu(), select_oracle(x, keep, n, sinks, recent))


def test_select_strides_and_all():
    x = torch.rand(6, 900).to(DEV)[::2, 3:800]
    got = select_positions(x, 50, sinks=2, recent=3)
    assert torch.equal(got.cpu(), select_oracle(x.cpu(), 50, 797, 2, 3))
    assert torch.equal(select_positions(x, 797).cpu(), torch.arange(797).int().expand(3, 797))


# ---------------------------------------------------------------- moved rows
def kept(B, n, keep, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.rand(B, n, generator=g).topk(keep, -1).indices.sort(-1).values.int() if keep else torch.zeros(B, 0).int()


@pytest.mark.parametrize("fmt", ["dense", "int8_g64", "reference"])
@pytest.mark.parametrize("B,n,keep,Rv,dtype", [
    (1, 1, 1, 1, torch.float16), (2, 2, 1, 3, torch.bfloat16), (3, 50, 0, 64, torch.float16), (2, 50, 50, 64, torch.float16),
    (1, 301, 128, 333, torch.bfloat16), (3, 1000, 999, 640, torch.float16), (2, 5000, 1700, 1228, torch.float16),
    (4, 700, 350, 17, torch.float16)])
def test_keep(fmt, B, n, keep, Rv, dtype):
    ranks = [1, 17, 64, 101, 128, 40]
    cache = LatentCache(B, ranks, Rv, n + 3, dtype, DEV, fmt)
    g = torch.Generator(device=DEV).manual_seed(n)
    buffers = [t for t in vars(cache).values() if isinstance(t, torch.Tensor)]
    for t in buffers:                                  # every byte of every buffer, padding included
        t.untyped_storage()
        flat = t if t.is_contiguous() else None
        if flat is not None:
            flat.view(torch.uint8 if t.element_size() == 1 else torch.int16).random_(generator=g)
    cache.length = n
    before_k, before_v = [x.clone() for x in raw_k(cache)], [x.clone() for x in raw_v(cache)]
    everything = [t.clone() for t in buffers]
    p = kept(B, n, keep, seed=n)
    scores = torch.rand(B, n + 3, generator=g, device=DEV)
    old = scores.clone()
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    cache.keep(p.to(DEV), scores, flag)
    assert cache.length == keep and flag.item() == 0
    at = p.long().to(DEV)
    for now, was in zip(raw_k(cache) + raw_v(cache), before_k + before_v):
        index = at.view(B, keep, *[1] * (was.dim() - 2)).expand(B, keep, *was.shape[2:])
        assert torch.equal(now[:, :keep], was.gather(1, index))
        assert torch.equal(now[:, keep:], was[:, keep:])
    assert torch.equal(scores[:, :keep], old.gather(1, at))
    assert (scores[:, keep:n] == 0).all() and torch.equal(scores[:, n:], old[:, n:])
    # padding behind a row's bytes stays
    if fmt == "int8_g64":
        for h, r in enumerate(ranks):
            o, w = cache._k["head_offset"][h], cache._k["pos_stride"][h]
            rows = cache.k_data[:, o:o + cache.cap * w].view(B, cache.cap, w)[..., r:]
            was = everything[[id(b) for b in buffers].index(id(cache.k_data))]
            assert torch.equal(rows, was[:, o:o + cache.cap * w].view(B, cache.cap, w)[..., r:])


def raw_k(c):
    """Stored K bytes and scales by position: [B, capacity, ...] each."""
    out = []
    for h, r in enumerate(c.ranks):
        o, p = c._k["head_offset"][h], c._k["pos_stride"][h]
        nb = r if c.fmt != "reference" else min(r, 16)
        out.append(c.k_data[:, o:o + c.cap * p].view(c.B, c.cap, p)[..., :nb])
        if c.fmt == "reference" and r > 16:
            o, p = c._k["head_offset2"][h], c._k["pos_stride2"][h]
            out.append(c.k_data2[:, o:o + c.cap * p].view(c.B, c.cap, p)[..., :(r - 15) // 2])
    if c.fmt != "dense":
        out.append(c.k_scale[:, :, :c.cap].transpose(1, 2).view(torch.int16))
    if c.fmt == "reference":
        out.append(c.k_scale2.transpose(1, 2).view(torch.int16))
    return [t.view(torch.int16) if t.dtype in (torch.float16, torch.bfloat16) else t for t in out]


def raw_v(c):
    out = [c.v_data]
    for name in ("v_scale", "v_zero", "v_data2", "v_scale2"):
        if hasattr(c, name):
            out.append(getattr(c, name))
    return [t.view(torch.int16) if t.dtype in (torch.float16, torch.bfloat16) else t for t in out]


def test_keep_refuses_positions_row_by_row():
    """Positions below their own row or past the length leave the row and set the flag."""
    x = torch.arange(2 * 10 * 8, device=DEV).half().view(2, 1, 10, 8)
    v = torch.arange(2 * 10 * 5, device=DEV).half().view(2, 10, 5).clone()
    k = KLatentSpec(x, [8], [0], [8], x.stride(0), x, [0], 128)
    kx, vx = x.clone(), v.clone()
    p = torch.tensor([[0, 3, 1, 10], [1, 2, -1, 9]], dtype=torch.int32, device=DEV)
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    keep_positions(k, v, p, 10, error_flag=flag)
    assert flag.item() == 1
    for b, moved in enumerate(([0, 3, 2, 3], [1, 2, 2, 9])):
        assert torch.equal(x[b, 0, :4], kx[b, 0, moved]) and torch.equal(v[b, :4], vx[b, moved])
    assert torch.equal(x[:, :, 4:], kx[:, :, 4:])


def test_keep_many_rows_in_place():
    """Long rows moved a little and a lot: every source is read before it is overwritten."""
    for step in (1, 2, 7):
        n, Rv = 20000, 200
        v = torch.randint(-30000, 30000, (2, n, Rv), device=DEV, dtype=torch.int16).view(torch.float16)
        x = torch.randint(-30000, 30000, (2, 2, n, 24), device=DEV, dtype=torch.int16).view(torch.float16)
        k = KLatentSpec(x, [24, 5], [0, x.stride(1)], [24, 24], x.stride(0), x, [0, 0], 128)
        p = (torch.arange(0, n - 3, step, device=DEV, dtype=torch.int32) + 3).expand(2, -1).contiguous()
        wv, wk = v.view(torch.int16).clone(), x.view(torch.int16).clone()
        keep_positions(k, v, p, n)
        m = p.shape[1]
        assert torch.equal(v.view(torch.int16)[:, :m], wv[:, p[0].long()])
        assert torch.equal(x.view(torch.int16)[:, 0, :m], wk[:, 0, p[0].long()])
        assert torch.equal(x.view(torch.int16)[:, 1, :m, :5], wk[:, 1, p[0].long(), :5])
        assert torch.equal(x.view(torch.int16)[:, 1, :m, 5:], wk[:, 1, :m, 5:])
        assert torch.equal(v.view(torch.int16)[:, m:], wv[:, m:])


def test_bounded_decode_together():
    """A cache that is decoded with scores, bounded, appended to and decoded again equals one that held the kept rows
    from the start."""
    B, ranks, Rv, cap = 2, [16, 24, 40], 96, 64
    g = torch.Generator(device=DEV).manual_seed(3)
    mk = lambda *s: torch.randn(*s, generator=g, device=DEV).half()
    bk, uv = mk(3, 40, 128) / 6, mk(384, Rv) / 9
    for fmt in ("dense", "int8_g64", "reference"):
        cache = LatentCache(B, ranks, Rv, cap, torch.float16, DEV, fmt)
        k0, v0 = mk(B, 3, 60, 40), mk(B, 60, Rv)
        ks, vs, n = cache.append(k0, v0, bk)
        scores = torch.zeros(B, cap, device=DEV)
        for _ in range(3):
            starkv.decode_attention(mk(B, 6, 128), ks, vs, uv, seq_len=n, scores=scores)
        assert abs(scores.sum().item() - 3 * B * 6) < 0.1
        p = cache.bound(20, scores, sinks=2, recent=5)
        assert torch.equal(p.cpu(), select_oracle_of(scores_before=None, p=p.cpu()))
        k1, v1, q = mk(B, 3, 1, 40), mk(B, 1, Rv), mk(B, 6, 128)
        ks, vs, n = cache.append(k1, v1, bk)
        assert n == 21 and (scores[:, 20:60] == 0).all()
        got = starkv.decode_attention(q, ks, vs, uv, seq_len=n)
        other = LatentCache(B, ranks, Rv, cap, torch.float16, DEV, fmt)
        i = p.long()
        other.append(k0.gather(2, i[:, None, :, None].expand(B, 3, 20, 40)), v0.gather(1, i[..., None].expand(B, 20, Rv)), bk)
        ks, vs, n = other.append(k1, v1, bk)
        assert torch.equal(got, starkv.decode_attention(q, ks, vs, uv, seq_len=n))


def select_oracle_of(scores_before, p):
    """What any selection with two sinks and five recent ones of 60 has to look like."""
    assert (p[:, :2] == torch.tensor([0, 1])).all() and (p[:, -5:] == torch.arange(55, 60)).all()
    assert (p[:, 1:] > p[:, :-1]).all()
    return p


def test_graph_of_scores_selection_and_move():
    """Scores, selection and move captured together and replayed, against the same eagerly."""
    B, H, n, keep = 2, 6, 900, 300
    logits = torch.randn(B, H, n, device=DEV)
    v = torch.randn(B, n, 40, device=DEV).half()
    x = torch.randn(B, 1, n, 16, device=DEV).half()
    spec = lambda t: KLatentSpec(t, [16], [0], [16], t.stride(0), t, [0], 128)

    def run(x, v):
        s = attention_scores(logits)
        p = select_positions(s, keep, sinks=1, recent=9)
        keep_positions(spec(x), v, p, n, s)
        return s, p

    run(x.clone(), v.clone())
    g = torch.cuda.CUDAGraph()
    gx, gv = x.clone(), v.clone()
    with torch.cuda.graph(g):
        gs, gp = run(gx, gv)
    for step in range(4):
        logits.copy_(torch.randn(B, H, n))
        gx.copy_(x)
        gv.copy_(v)
        ex, ev = x.clone(), v.clone()
        es, ep = run(ex, ev)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in ((gs, es), (gp, ep), (gx, ex), (gv, ev))), step


def test_refusals():
    x = torch.zeros(2, 4, 8, device=DEV)
    s = torch.zeros(2, 8, device=DEV)
    v = torch.zeros(2, 8, 16, device=DEV).half()
    kx = torch.zeros(2, 1, 8, 16, device=DEV).half()
    k = KLatentSpec(kx, [16], [0], [16], kx.stride(0), kx, [0], 128)
    one = KLatentSpec(kx, [16], [0], [16], 0, kx, [0], 128)
    p = torch.arange(3, dtype=torch.int32, device=DEV).expand(2, 3).contiguous()
    bad = [
        lambda: attention_scores(x.cpu()), lambda: attention_scores(x[0]), lambda: attention_scores(x.double()),
        lambda: attention_scores(x.transpose(1, 2)), lambda: attention_scores(x, s[:, :7]), lambda: attention_scores(x, s.half()),
        lambda: attention_scores(x[:, :0]), lambda: attention_scores(torch.zeros(1, 1025, 2, device=DEV)),
        lambda: attention_scores(x, s[:1].expand(2, 8)),
        lambda: select_positions(s, 9), lambda: select_positions(s, 3, sinks=2, recent=2), lambda: select_positions(s, -1),
        lambda: select_positions(s, 3, length=9), lambda: select_positions(s.half(), 3), lambda: select_positions(s.t(), 1),
        lambda: select_positions(s, 3, sinks=-1), lambda: select_positions(s.cpu(), 3),
        lambda: keep_positions(k, v, p.long(), 8), lambda: keep_positions(k, v, p[:1], 8), lambda: keep_positions(k, v, p, 2),
        lambda: keep_positions(k, v, p, 9), lambda: keep_positions(one, v, p, 8), lambda: keep_positions(k, v, p.cpu(), 8),
        lambda: keep_positions(k, v, p, 8, scores=s[:, :7]), lambda: keep_positions(k, v, p[:1].expand(2, 3), 8),
        lambda: keep_positions(k, v[:1].expand(2, 8, 16), p, 8),
        lambda: keep_positions(k, v, p, 8, error_flag=torch.zeros(1, device=DEV)),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(StarKVError):
            f()
            pytest.fail(f"call {i} was not refused")


def test_keep_offsets_past_32_bits():
    """A V latent of 4.9 GB, in pieces that are checked one by one."""
    n, w = 300000, 8192
    v = torch.empty(1, n, w, dtype=torch.float16, device=DEV)
    rows = torch.arange(n, device=DEV)
    v.copy_((rows % 2039)[None, :, None])                                          # exact in fp16
    v[0, :, -1] = (rows // 2039).half()
    k = torch.stack((rows % 2039, rows // 2039), -1).half()[None, None].contiguous()
    spec = KLatentSpec(k, [2], [0], [2], k.stride(0), k, [0], 128)
    pos = torch.cat((torch.arange(3), torch.arange(n - 280001, n - 1)))[None].int().to(DEV)
    keep_positions(spec, v, pos, n)
    for i in range(0, pos.shape[1], 20000):
        want = pos[0, i:i + 20000].long()
        got = v[0, i:i + len(want)]
        assert torch.equal(got[:, :-1], (want % 2039).half()[:, None].expand(-1, w - 1))
        assert torch.equal(got[:, -1], (want // 2039).half())
        assert torch.equal(k[0, 0, i:i + len(want)], torch.stack((want % 2039, want // 2039), -1).half())
    assert torch.equal(v[0, pos.shape[1]:, 0], (rows[pos.shape[1]:] % 2039).half())


@pytest.mark.parametrize("order", ["position, sequence, head", "head, sequence, position", "sequence, position, head"])
def test_keep_of_other_orders(order):
    """Latents whose sequences or heads lie inside a position's row, or behind another."""
    B, H, n, r = 3, 2, 50, 24
    dims = {"sequence": B, "position": n, "head": H}
    names = order.split(", ")
    g = torch.Generator().manual_seed(7)
    x = torch.randn(*(dims[a] for a in names), r, generator=g).half().to(DEV)
    x = x.permute(*(names.index(a) for a in ("sequence", "head", "position")), 3)  # [B, H, n, r]
    spec = KLatentSpec(x, [r] * H, [h * x.stride(1) for h in range(H)], [x.stride(2)] * H, x.stride(0), x, [0] * H, 128)
    v = torch.randn(n, B, 16, generator=g).half().to(DEV).transpose(0, 1)
    pos = kept(B, n, 20).to(DEV)
    at = pos.long()
    want_k = x.gather(2, at[:, None, :, None].expand(B, H, 20, r))
    want_v, rest = v.gather(1, at[..., None].expand(B, 20, 16)), v[:, 20:].clone()
    keep_positions(spec, v, pos, n)
    assert torch.equal(x[:, :, :20], want_k) and torch.equal(v[:, :20], want_v) and torch.equal(v[:, 20:], rest)


def test_keep_refuses_shared_rows():
    k0 = torch.zeros(2, 1, 8, 16, device=DEV).half()
    v = torch.zeros(2, 8, 16, device=DEV).half()
    p = torch.arange(3, dtype=torch.int32, device=DEV).expand(2, 3).contiguous()
    for x in (k0.expand(2, 3, 8, 16), k0[:1].expand(2, 1, 8, 16)):
        spec = KLatentSpec(x, [16] * x.shape[1], [h * x.stride(1) for h in range(x.shape[1])], [16] * x.shape[1], x.stride(0),
                           k0, [0] * x.shape[1], 128)
        with pytest.raises(StarKVError):
            keep_positions(spec, v, p, 8)
    with pytest.raises(StarKVError):
        keep_positions(KLatentSpec(k0[:, :, :7], [16], [0], [16], k0.stride(0), k0, [0], 128), v, p, 8)


@pytest.mark.parametrize("between", [28672, 28673, 57345])
@pytest.mark.parametrize("kind", ["spread", "one value", "all -inf"])
def test_select_where_rows_begin_to_be_split(between, kind):
    """The longest row of one workgroup, the shortest in pieces, and a last piece of one position."""
    g = torch.Generator().manual_seed(between)
    x = torch.exp(2 * torch.randn(2, between + 9, generator=g))
    if kind != "spread":
        x.fill_(1.5 if kind == "one value" else -math.inf)
    for keep in (10, between // 3, between + 8):
        got = select_positions(x.to(DEV), keep, sinks=4, recent=5)
        assert torch.equal(got.cpu(), select_oracle(x, keep, between + 9, 4, 5))
