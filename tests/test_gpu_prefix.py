"""Decode over a shared prefix (starkv.prefix_decode_attention) against its definition in 64 bits.

Tolerance.  A logit's relative roundings: the query after its turn and the key after its rotation to fp16 (each 2^-11,
of the vector's length: a rotation's two products share it), and the table's cosines and sines (2^-11 of the same
length); bf16 latents are met as they are.  So it is off by at most d = 3 * 2^-11 * |scale| |q| |k| (lengths), to which
own positions, whose kernels round W or the key, add 2^-11 more of it: d = 4 * 2^-11 * max |scale| |q| |k|.  Weights
are off by a factor exp(+-2 d) and two roundings to fp16 (2^-11 each, the strip factor a third), a split's mean by one:
4 * 2^-11.  With a = sum_p w_p |v_p| the latents' error is at most (exp(2 d) - 1 + 4 * 2^-11) a, the output's that
through |U_v|, plus the output's own rounding, plus fp32 sums (2^-16 of a covers those of up to 2^8 roundings)."""
import math

import pytest
import torch

import starkv
from starkv import KLatentSpec, RopeConfig, SharedPrefix, StarKVError, VLatentSpec, prefix_decode_attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ranks_of(n, lo, hi, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(lo, hi + 1, (n,), generator=g).tolist()


def fin_eps(dtype):
    return 2.0 ** -9 if dtype == torch.bfloat16 else 2.0 ** -11


class Case:
    """Latents padded to one width (garbage behind a head's rank), every tensor with strides of its own."""

    def __init__(self, B, Hq, Hkv, P, S, lo, hi, Rv, dtype, seed=0, theta=1e4, pad=0, kx=1.0, vx=1.0, qx=1.0):
        g = torch.Generator().manual_seed(seed)
        self.B, self.Hq, self.Hkv, self.P, self.S, self.Rv, self.dtype = B, Hq, Hkv, P, S, Rv, dtype
        self.ranks = ranks_of(Hkv, lo, hi, seed)
        self.rope = RopeConfig(theta=theta)
        w = max(self.ranks) + pad
        mk = lambda *s: torch.randn(*s, generator=g)
        self.pk = (mk(Hkv, P, w) * kx).to(dtype)
        self.pv = (mk(P, Rv + pad) * vx).to(dtype)[:, :Rv]
        self.bk = (mk(Hkv, w, 128) / math.sqrt(hi)).to(dtype)
        self.k = (mk(B, Hkv, max(S, 1), w) * kx).to(dtype)
        self.v = (mk(B, max(S, 1), Rv + pad) * vx).to(dtype)[..., :Rv]
        self.uv = (mk(Hkv * 128, Rv + pad) / math.sqrt(Rv)).to(dtype)[:, :Rv]
        self.q = (mk(B, Hq, 128) * 2 * qx).to(dtype)

    def spec(self, x, bk):
        n = self.Hkv
        return KLatentSpec(x, self.ranks, [h * x.stride(1) for h in range(n)], [x.stride(2)] * n, x.stride(0), bk,
                           [h * bk.stride(0) for h in range(n)], bk.stride(1))

    def prefix(self):
        bk = self.bk.to(DEV)
        return SharedPrefix(self.spec(self.pk[None].to(DEV), bk), self.dev(self.pv)[None], rope=self.rope)

    @staticmethod
    def dev(t):
        """On the GPU with the strides it has here."""
        if t.is_contiguous():
            return t.to(DEV)
        base = t._base if t._base is not None else t
        return base.to(DEV)[tuple(slice(0, n) for n in t.shape)]

    def run(self, mask=None, **kw):
        own = self.S > 0
        k = self.spec(self.k.to(DEV), self.bk.to(DEV)) if own else None
        return prefix_decode_attention(self.q.to(DEV), self.prefix(), k, self.dev(self.v) if own else None,
                                       self.dev(self.uv), mask=None if mask is None else mask.to(DEV), **kw)

    def turned(self, x, first):
        """Rotary positions first, first + 1, ... of [..., n, 128]."""
        ang = torch.arange(first, first + x.shape[-2]).double()[:, None] * self.rope.inv_freq().double()
        z = torch.complex(x[..., :64], x[..., 64:]) * torch.polar(torch.ones_like(ang), ang)
        return torch.cat((z.real, z.imag), -1)

    def oracle(self, mask=None, scale=None, shift=0):
        """(output, bound, weights [B, Hq, P + S]) in fp64; `shift` plants a mistake: own keys that many positions on."""
        B, Hq, Hkv, P, S = self.B, self.Hq, self.Hkv, self.P, self.S
        gs, scale = Hq // Hkv, 1 / math.sqrt(128) if scale is None else scale
        out, bound, weights = [], [], []
        q = self.q.double()
        u = self.uv.double().view(Hkv, 128, -1)
        fin = torch.finfo(self.dtype)
        for h in range(Hkv):
            r = self.ranks[h]
            bk = self.bk[h, :r].double()
            qh = q[:, h * gs:(h + 1) * gs]                                         # [B, gs, 128]
            keys = self.turned(self.pk[h, :, :r].double() @ bk, -P)                # the query's turn, on the keys
            l = qh @ keys.t()
            long = keys.norm(dim=-1).max()
            if S:
                own = self.turned(self.k[:, h, :S, :r].double() @ bk, shift)       # [B, S, 128]
                y = qh @ own.transpose(1, 2)
                l = torch.cat((l, y), -1)
                long = torch.maximum(long, own.norm(dim=-1).max())
            l = l * scale
            if mask is not None:
                l[..., P:] += mask.double().reshape(B, -1, S)[:, :1]
            w = torch.softmax(l, -1)
            weights.append(w)
            lat = w[..., :P] @ self.pv.double()
            a = w[..., :P] @ self.pv.double().abs()
            if S:
                lat = lat + w[..., P:] @ self.v[:, :S].double()
                a = a + w[..., P:] @ self.v[:, :S].double().abs()
            o = lat @ u[h].t()
            d = 4 * 2.0 ** -11 * abs(scale) * qh.norm(dim=-1).max() * long
            rel = torch.expm1(2 * d) + 4 * 2.0 ** -11 + 2.0 ** -16
            out.append(o)
            bound.append(rel * (a @ u[h].abs().t()) + fin.eps / 2 * o.abs() + fin.tiny * fin.eps)
        return torch.cat(out, 1), torch.cat(bound, 1), torch.cat(weights, 1)

    def second_gap(self):
        """[B, Hq]: how far the second largest prefix logit lies below the largest, relative to |q| |k|."""
        gs, out = self.Hq // self.Hkv, []
        for h in range(self.Hkv):
            keys = self.turned(self.pk[h, :, :self.ranks[h]].double() @ self.bk[h, :self.ranks[h]].double(), -self.P)
            q = self.q[:, h * gs:(h + 1) * gs].double()
            top = (q @ keys.t()).topk(2, -1).values
            out.append((top[..., 0] - top[..., 1]) / q.norm(dim=-1) / keys.norm(dim=-1).max())
        return torch.cat(out, 1)

    def check(self, got, mask=None, scale=None):
        want, bound, w = self.oracle(mask, scale)
        err = (got.double().cpu() - want).abs()
        assert torch.isfinite(got).all()
        assert (err <= bound).all(), f"largest error over bound {(err / bound).max().item():.3f}"
        # That is the worst case of 128 roundings a logit.  Independent ones add by their squares: 2^-11 |scale q| |k| /
        # sqrt(128) for the three of them, 2^-10 at the |q| = 22, |k| = 11 of these cases; with the weights' and means'
        # own (2^-11 each, over sqrt(3)) and the output's (bf16 2^-9) the 2-norm stays below 2^-8, bf16 2^-7.
        rel = err.norm() / want.norm()
        assert rel < 4 * max(fin_eps(self.dtype), 2.0 ** -10), rel
        return want


CASES = [
    # B, Hq, Hkv, P, S, lo, hi, Rv
    (1, 1, 1, 1, 0, 1, 1, 1), (1, 1, 1, 1, 1, 128, 128, 1), (2, 8, 8, 64, 0, 16, 16, 32), (2, 8, 8, 63, 1, 8, 64, 33),
    (3, 4, 2, 65, 5, 1, 17, 255), (2, 32, 8, 300, 33, 33, 127, 257), (5, 8, 8, 1000, 64, 8, 96, 512),
    (4, 32, 32, 129, 7, 8, 40, 100), (7, 10, 5, 513, 31, 20, 128, 300), (33, 4, 4, 200, 3, 16, 64, 64),
    (40, 8, 1, 257, 2, 100, 128, 96), (9, 64, 8, 191, 40, 50, 100, 130), (17, 16, 2, 2111, 0, 64, 64, 31),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", CASES, ids=str)
def test_matches_definition(shape, dtype):
    c = Case(*shape, dtype, seed=sum(shape), pad=shape[3] % 3)
    got = c.run()
    assert got.dtype == dtype and got.shape == (c.B, c.Hq, 128)
    c.check(got)


def test_mean_bound_would_catch_a_shifted_key():
    """The oracle with own keys one position on is far outside the bound of the mean error."""
    c = Case(2, 8, 8, 40, 200, 16, 64, 64, torch.float16, seed=3)
    want, _, _ = c.oracle()
    wrong, _, _ = c.oracle(shift=1)
    assert (wrong - want).norm() / want.norm() > 1 / 32


def ragged(B, S, value=-math.inf, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = torch.randint(0, S + 1, (B,), generator=g)
    n[0], n[-1] = S, 0
    return torch.where(torch.arange(S) < n[:, None], 0.0, value).to(dtype)


@pytest.mark.parametrize("value,mdtype", [(-math.inf, torch.float32), (-math.inf, torch.float16),
                                          (torch.finfo(torch.float32).min, torch.float32),
                                          (torch.finfo(torch.float16).min, torch.float16),
                                          (torch.finfo(torch.bfloat16).min, torch.bfloat16), (-1e30, torch.float32)])
def test_masks_that_leave_nothing(value, mdtype):
    for Hq, Hkv in ((8, 8), (16, 4)):
        c = Case(5, Hq, Hkv, 150, 70, 16, 64, 96, torch.float16, seed=5)
        m = ragged(5, 70, value, mdtype)
        got = c.run(m)
        want = c.check(got, m)
        # the last sequence has nothing of its own: the prefix alone
        c2 = Case(5, Hq, Hkv, 150, 0, 16, 64, 96, torch.float16, seed=5)
        c2.q, c2.pk, c2.pv, c2.bk, c2.uv = c.q, c.pk, c.pv, c.bk, c.uv
        alone, bound, _ = c2.oracle()
        assert ((got[-1].double().cpu() - alone[-1]).abs() <= bound[-1]).all()
        assert torch.allclose(want[-1], alone[-1])


def test_last_pos_and_scores():
    c = Case(3, 8, 4, 100, 50, 16, 64, 64, torch.float16, seed=8)
    pos = torch.tensor([20], dtype=torch.int32, device=DEV)
    m = torch.zeros(3, 50)
    m[:, 21:] = -math.inf
    sc = torch.full((3, 60), 2.0, device=DEV)
    got = c.run(last_pos=pos, scores=sc)
    c.check(got, m)
    _, _, w = c.oracle(m)
    want = w[..., 100:].sum(1)
    # weights off by exp(2 d) with d of the module's note, two fp16 roundings in the prefix's sum
    d = 4 * 2.0 ** -11 / math.sqrt(128) * c.q.double().norm(dim=-1).max() * 40
    err = (sc[:, :50].double().cpu() - 2 - want).abs()
    assert (err <= want * (torch.expm1(2 * d) + 2.0 ** -10) + 2.0 ** -20).all()
    assert (sc[:, 21:] == 2).all()


def test_same_bits_twice_and_poisoned_workspace():
    c = Case(6, 32, 8, 900, 33, 20, 90, 300, torch.float16, seed=11)
    a = c.run()
    assert torch.equal(a, c.run())


def test_one_sequence_equals_decode_over_the_whole():
    """A batch of one behind its prefix is decode over prefix and own positions in one cache."""
    P, S = 200, 30
    c = Case(1, 8, 8, P, S, 16, 64, 96, torch.float16, seed=13)
    got = c.run()
    x = torch.cat((c.pk[None], c.k), 2).to(DEV)
    q = starkv.rope_apply(c.q.to(DEV).unsqueeze(2).clone(), c.rope, pos0=P)[:, :, 0]
    v = torch.cat((c.pv[None], c.v), 1).to(DEV).contiguous()
    ref = starkv.decode_attention(q, c.spec(x, c.bk.to(DEV)), v, c.dev(c.uv), rope=c.rope)
    want, bound, _ = c.oracle()
    assert ((got.double().cpu() - want).abs() <= bound).all()
    assert ((ref.double().cpu() - want).abs() <= 2 * bound).all()


@pytest.mark.parametrize("kx,vx,qx", [(30000.0, 1.0, 2e-5), (1.0, 1e5, 1.0), (1.0, 1e-6, 1.0), (1e-5, 1.0, 1e5),
                                      (3e4, 3e30, 1e-4), (1e4, 1.0, 1e4)])
def test_magnitudes_bf16(kx, vx, qx):
    """Keys, values and queries outside fp16's range."""
    c = Case(3, 8, 4, 130, 0, 16, 64, 64, torch.bfloat16, seed=17, kx=kx, vx=vx, qx=qx)
    got = c.run()
    if kx * qx > 100:                                # logits near 1e8, so far apart that one weight is 1: the position's value
        want, _, w = c.oracle()
        assert torch.isfinite(got).all()
        far = w.topk(2, -1).values[..., 0] == 1
        clear = far & (c.second_gap() > 2.0 ** -7)   # four times the logits' error, 2^-9 |q| |k|
        assert clear.sum() >= 6
        assert ((got.double().cpu() - want).abs() <= 2.0 ** -6 * want.abs().amax(-1, keepdim=True))[clear].all()
        return
    c.check(got)


def test_large_values_fp16():
    c = Case(2, 4, 4, 300, 0, 16, 64, 64, torch.float16, seed=19)
    c.pv = torch.full_like(c.pv, 65504.0)
    c.uv = (c.uv * 0 + 2.0 ** -10).to(torch.float16)
    got = c.run()
    assert torch.allclose(got.double().cpu(), torch.tensor(65504.0 * 64 / 1024, dtype=torch.float64), rtol=2.0 ** -9)


def test_large_keys_fp16():
    c = Case(2, 4, 4, 300, 0, 64, 64, 64, torch.float16, seed=20, kx=10000.0, qx=2e-5)   # 20000 overflows fp16 in the inputs themselves
    c.check(c.run())


def test_far_strips_keep_their_weight():
    """One position far above all others, which together weigh more than it: weights 2^-20 of the largest count."""
    P = 32768
    c = Case(1, 1, 1, P, 0, 16, 16, 32, torch.float16, seed=23, theta=1e9)
    c.pk.zero_()
    c.q.zero_()
    c.bk.zero_()
    c.q[..., 63] = 8                                   # the slowest frequency: no turn to speak of
    c.bk[0, 0, 63] = 1
    c.pk[0, 17, 0] = 14 * math.log(2) * math.sqrt(128) / 8    # 2^14 times the others' weight
    c.pv = torch.ones_like(c.pv)
    c.pv[17] = -1
    got = c.run()
    want, bound, w = c.oracle()
    assert 0.2 < w[0, 0, 17] < 0.5
    assert ((got.double().cpu() - want).abs() <= bound).all()


def test_infinite_and_nan_latents_show():
    c = Case(2, 4, 4, 130, 0, 16, 64, 64, torch.float16, seed=29)
    c.pv[5, 3] = math.nan
    assert torch.isnan(c.run()).all()                  # through U_v's column 3
    c = Case(2, 4, 4, 130, 0, 16, 64, 64, torch.float16, seed=29)
    c.pk[1, 7, 0] = math.nan
    got = c.run()
    assert torch.isnan(got[:, 1]).all() and torch.isfinite(got[:, 0]).all() and torch.isfinite(got[:, 2:]).all()


def test_prefix_row_and_length_of_a_batch():
    """A prefix from row 2 of a batch, shorter than the cache."""
    c = Case(3, 8, 4, 90, 9, 16, 50, 70, torch.float16, seed=31)
    big_k = torch.randn(4, c.Hkv, 120, c.pk.shape[2]).half()
    big_v = torch.randn(4, 120, c.Rv).half()
    big_k[2, :, :90], big_v[2, :90] = c.pk, c.pv
    p = SharedPrefix(c.spec(big_k.to(DEV), c.bk.to(DEV)), big_v.to(DEV), 90, c.rope, row=2)
    got = prefix_decode_attention(c.q.to(DEV), p, c.spec(c.k.to(DEV), c.bk.to(DEV)), c.dev(c.v), c.dev(c.uv))
    c.check(got)


def test_outputs_and_strides():
    c = Case(3, 8, 4, 90, 9, 16, 50, 70, torch.bfloat16, seed=37)
    q = torch.zeros(3, 16, 200, dtype=torch.bfloat16, device=DEV)[:, ::2, 5:133]
    q.copy_(c.q)
    out = torch.full((3, 9, 140), 7.0, device=DEV)
    k, v, uv = c.spec(c.k.to(DEV), c.bk.to(DEV)), c.dev(c.v), c.dev(c.uv)
    got = prefix_decode_attention(q, c.prefix(), k, v, uv, out=out[:, :8, 3:131])
    assert (out[:, 8] == 7).all() and (out[:, :, :3] == 7).all() and (out[:, :, 131:] == 7).all()
    want, bound, _ = c.oracle()
    assert ((got.double().cpu() - want).abs() <= bound).all()
    f32 = prefix_decode_attention(q, c.prefix(), k, v, uv, out_dtype=torch.float32)
    assert torch.equal(f32, got)


def test_quantised_own_latents():
    """A prefix shared from a quantised cache, own latents in another one."""
    from starkv.cache import LatentCache
    ranks, Rv, P, S, B = [16, 40, 64, 24], 128, 150, 20, 3
    g = torch.Generator(device=DEV).manual_seed(2)
    mk = lambda *s: torch.randn(*s, generator=g, device=DEV).half()
    bk = (mk(4, 64, 128) / 8)
    rope = RopeConfig()
    for fmt in ("dense", "int8_g64", "reference"):
        whole = LatentCache(1, ranks, Rv, P, torch.float16, DEV, fmt)
        whole.append(mk(1, 4, P, 64), mk(1, P, Rv), bk)
        prefix = whole.share(bk, rope)
        own = LatentCache(B, ranks, Rv, 32, torch.float16, DEV, fmt)
        ks, vs, n = own.append(mk(B, 4, S, 64), mk(B, S, Rv), bk)
        q, uv = mk(B, 8, 128), mk(512, Rv) / 11
        got = prefix_decode_attention(q, prefix, ks, vs, uv, seq_len=n)
        c = Case(B, 8, 4, P, S, 64, 64, Rv, torch.float16)
        c.ranks, c.rope, c.q, c.uv, c.bk = ranks, rope, q.cpu(), uv.cpu(), bk.cpu()
        pad = lambda x: torch.nn.functional.pad(x.cpu(), (0, 64 - x.shape[-1]))
        c.pk = torch.stack([pad(x[0]) for x in whole.dequant_k()])
        c.k = torch.stack([pad(x) for x in own.dequant_k()], 1)
        c.pv, c.v = whole.dequant_v()[0].cpu(), own.dequant_v().cpu()
        c.check(got)


def test_graph_of_two_calls_replayed():
    """Two calls captured into one graph, replayed with eager work between, against the eager results."""
    a, b = Case(4, 8, 8, 300, 20, 16, 64, 96, torch.float16, seed=41), Case(2, 16, 4, 130, 0, 30, 99, 64, torch.float16, seed=42)
    pa, pb = a.prefix(), b.prefix()
    ka, va, ua, qa = a.spec(a.k.to(DEV), a.bk.to(DEV)), a.dev(a.v), a.dev(a.uv), a.q.to(DEV)
    ub, qb = b.dev(b.uv), b.q.to(DEV)
    run = lambda: (prefix_decode_attention(qa, pa, ka, va, ua), prefix_decode_attention(qb, pb, None, None, ub))
    run()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ga, gb = run()
    for step in range(4):
        qa.copy_(torch.randn(qa.shape).half())
        qb.copy_(torch.randn(qb.shape).half())
        ea, eb = run()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(ga, ea) and torch.equal(gb, eb), step


def test_on_another_stream_beside_an_eager_call():
    a = Case(4, 8, 8, 300, 20, 16, 64, 96, torch.float16, seed=43)
    pa = a.prefix()
    ka, va, ua, qa = a.spec(a.k.to(DEV), a.bk.to(DEV)), a.dev(a.v), a.dev(a.uv), a.q.to(DEV)
    want = prefix_decode_attention(qa, pa, ka, va, ua)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            one = prefix_decode_attention(qa, pa, ka, va, ua)
        two = prefix_decode_attention(qa, pa, ka, va, ua)
        torch.cuda.synchronize()
        assert torch.equal(one, want) and torch.equal(two, want)


def test_refusals():
    c = Case(2, 8, 4, 64, 8, 16, 32, 64, torch.float16, seed=47)
    p, k, v, uv, q = c.prefix(), c.spec(c.k.to(DEV), c.bk.to(DEV)), c.dev(c.v), c.dev(c.uv), c.q.to(DEV)
    bad = [
        lambda: prefix_decode_attention(q.bfloat16(), p, k, v, uv),
        lambda: prefix_decode_attention(q, p, k, None, uv),
        lambda: prefix_decode_attention(q, p, None, None, uv, seq_len=3),
        lambda: prefix_decode_attention(q, p, None, None, uv[:-1]),
        lambda: prefix_decode_attention(q, p, k, v, uv, seq_len=9),
        lambda: prefix_decode_attention(q, p, k, v, uv, seq_len=-1),
        lambda: prefix_decode_attention(q[:, :7], p, None, None, uv),
        lambda: prefix_decode_attention(q, p, k, v[..., :63], uv),
        lambda: prefix_decode_attention(q, p, k, v, uv, scores=torch.zeros(2, 7, device=DEV)),
        lambda: prefix_decode_attention(q, p, k, v, uv, scores=torch.zeros(2, 8, device=DEV).half()),
        lambda: prefix_decode_attention(q, p, None, None, uv, out=torch.empty(2, 8, 128, device=DEV).double()),
        lambda: SharedPrefix(k, v, 9),
        lambda: SharedPrefix(k, v, 8, row=2),
        lambda: SharedPrefix(k, v.bfloat16()),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(StarKVError):
            f()
            pytest.fail(f"call {i} was not refused")


@pytest.mark.parametrize("dense", [True, False])
def test_own_latents_that_are_no_numbers_show(dense):
    c = Case(3, 8, 4, 70, 5, 16, 32, 64, torch.float16, seed=51)
    c.ranks = [16] * 4
    bk = c.bk[:, :16].contiguous().to(DEV)
    if dense:
        k = c.k[..., :16].contiguous().to(DEV)
        k[1] = math.nan
        k = KLatentSpec.from_reference(k, bk)
    else:
        scale = torch.full((3, 4, 5, 1), 0.01, device=DEV).half()
        scale[1] = math.nan
        k = KLatentSpec.from_reference_quant(torch.ones(3, 4, 5, 16, dtype=torch.int8, device=DEV), scale, bk, 16)
    args = c.q.to(DEV), c.prefix(), k, c.v.to(DEV), c.uv.to(DEV)
    got = prefix_decode_attention(*args)
    assert torch.isnan(got[1]).all() and torch.isfinite(got[::2]).all()
    alone = prefix_decode_attention(args[0], args[1], None, None, args[4])
    for low in (-math.inf, torch.finfo(torch.float32).min):
        mask = torch.zeros(3, 1, 5)
        mask[1] = low
        got = prefix_decode_attention(*args, mask=mask.to(DEV))
        # nothing that is masked is looked at: the prefix alone, whose sums another split count may round anew
        # (fp32, 2^-16 as above) before the output's rounding
        want = alone[1].float()
        assert ((got[1].float() - want).abs() <= 2.0 ** -10 * want.abs() + 2.0 ** -14).all()


def test_offsets_past_32_bits():
    """Latents whose rows lie so far apart that byte offsets pass 2^32: the same bits as the same rows packed."""
    g = torch.Generator().manual_seed(3)
    P, S, wide = 700, 40, 1 << 22
    bk = torch.randn(1, 16, 128, generator=g).half().to(DEV)
    uv, q = torch.randn(128, 32, generator=g).half().to(DEV), torch.randn(2, 2, 128, generator=g).half().to(DEV)
    base = torch.empty(P, wide, dtype=torch.float16, device=DEV)                   # 5.9 GB
    pk, pv = base[:, :16], base[:, 64:96]
    own_k, own_v = [base[:2 * S, a:b].unflatten(0, (S, 2)).transpose(0, 1) for a, b in ((128, 144), (192, 224))]
    for t in (pk, pv, own_k, own_v):
        t.copy_(torch.randn(t.shape, generator=g))
    spec = lambda x: KLatentSpec(x, [16], [0], [x.stride(1)], x.stride(0), bk, [0], 128)
    run = lambda f: prefix_decode_attention(q, SharedPrefix(spec(f(pk[None])), f(pv[None])), spec(f(own_k)), f(own_v), uv)
    assert torch.equal(run(lambda t: t), run(lambda t: t.contiguous()))


def test_refuses_latents_that_end_before():
    c = Case(2, 8, 4, 64, 8, 16, 32, 64, torch.float16, seed=47)
    p, v, uv, q = c.prefix(), c.dev(c.v), c.dev(c.uv), c.q.to(DEV)
    short = c.spec(c.k[:, :, :7].contiguous().to(DEV), c.bk.to(DEV))
    one = c.spec(c.k[:1].to(DEV), c.bk.to(DEV))
    k = c.spec(c.k.to(DEV), c.bk.to(DEV))
    bad = [
        lambda: prefix_decode_attention(q, p, short, v, uv),
        lambda: prefix_decode_attention(q, p, one, v, uv),
        lambda: prefix_decode_attention(q, p, k, v, uv, out=torch.empty(1, 8, 128, device=DEV).half()),
        lambda: prefix_decode_attention(q, p, None, None, uv, out=torch.empty(2, 8, 64, device=DEV).half()),
        lambda: SharedPrefix(short, v, 8, row=1),
        lambda: SharedPrefix(one, v, 8, row=1),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(StarKVError):
            f()
            pytest.fail(f"call {i} was not refused")


@pytest.mark.parametrize("mdtype", [torch.float32, torch.float16, torch.bfloat16])
def test_padding_that_is_no_number_is_not_looked_at(mdtype):
    """Own dense K latents of NaN in masked places of rows that keep others: as if they held zeros."""
    c = Case(3, 8, 4, 130, 40, 16, 32, 64, torch.bfloat16, seed=53)
    keep = torch.tensor([40, 17, 0])
    mask = torch.zeros(3, 1, 40).masked_fill_(torch.arange(40) >= keep[:, None, None], torch.finfo(mdtype).min).to(mdtype)
    pad = (mask[:, 0] < 0)[:, None, :, None]
    c.k = c.k.masked_fill(pad, 0.0)
    want = c.run(mask)
    c.k = c.k.masked_fill(pad, math.nan)
    assert torch.equal(c.run(mask), want)
    c.k[1, :, 3] = math.nan
    got = c.run(mask)
    assert torch.isnan(got[1]).all() and torch.equal(got[::2], want[::2])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [
    # more than 32 query heads a KV head; the widest V; column slices of 128 and 64; KV heads up to 64, one query head each
    (2, 64, 1, 100, 40, 100, 128, 65), (3, 40, 1, 70, 33, 17, 33, 40), (2, 64, 1, 64, 1, 1, 7, 33), (3, 16, 4, 500, 77, 64, 128, 8192),
    (16, 32, 32, 200, 9, 8, 96, 1000), (2, 32, 32, 130, 70, 8, 96, 600), (1, 64, 64, 90, 300, 1, 128, 200)], ids=str)
def test_matches_definition_at_the_ends(shape, dtype):
    c = Case(*shape, dtype, seed=sum(shape), pad=shape[3] % 3)
    c.check(c.run())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_long_splits(dtype):
    """So many tiles of P V that a split holds all 121 strips: the strips' factors are formed anew on the way."""
    c = Case(64, 32, 1, 7700, 0, 128, 128, 8192, dtype, seed=61)
    got = c.run()
    pick = [0, 17, 63]
    c.q, c.B = c.q[pick], len(pick)                       # the definition of some sequences
    c.check(got[pick])
