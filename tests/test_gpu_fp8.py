"""GPU checks of the 8-bit floating point projections (starkv.fp8_quantize,
fp8_matmul, fp8_linear) against their definitions in 64 bits.

The quantiser is exact: its values and scales are compared bit for bit with a
restatement that rounds in 64 bits.

Products: for 16-bit outputs the matrix instruction adds each run of eight
products with 13 bits below its largest one or more, so a run is at most
7 * 2^-13 of its largest product off, hence an output at most 7 * 2^-13
sum |x||w|; fp32 outputs add k products of exact values in fp32, at most
(k + 8) 2^-24 sum |x||w| off.  Then one rounding: half a step, eps / 2 of the
result.  Over many outputs these errors are independent, and the norm of the
difference is far below those sums: measured 1.5e-5 of the result's norm for
the instruction, so 1e-4 is asked for beside the rounding's eps / 2."""
import math
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

E8, F32 = torch.float8_e8m0fnu, torch.float32
F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


def _flush(msg):
    print(msg, flush=True)
    sys.stdout.flush()


# ---------------------------------------------------------------- the definition
def _round_e4m3(v):
    """fp64 to the nearest e4m3 value (|v| <= 448 (1 + 2^-5)), ties to even; NaN stays."""
    _, e = torch.frexp(v)
    step = torch.exp2((e.double() - 4).clamp_min(-9))
    return torch.round(v / step) * step


def ref_quantize(x, scale_dtype):
    """(values fp64 [rows, k], scales fp64 [rows, ceil(k / 128)]) of the rows x."""
    rows, k = x.shape
    nb = -(-k // 128)
    p = torch.zeros(rows, nb * 128, dtype=torch.float64)
    p[:, :k] = x.double().cpu()
    p = p.view(rows, nb, 128)
    a = p.abs().amax(-1)                              # a NaN wins
    bad = ~torch.isfinite(a)
    af = torch.where(bad, 1.0, a)
    if scale_dtype == E8:
        # least e with a <= 448 2^e
        e = torch.ceil(torch.log2(torch.where(af > 0, af, 448.0) / 448.0)).clamp(-126, 127)
        e = torch.where(af > 448.0 * torch.exp2(e), e + 1, e)
        e = torch.where(af <= 448.0 * torch.exp2((e - 1)), (e - 1).clamp_min(-126), e)
        s = torch.where(af > 0, torch.exp2(e), 1.0)
        q = p / s[..., None]
    else:
        a1 = af.clamp_min(2.0 ** -100)
        s = torch.where(af > 0, (a1 / 448.0).float().double(), 1.0)
        q = (p * (448.0 / a1).float().double()[..., None]).float().double()
    nan = torch.full_like(s, math.nan)
    s = torch.where(bad, nan, s)
    q = torch.where(bad[..., None], torch.full_like(q, math.nan), _round_e4m3(q))
    return q.reshape(rows, -1)[:, :k], s


def _deq(q, s):
    k = q.shape[1]
    return q * s.repeat_interleave(128, 1)[:, :k]


def ref_weight(w, ws):
    n = w.shape[0]
    return _deq(w.double().cpu(), ws.double().cpu().repeat_interleave(128, 0)[:n])


def _eq(a, b):
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


# ---------------------------------------------------------------- quantiser
@pytest.mark.parametrize("scale", [E8, F32], ids=["e8m0", "f32"])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 16), (3, 127), (5, 128), (17, 129), (33, 1640), (2, 16387), (700, 264)])
def test_quantize_is_exact(rows, k, dtype, scale):
    from starkv import fp8_quantize
    _flush(f"[quantize] {rows}x{k} {dtype} {scale}")
    g = torch.Generator(device="cuda").manual_seed(rows + k)
    x = torch.randn(rows, k, generator=g, device="cuda") * torch.exp2(torch.randint(-12, 8, (rows, 1), generator=g, device="cuda").float())
    x = x.to(dtype)
    q, s = fp8_quantize(x, scale)
    torch.cuda.synchronize()
    assert q.dtype == E4M3 and s.dtype == scale and q.shape == x.shape and s.shape == (rows, -(-k // 128))
    rq, rs = ref_quantize(x, scale)
    assert _eq(s.double().cpu(), rs)
    assert _eq(q.double().cpu(), rq)
    # the padding up to whole 16-byte pieces is zero
    whole = q.as_strided((rows, -(-k // 16) * 16), (q.stride(0), 1)).view(torch.uint8)
    assert int(whole[:, k:].sum()) == 0


@pytest.mark.parametrize("scale", [E8, F32], ids=["e8m0", "f32"])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
def test_quantize_borders(dtype, scale):
    """Zero blocks, block maxima at and next to 448 2^e, subnormal and largest values, NaN and infinity."""
    from starkv import fp8_quantize
    fi = torch.finfo(dtype)
    x = torch.zeros(12, 256, dtype=torch.float64)
    g = torch.Generator().manual_seed(3)
    noise = torch.rand(12, 256, generator=g, dtype=torch.float64) * 2 - 1
    tops = [0.0, 448.0, 449.0 if dtype == F16 else 450.0, 447.5, 224.0, 1.0, 2.0 ** -14, float(fi.smallest_normal) / 8,
            float(fi.max), 1.75, 1.7509765625, 3.0]
    for i, t in enumerate(tops):
        x[i, :128] = noise[i, :128] * t
        x[i, 5] = -t
        x[i, 128:] = noise[i, 128:]
    x = x.to(dtype).cuda()
    x[10, 200] = math.inf
    x[11, 130] = math.nan
    q, s = fp8_quantize(x, scale)
    rq, rs = ref_quantize(x, scale)
    assert _eq(s.double().cpu(), rs) and _eq(q.double().cpu(), rq)
    assert s[0, 0].double() == 1.0 and torch.isnan(s[10, 1].float()) and not torch.isnan(s[10, 0].float())


def test_quantize_layouts():
    """Rows at odd element offsets and strides, leading dims, no rows."""
    from starkv import fp8_quantize
    g = torch.Generator(device="cuda").manual_seed(5)
    wide = torch.randn(2, 7, 700, generator=g, device="cuda").half()
    for x in (wide[..., 1:302], wide[..., :264], wide[:, :, 8:8 + 129], wide[0, 0, 3:]):
        q, s = fp8_quantize(x)
        rq, rs = ref_quantize(x.reshape(-1, x.shape[-1]), E8)
        assert q.shape == x.shape and s.shape == (*x.shape[:-1], -(-x.shape[-1] // 128))
        assert _eq(q.double().cpu().reshape(rq.shape), rq) and _eq(s.double().cpu().reshape(rs.shape), rs)
    q, s = fp8_quantize(wide[:0])
    assert q.shape == (0, 7, 700) and s.shape == (0, 7, 6)


@pytest.mark.parametrize("scale", [E8, F32], ids=["e8m0", "f32"])
def test_quantize_weight_on_device_and_host_agree(scale):
    from starkv import fp8_quantize_weight
    g = torch.Generator().manual_seed(6)
    w, nw = torch.randn(300, 200, generator=g).half(), 1 + 0.2 * torch.randn(200, generator=g).half()
    q, s = fp8_quantize_weight(w, scale, norm_weight=nw)
    qd, sd = fp8_quantize_weight(w.cuda(), scale, norm_weight=nw.cuda())
    assert torch.equal(q.view(torch.uint8), qd.view(torch.uint8).cpu()) and torch.equal(s.float(), sd.float().cpu())


# ---------------------------------------------------------------- products
def _rows8(g, rows, k, pad=0x7F):
    """e4m3 rows whose bytes behind column k are NaN."""
    t = torch.full((rows, -(-k // 16) * 16 + 16), pad, dtype=torch.uint8, device="cuda").view(E4M3)
    v = (torch.randn(rows, k, generator=g, device="cuda") * 100).clamp(-448, 448)
    t[:, :k] = v.to(E4M3)
    return t[:, :k]


def _scales(g, shape, kind, e):
    if kind == F32:
        return torch.exp2(torch.rand(*shape, generator=g, device="cuda") * 2 + e)
    return torch.exp2(torch.randint(e, e + 3, shape, generator=g, device="cuda").float()).to(E8)


def make(m, n, k, dtype, out, scale, epilogue, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + m * 31 + n * 7 + k)
    c = dict(m=m, n=n, k=k, out=out, scale=scale, epilogue=epilogue, dtype=dtype)
    if dtype == E4M3:
        c["x"], c["xs"] = _rows8(g, m, k), _scales(g, (m, -(-k // 128)), scale, -8)
    else:
        c["x"] = torch.randn(m, k, generator=g, device="cuda").to(dtype)
        if k > 20:
            c["x"][:, 17] *= 20
    c["w"], c["ws"] = _rows8(g, n, k), _scales(g, (-(-n // 128), -(-k // 128)), scale, -8 - int(math.log2(k) / 2))
    c["res"] = torch.randn(m, n, generator=g, device="cuda").to(out) if epilogue == "residual" else None
    return c


def call(c, **kw):
    from starkv import fp8_linear, fp8_matmul
    kw = dict(residual=c["res"], silu_mul=c["epilogue"] == "silu_mul", out_dtype=c["out"]) | kw
    if c["dtype"] == E4M3:
        return fp8_matmul(c["x"], c["xs"], c["w"], c["ws"], **kw)
    return fp8_linear(c["x"], c["w"], c["ws"], **kw)


def reference(c, rms_eps=None):
    """(result fp64, the bound of its error before the last rounding)."""
    xd = _deq(c["x"].double().cpu(), c["xs"].double().cpu()) if c["dtype"] == E4M3 else _deq(*ref_quantize(c["x"], c["scale"]))
    wd = ref_weight(c["w"], c["ws"])
    y, mag = xd @ wd.t(), xd.abs() @ wd.abs().t()
    bound = mag * ((c["k"] + 8) * 2.0 ** -24 if c["out"] == F32 else 7 * 2.0 ** -13)
    if rms_eps is not None:
        x = c["x"].double().cpu()
        r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + rms_eps)
        # the row factor: a mean of k squares in fp32 and a reciprocal root, of a few units each
        y, bound = y * r, bound * r + (y * r).abs() * (c["k"] / 64 + 8) * 2.0 ** -24
    if c["res"] is not None:
        y = y + c["res"].double().cpu()
        bound = bound + y.abs() * 2.0 ** -24
    if c["epilogue"] == "silu_mul":
        h = c["n"] // 2
        gt, up, bg, bu = y[:, :h], y[:, h:], bound[:, :h], bound[:, h:]
        sg = torch.sigmoid(gt)
        y = gt * sg * up
        # |d silu| <= 1.1; exp, the quotient and the products: a few units of fp32 and exp2's argument
        bound = 1.1 * bg * up.abs() + (gt * sg).abs() * bu + 1.1 * bg * bu + y.abs() * (8 + gt.abs()) * 2.0 ** -23
    return y, bound


def check(out, c, rms_eps=None):
    ref, bound = reference(c, rms_eps)
    o = out.double().cpu()
    half = torch.finfo(c["out"]).eps / 2
    lim = bound * (1 + half) + half * ref.abs() + torch.finfo(c["out"]).tiny * half
    err = (o - ref).abs()
    assert torch.isfinite(o).all()
    worst = float((err / lim.clamp_min(1e-300)).max())
    rel = float(err.norm() / ref.norm().clamp_min(1e-300))
    _flush(f"   worst error / bound = {worst:.3f}, norm {rel:.2e}")
    assert worst <= 1.0
    assert rel <= half + (1e-4 if c["out"] != F32 else 2e-6)


CASES = []
for _i, (_m, _n, _k) in enumerate([
        (1, 1, 1), (1, 16, 16), (2, 17, 130), (7, 100, 127), (15, 512, 1640), (16, 200, 2049), (1, 4096, 4096),
        (17, 1, 1), (17, 130, 100), (31, 512, 128), (33, 257, 129), (64, 128, 1000), (65, 384, 1640), (100, 4096, 256),
        (129, 131, 2000), (200, 1000, 384), (257, 512, 640), (515, 300, 1023)]):
    for _s in (E8, F32):
        _d = (F16, BF16, E4M3)[(_i + (_s == F32)) % 3]
        _o = (F16, BF16, F32)[(_i // 2 + (_s == F32)) % 3]
        CASES.append((_m, _n, _k, _d, _o, _s, ("none", "residual")[_i % 2]))
for _i, (_m, _n, _k) in enumerate([(1, 256, 128), (8, 512, 300), (16, 1024, 2048), (20, 256, 130), (70, 768, 1640), (300, 512, 500)]):
    for _s in (E8, F32):
        CASES.append((_m, _n, _k, (F16, BF16, E4M3)[(_i + (_s == F32)) % 3], (BF16, F16, F32)[(_i + (_s == F32)) % 3], _s, "silu_mul"))


def _id(c):
    return "m%dn%dk%d-%s-%s-%s-%s" % (*c[:3], *(str(t).replace("torch.", "") for t in c[3:6]), c[6])


@pytest.mark.parametrize("case", CASES, ids=_id)
def test_product(case):
    _flush(f"[product] {_id(case)}")
    c = make(*case)
    out = call(c)
    torch.cuda.synchronize()
    check(out, c)
    again = call(c)
    assert torch.equal(out, again)                   # the same bits


@pytest.mark.parametrize("scale", [E8, F32], ids=["e8m0", "f32"])
@pytest.mark.parametrize("m,n,k", [(1, 300, 1000), (16, 256, 4096), (40, 256, 1640), (300, 512, 777)])
def test_product_with_rms(m, n, k, scale):
    _flush(f"[rms] {m} {n} {k} {scale}")
    for epilogue, out in (("none", F16), ("silu_mul" if n % 256 == 0 else "residual", F32)):
        c = make(m, n, k, F16, out, scale, epilogue)
        check(call(c, rms_eps=1e-5), c, rms_eps=1e-5)


def test_large_tiles():
    """Enough tiles for the largest workgroup tile, ragged at every edge: checked on rows and columns at the edges."""
    for scale, epi in ((E8, "none"), (F32, "silu_mul"), (E8, "silu_mul"), (F32, "residual")):
        m, n, k = 4100, 4352 if epi == "silu_mul" else 4300, 400
        c = make(m, n, k, BF16, BF16, scale, epi)
        out = call(c)
        rows = torch.tensor([0, 1, 63, 64, 255, 256, 2047, 2048, 4094, 4095, 4096, 4099])
        sub = dict(c, m=len(rows), x=c["x"][rows.cuda()], res=None if c["res"] is None else c["res"][rows.cuda()])
        check(out[rows.cuda()], sub)
        assert torch.isfinite(out.float()).all()


@pytest.mark.parametrize("scale,out,epilogue", [(E8, BF16, "none"), (F32, BF16, "residual"), (F32, F32, "none"),
                                                (E8, F16, "silu_mul"), (F32, F16, "silu_mul")])
def test_long_products_of_some_rows(scale, out, epilogue):
    """A tile for nearly every compute unit and many blocks (eight waves to a workgroup), ragged at every edge:
    checked on rows at the tiles' edges, every column."""
    m, n, k = 2000, 4096 if epilogue == "silu_mul" else 4092, 5000
    _flush(f"[long] {scale} {out} {epilogue}")
    c = make(m, n, k, BF16, out, scale, epilogue)
    got = call(c)
    assert torch.isfinite(got.float()).all()
    rows = torch.tensor([0, 1, 31, 32, 127, 128, 1023, 1024, 1919, 1920, 1998, 1999])
    sub = dict(c, m=len(rows), x=c["x"][rows.cuda()], res=None if c["res"] is None else c["res"][rows.cuda()])
    check(got[rows.cuda()], sub)
    assert torch.equal(got, call(c))


@pytest.mark.parametrize("epilogue,rms", [("none", None), ("none", 1e-5), ("residual", None), ("residual", 1e-5),
                                          ("silu_mul", None), ("silu_mul", 1e-5)])
@pytest.mark.parametrize("m,n,k", [(8192, 4608, 128), (4300, 8448, 264), (6000, 5888, 1000)])
def test_every_tile_of_a_workgroup(m, n, k, epilogue, rms):
    """Workgroups that take two and three tiles, whole and ragged ones: every result against the fp32 output of the
    same product (another kernel, checked above on its own), odd rows into a wider buffer whose rest stays."""
    _flush(f"[tiles] {m} {n} {k} {epilogue} {rms}")
    n -= 0 if epilogue == "silu_mul" else m % 8          # (ragged columns, too, where m is)
    c = make(m, n, k, BF16, BF16, E8, epilogue)
    kw = {} if rms is None else dict(rms_eps=rms)
    wide = n // 2 if epilogue == "silu_mul" else n
    buf = torch.full((m + 1, wide + 8), 7.0, dtype=BF16, device="cuda")
    out = buf[:m, :wide]
    if c["res"] is not None:
        out.copy_(c["res"])
        c["res"] = out                                    # in place
    want = call(c | dict(res=None if c["res"] is None else c["res"].float()), out_dtype=F32, **kw).double()
    got = call(c, out=out, out_dtype=None, **kw)
    assert got.data_ptr() == out.data_ptr()
    torch.cuda.synchronize()
    assert bool((buf[m] == 7.0).all()) and bool((buf[:, wide:] == 7.0).all())
    # the instruction's 7 * 2^-13 of sum |x||w| (test_product's bound), by a product of magnitudes in fp32
    from starkv import fp8_quantize
    q, s = fp8_quantize(c["x"], E8)
    xa = (q.float() * s.float().repeat_interleave(128, 1)[:, :k]).abs()
    wa = (c["w"].float() * c["ws"].float().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]).abs()
    mag = (xa @ wa.t().contiguous()).double()
    if rms is not None:
        mag = mag / torch.sqrt(c["x"].double().square().mean(-1, keepdim=True) + rms)
    bound = mag * (7 * 2.0 ** -13 + 2.0 ** -20)
    if epilogue == "silu_mul":
        # d(silu(g) u): |silu'| <= 1.1 and |silu(g)| <= |g| <= mag
        bg, bu = bound[:, :wide], bound[:, wide:]
        bound = 1.1 * bg * mag[:, wide:] + mag[:, :wide] * bu + 1.1 * bg * bu
    lim = bound + (want.abs() + bound) * torch.finfo(BF16).eps / 2
    worst = float(((out.double() - want).abs() / lim.clamp_min(1e-30)).max())
    _flush(f"   worst error / bound = {worst:.3f}")
    assert worst <= 1.0


@pytest.mark.parametrize("m,n,k,scale,epilogue", [(4300, 8443, 264, E8, "residual"), (2000, 4091, 5000, E8, "none"),
                                                 (2000, 4091, 5000, F32, "residual"), (700, 4093, 1000, F32, "residual"),
                                                 (4300, 8448, 264, E8, "silu_mul"), (300, 1025, 640, F32, "residual")])
@pytest.mark.parametrize("out", [F16, F32], ids=["f16", "f32"])
def test_odd_rows_of_large_tiles(m, n, k, scale, epilogue, out):
    """Results, and the residual in place, whose rows start at every alignment of their elements: the same bits as
    into rows that are aligned, and nothing beside them."""
    c = make(m, n, k, F16, out, scale, epilogue)
    want = call(c)
    wide = want.shape[1]
    buf = torch.full((m + 2, wide + 3 + wide % 2), 7.0, dtype=out, device="cuda")     # an odd pitch
    to = buf[1:m + 1, 1:wide + 1]
    if c["res"] is not None:
        to.copy_(c["res"])
        c["res"] = to
    got = call(c, out=to, out_dtype=None)
    assert got.data_ptr() == to.data_ptr() and torch.equal(got, want)
    to.fill_(7.0)
    assert bool((buf == 7.0).all())


@pytest.mark.parametrize("m", [5, 40])
def test_layouts_and_in_place(m):
    """Activations at odd offsets, a padded output whose other columns and rows stay, the residual in place, leading dims."""
    from starkv import fp8_linear
    g = torch.Generator(device="cuda").manual_seed(m)
    c = make(m, 150, 333, F16, F16, E8, "residual")
    wide = torch.randn(m, 400, generator=g, device="cuda").half()
    c["x"] = wide[:, 5:338]
    buf = torch.full((m + 3, 171), 7.0, dtype=F16, device="cuda")
    out = buf[1:m + 1, 9:159]
    out.copy_(c["res"])
    got = fp8_linear(c["x"], c["w"], c["ws"], residual=out, out=out)
    assert got.data_ptr() == out.data_ptr()
    check(out, c)
    keep = torch.ones_like(buf, dtype=torch.bool)
    keep[1:m + 1, 9:159] = False
    assert bool((buf[keep] == 7.0).all())
    x3 = c["x"].reshape(m, 1, 333)
    assert torch.equal(fp8_linear(x3, c["w"], c["ws"], residual=c["res"].view(m, 1, 150)), out.reshape(m, 1, 150))
    assert fp8_linear(c["x"][:0], c["w"], c["ws"]).shape == (0, 150)
    assert fp8_linear(c["x"][0], c["w"], c["ws"]).shape == (150,)


@pytest.mark.parametrize("scale", [E8, F32], ids=["e8m0", "f32"])
@pytest.mark.parametrize("m", [4, 50])
def test_a_nan_stays_in_its_row(m, scale):
    from starkv import fp8_linear, fp8_matmul, fp8_quantize
    c = make(m, 200, 300, BF16, BF16, scale, "none")
    clean = call(c)
    c["x"][m - 2, 140] = math.nan
    c["x"][1, 299] = math.inf
    out = call(c)
    rows = torch.arange(m, device="cuda")
    bad = (rows == 1) | (rows == m - 2)
    assert bool(out[bad].isnan().all()) and torch.equal(out[~bad], clean[~bad])
    q, s = fp8_quantize(c["x"], scale)
    two = fp8_matmul(q, s, c["w"], c["ws"])
    assert bool(two[bad].isnan().all())


@pytest.mark.parametrize("m", [3, 16, 17, 200])
@pytest.mark.parametrize("scale", [E8, F32], ids=["e8m0", "f32"])
def test_linear_is_quantize_then_matmul(m, scale):
    """fp8_linear quantises exactly as fp8_quantize does: the same bits."""
    from starkv import fp8_linear, fp8_matmul, fp8_quantize
    c = make(m, 260, 1000, F16, F16, scale, "none")
    q, s = fp8_quantize(c["x"], scale)
    assert torch.equal(fp8_linear(c["x"], c["w"], c["ws"]), fp8_matmul(q, s, c["w"], c["ws"], out_dtype=F16))


def test_offsets_past_32_bits():
    """Activations, weights and results of more than 2^31 elements: the rows and columns at their ends."""
    from starkv import fp8_linear, fp8_matmul, fp8_quantize
    g = torch.Generator(device="cuda").manual_seed(9)
    # quantiser: 2^20 + 3 rows of 4096
    m, k = (1 << 20) + 3, 4096
    x = torch.zeros(m, k, dtype=F16, device="cuda")
    rows = torch.tensor([0, (1 << 19) - 1, 1 << 19, m - 2, m - 1])
    x[rows.cuda()] = torch.randn(len(rows), k, generator=g, device="cuda").half()
    q, s = fp8_quantize(x)
    rq, rs = ref_quantize(x[rows.cuda()], E8)
    assert _eq(q[rows.cuda()].double().cpu(), rq) and _eq(s[rows.cuda()].double().cpu(), rs)
    del x, q, s
    # weight: 4.3 GB, by the stream (m 3) and by tiles (m 40)
    n = (1 << 20) + 130
    w = torch.zeros(n, 4096, dtype=torch.uint8, device="cuda").view(E4M3)
    ws = torch.ones(-(-n // 128), 32, device="cuda").to(E8)
    n0 = (n - 300) // 128 * 128
    w[n0:] = (torch.randn(n - n0, 4096, generator=g, device="cuda") * 20).to(E4M3)
    for m in (3, 40):
        x = torch.randn(m, 4096, generator=g, device="cuda").half()
        out = fp8_linear(x, w, ws)
        assert int(out[:, :n0].count_nonzero()) == 0
        check(out[:, n0:], dict(m=m, n=n - n0, k=4096, x=x, w=w[n0:], ws=ws[n0 // 128:], dtype=F16, out=F16, scale=E8,
                                res=None, epilogue="none"))
    del w, ws, out
    # results: 70001 x 32768
    m, n, k = 70001, 32768, 128
    c = make(m, n, k, BF16, BF16, E8, "none")
    out = call(c)
    rows = torch.tensor([0, 32767, 32768, 65535, 65536, 69999, 70000])
    check(out[rows.cuda()], dict(c, m=len(rows), x=c["x"][rows.cuda()]))


def test_streams_and_graphs():
    """On another stream, and captured once and replayed with new inputs beside eager calls of other sizes."""
    from starkv import fp8_linear, fp8_quantize
    cs = [make(m, 512, 700, F16, F16, sc, "none") for m, sc in ((9, E8), (300, F32), (40, E8))]
    want = [call(c) for c in cs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [call(c) for c in cs]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for c in cs:
        x = c["x"].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = fp8_linear(x, c["w"], c["ws"])
            q, s = fp8_quantize(x, c["scale"])
        for i in range(4):
            x.copy_(c["x"] * (0.5 + i))
            graph.replay()
            eager = fp8_linear(c["x"] * (0.5 + i), c["w"], c["ws"])
            other = call(cs[(i + 1) % 3])            # eager work between the replays
            torch.cuda.synchronize()
            assert torch.equal(y, eager) and torch.equal(other, want[(i + 1) % 3])
            eq, es = fp8_quantize(c["x"] * (0.5 + i), c["scale"])
            assert torch.equal(q.view(torch.uint8), eq.view(torch.uint8)) and torch.equal(s.float(), es.float())


def test_refusals():
    from starkv import StarKVError, fp8_linear, fp8_matmul, fp8_quantize
    c = make(4, 256, 320, F16, F16, E8, "none")
    x, w, ws = c["x"], c["w"], c["ws"]
    q, s = fp8_quantize(x)
    bad = [
        lambda: fp8_quantize(x.float()), lambda: fp8_quantize(x, torch.float16), lambda: fp8_quantize(x.t()),
        lambda: fp8_linear(x.float(), w, ws), lambda: fp8_linear(x[:, :300], w, ws), lambda: fp8_linear(x, w.float(), ws),
        lambda: fp8_linear(x, w, ws[:1]), lambda: fp8_linear(x, w, ws.float().half()), lambda: fp8_linear(x, w, ws.cpu()),
        lambda: fp8_linear(x, w.view(torch.uint8)[:, :319].contiguous().view(E4M3), ws),            # rows 319 bytes apart
        lambda: fp8_linear(x, w.view(torch.uint8)[:, 1:].view(E4M3), ws),
        lambda: fp8_linear(x, w[:128], ws[:1], silu_mul=True),
        lambda: fp8_linear(x, w, ws, silu_mul=True, residual=torch.zeros(4, 128, device="cuda").half()),
        lambda: fp8_linear(x, w, ws, residual=torch.zeros(4, 256, device="cuda")),
        lambda: fp8_linear(x, w, ws, out=torch.zeros(4, 255, device="cuda").half()),
        lambda: fp8_linear(x, w, ws, out_dtype=torch.float64), lambda: fp8_linear(x, w, ws, rms_eps=-1.0),
        lambda: fp8_matmul(x, s, w, ws), lambda: fp8_matmul(q, s.float(), w, ws), lambda: fp8_matmul(q, s[:, :2], w, ws),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(StarKVError):
            f()
            _flush(f"   call {i} was not refused")
