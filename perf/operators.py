"""The operators of a model in 8-bit floating point, and of its answers, as cases that can be timed and checked.

* quantize: activations to e4m3 with one scale for each row's block of 128 columns;
* linear: a projection of activations by an e4m3 weight that has one scale for each block of 128 x 128 (the
  activations are quantised on the way), with what a decoder layer fuses to it;
* matmul: the same product of activations that are quantised already;
* logprobs: the log probability of a given token in each row of logits, the row's entropy and its top alternatives.

``run`` computes them in plain fp32 torch, or with ``own`` by the library's calls; ``exact`` restates them in fp64.
"""
import math
import os
import sys

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
F32_AMAX_FLOOR = 2.0 ** -100          # least block maximum of fp32 scales
_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32, "e8m0": torch.float8_e8m0fnu}


def listed():
    return [
        # a prompt's activations of the 4096-wide model, batch times length 8192
        dict(name="quantize_prompt", op="quantize", rows=8192, k=4096, dtype="bf16", scale="e8m0"),
        # a ragged chunk of value latents: the width is no whole number of blocks
        dict(name="quantize_ragged", op="quantize", rows=777, k=1640, dtype="f16", scale="f32"),
        # the smallest call: one token's merged query and latent projections, the layer's norm folded in
        dict(name="linear_token_qkv", op="linear", m=1, n=7376, k=4096, dtype="f16", out="f16", scale="e8m0", rms=True,
             epilogue="none"),
        # a decode step of batch 8: the merged gate and up projections with SiLU(gate) * up
        dict(name="linear_decode8_mlp", op="linear", m=8, n=22016, k=4096, dtype="f16", out="f16", scale="e8m0", rms=True,
             epilogue="silu_mul"),
        # a decode step of batch 16: the down projection onto the residual stream, a checkpoint's fp32 scales
        dict(name="linear_decode16_down", op="linear", m=16, n=4096, k=11008, dtype="bf16", out="bf16", scale="f32",
             rms=False, epilogue="residual"),
        # a ragged chunk through the value up-projection (the latent's 1640 columns)
        dict(name="linear_chunk_latent", op="linear", m=333, n=4096, k=1640, dtype="bf16", out="bf16", scale="f32",
             rms=False, epilogue="none"),
        # a hundred rows that several projections share, quantised once
        dict(name="matmul_shared_rows", op="matmul", m=100, n=4096, k=4096, dtype="bf16", out="bf16", scale="e8m0",
             rms=False, epilogue="none"),
        # the largest: the gate and up projections of an 8192-token prompt
        dict(name="linear_prompt_mlp", op="linear", m=8192, n=22016, k=4096, dtype="f16", out="f16", scale="e8m0", rms=True,
             epilogue="silu_mul"),
        # a 2048-token prompt's down projection, a checkpoint's fp32 scales
        dict(name="linear_prompt_down", op="linear", m=2048, n=4096, k=11008, dtype="bf16", out="bf16", scale="f32",
             rms=False, epilogue="residual"),
        # a decode step of batch 8 that reports its tokens' probabilities
        dict(name="logprobs_decode8", op="logprobs", rows=8, vocab=32000, dtype="f16", top=5, masked=0.0),
        # scoring a text: half of an 8192-token prompt's logits
        dict(name="logprobs_score", op="logprobs", rows=4096, vocab=32000, dtype="bf16", top=8, masked=0.0),
        # one user, a large vocabulary in fp32, most of it barred by a grammar
        dict(name="logprobs_constrained", op="logprobs", rows=1, vocab=131072, dtype="f32", top=20, masked=0.9),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "linear", "linear", "matmul", "logprobs", "logprobs"])
    if op == "quantize":
        c = dict(op=op, rows=_log(rng, 1, 16384), k=_log(rng, 64, 16384), dtype=rng.choice(["f16", "bf16"]),
                 scale=rng.choice(["e8m0", "f32"]))
        c["rows"] = max(1, min(c["rows"], 8192 * 4096 // c["k"]))
        return c
    if op == "logprobs":
        c = dict(op=op, rows=_log(rng, 1, 4096), vocab=_log(rng, 1000, 262144), dtype=rng.choice(["f16", "bf16", "f32"]),
                 top=rng.choice([0, 1, 5, rng.randint(2, 32)]), masked=rng.choice([0.0, 0.0, 0.5, 0.95]))
        c["rows"] = max(1, min(c["rows"], 4096 * 32000 // c["vocab"] // (2 if c["dtype"] == "f32" else 1)))
        return c
    m = rng.choice([rng.randint(1, 16), _log(rng, 1, 8192)])
    k = rng.choice([_log(rng, 64, 11008), 128 * rng.randint(4, 86)])
    epilogue = rng.choice(["none", "none", "residual", "silu_mul"])
    n = 256 * rng.randint(1, 86) if epilogue == "silu_mul" else rng.choice([_log(rng, 64, 16384), 128 * rng.randint(4, 128)])
    dtype = rng.choice(["f16", "bf16"])
    return dict(op=op, m=m, n=n, k=k, dtype=dtype, out=rng.choice([dtype, dtype, dtype, "f32"]),
                scale=rng.choice(["e8m0", "f32"]), rms=op == "linear" and rng.random() < 0.4, epilogue=epilogue)


# ---------------------------------------------------------------- inputs (from the seed alone)
def _ceil(a, b):
    return -(-a // b)


def _activations(g, rows, k, dtype):
    """N(0, 1) with one channel in a hundred ten times as large."""
    wide = torch.where(torch.rand(k, generator=g, device="cuda") < 0.01, 10.0, 1.0)
    return (torch.randn(rows, k, generator=g, device="cuda") * wide).to(dtype)


def _scales(g, shape, kind, typical):
    """Scales around `typical`, an octave to either side."""
    if kind == "f32":
        return typical * 2.0 ** (2 * torch.rand(*shape, generator=g, device="cuda") - 1)
    e = round(math.log2(typical)) + 127
    return torch.randint(e - 1, e + 2, shape, generator=g, device="cuda").to(torch.uint8).view(torch.float8_e8m0fnu)


def _rows8(g, rows, k):
    """e4m3 rows as a checkpoint's quantiser leaves them (largest values near 448), whole 16-byte pieces apart."""
    t = torch.empty(rows, 16 * _ceil(k, 16), dtype=torch.float8_e4m3fn, device="cuda")[:, :k]
    t.copy_((torch.randn(rows, k, generator=g, device="cuda") * 110).clamp(-E4M3_MAX, E4M3_MAX))
    return t


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = case
    if c["op"] == "quantize":
        return dict(case=c, x=_activations(g, c["rows"], c["k"], _TYPES[c["dtype"]]))
    if c["op"] == "logprobs":
        rows, v = c["rows"], c["vocab"]
        x = torch.randn(rows, v, generator=g, device="cuda") * 2.5
        if c["masked"]:
            x.masked_fill_(torch.rand(rows, v, generator=g, device="cuda") < c["masked"], -math.inf)
        x = x.to(_TYPES[c["dtype"]])
        # the token that was taken: mostly one of the likely ones (a draw by Gumbel noise), as a text's tokens are
        noise = -torch.log(-torch.log(torch.rand(rows, v, generator=g, device="cuda").clamp(1e-20, 1 - 1e-7)))
        return dict(case=c, logits=x, tokens=(x.float() + noise).argmax(-1))
    m, n, k = c["m"], c["n"], c["k"]
    s = dict(case=c)
    if c["op"] == "linear":
        s["x"] = _activations(g, m, k, _TYPES[c["dtype"]])
    else:
        s["x"] = _rows8(g, m, k)
        s["x_scale"] = _scales(g, (m, _ceil(k, BLOCK)), c["scale"], 2.0 ** -7)
    s["w"] = _rows8(g, n, k)
    s["w_scale"] = _scales(g, (_ceil(n, BLOCK), _ceil(k, BLOCK)), c["scale"], 2.0 ** round(-7 - 0.5 * math.log2(k)))
    if c["epilogue"] == "residual":
        s["residual"] = torch.randn(m, n, generator=g, device="cuda").to(_TYPES[c["out"]])
    return s


# ---------------------------------------------------------------- the plain form
def _blocks(t):
    """[..., k] as [..., blocks, 128], zeros behind the last column."""
    pad = -t.shape[-1] % BLOCK
    return torch.nn.functional.pad(t, (0, pad)).unflatten(-1, (-1, BLOCK))


def _quantize(x, kind):
    """(e4m3 values, scales) of fp32 rows."""
    b = _blocks(x)
    a = b.abs().amax(-1)
    if kind == "e8m0":
        mant, e = torch.frexp(a)
        e = torch.where(a > 0, (e - 9 + (mant > 0.875).int()).clamp_min(-126), 0)
        q = b * ((127 - e).int() << 23).view(torch.float32).unsqueeze(-1)
        scale = (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)
    else:
        a1 = a.clamp_min(F32_AMAX_FLOOR)
        most = torch.full_like(a1, E4M3_MAX)          # a tensor: torch divides by a number through its reciprocal
        q = b * (most / a1).unsqueeze(-1)
        scale = torch.where(a > 0, a1 / most, 1.0)
    return q.to(torch.float8_e4m3fn).flatten(-2)[..., :x.shape[-1]], scale


def _values(q, scale):
    """The fp32 values that e4m3 rows with a scale for each block of 128 columns stand for."""
    return (_blocks(q.float()) * scale.float().unsqueeze(-1)).flatten(-2)[..., :q.shape[-1]]


def _silu(g):
    return g / (1 + torch.exp(-g))


def _plain(s):
    c = s["case"]
    if c["op"] == "quantize":
        return _quantize(s["x"].float(), c["scale"])
    if c["op"] == "logprobs":
        x = s["logits"].float()
        d = x - x.amax(-1, keepdim=True)
        lp = d - torch.log(torch.exp(d).sum(-1, keepdim=True))
        p = torch.exp(lp)
        entropy = -torch.where(p > 0, p * lp, 0.0).sum(-1)
        ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :c["top"]]
        return lp.gather(-1, s["tokens"].unsqueeze(-1)).squeeze(-1), entropy, lp.gather(-1, ids), ids
    if c["op"] == "linear":
        x = s["x"].float()
        q, sx = _quantize(x, c["scale"])
    else:
        q, sx = s["x"], s["x_scale"]
    w = _values(s["w"], s["w_scale"].float().repeat_interleave(BLOCK, 0)[:c["n"]])
    y = _values(q, sx) @ w.t()
    if c["rms"]:
        y = y * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5)
    if c["epilogue"] == "residual":
        y = y + s["residual"].float()
    elif c["epilogue"] == "silu_mul":
        y = _silu(y[:, :c["n"] // 2]) * y[:, c["n"] // 2:]
    return y.to(_TYPES[c["out"]])


# ---------------------------------------------------------------- the library's calls
def _library():
    pkg = os.path.join(os.getcwd(), "star-kv_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import starkv
    return starkv


def run(state):
    if not own:
        return _plain(state)
    starkv, s, c = _library(), state, state["case"]
    if c["op"] == "quantize":
        return starkv.fp8_quantize(s["x"], scale_dtype=_TYPES[c["scale"]])
    if c["op"] == "logprobs":
        return starkv.token_logprobs(s["logits"], s["tokens"], top=c["top"])
    fused = dict(residual=s.get("residual"), silu_mul=c["epilogue"] == "silu_mul", out_dtype=_TYPES[c["out"]])
    if c["op"] == "matmul":
        return starkv.fp8_matmul(s["x"], s["x_scale"], s["w"], s["w_scale"], **fused)
    return starkv.fp8_linear(s["x"], s["w"], s["w_scale"], rms_eps=1e-5 if c["rms"] else None, **fused)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    size = {"f16": 2, "bf16": 2, "f32": 4, "e8m0": 1}
    if c["op"] == "quantize":
        n = c["rows"] * c["k"]
        return {"bytes": n * size[c["dtype"]] + n + c["rows"] * _ceil(c["k"], BLOCK) * size[c["scale"]], "flops": 2 * n}
    if c["op"] == "logprobs":
        n = c["rows"] * c["vocab"]
        return {"bytes": n * size[c["dtype"]] + c["rows"] * (16 + 12 * c["top"]), "flops": 5 * n}
    m, n, k = c["m"], c["n"], c["k"]
    kb, so = _ceil(k, BLOCK), size[c["out"]]
    b = n * k + _ceil(n, BLOCK) * kb * size[c["scale"]]
    b += m * k * size[c["dtype"]] if c["op"] == "linear" else m * k + m * kb * size[c["scale"]]
    b += m * n * so // (2 if c["epilogue"] == "silu_mul" else 1)
    if c["epilogue"] == "residual":
        b += m * n * so
    return {"bytes": b, "flops": 2 * m * n * k}


# ---------------------------------------------------------------- the definitions in fp64
def _e4m3(v):
    """fp64 values of at most 448 (1 + 2^-6) to the nearest of e4m3 (ties to even): 4 significant bits, steps of at
    least 2^-9."""
    _, e = torch.frexp(v)
    step = ((e.long() - 4).clamp_min(-9) + 1023 << 52).view(torch.float64)
    return torch.round(v / step) * step


def _exact_quantize(x, kind):
    """Quantised values and scales, fp64, of fp64 rows.  With fp32 scales the reciprocal and the scaled value are fp32
    numbers by definition: a value half way between two of e4m3 is common there (x and the maximum are short numbers)."""
    rows, k = x.shape
    nb = _ceil(k, BLOCK)
    xp = torch.zeros(rows, nb * BLOCK, dtype=torch.float64, device=x.device)
    xp[:, :k] = x
    xp = xp.view(rows, nb, BLOCK)
    top = torch.maximum(xp.amax(2), -xp.amin(2))
    if kind == "e8m0":
        s = torch.exp2(torch.ceil(torch.log2(torch.where(top > 0, top, E4M3_MAX) / E4M3_MAX)).clamp(-126, 127))
        q = xp / s[..., None]
    else:
        floor = torch.maximum(top, torch.full_like(top, F32_AMAX_FLOOR))
        s = torch.where(top > 0, (floor / E4M3_MAX).float().double(), 1.0)
        q = (xp * (E4M3_MAX / floor).float().double()[..., None]).float().double()
    return _e4m3(q).view(rows, -1)[:, :k], s


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "quantize":
        return _exact_quantize(s["x"].double(), c["scale"])
    if c["op"] == "logprobs":
        x = s["logits"].double()
        lse = torch.logsumexp(x, -1)
        p = torch.softmax(x, -1)
        entropy = lse - (p * torch.where(p > 0, x, 0.0)).sum(-1)
        ids = torch.argsort(-x, dim=-1, stable=True)[:, :c["top"]]
        rows = torch.arange(x.shape[0], device=x.device)
        return x[rows, s["tokens"]] - lse, entropy, x[rows[:, None], ids] - lse[:, None], ids
    cols = torch.arange(c["k"], device="cuda") // BLOCK
    if c["op"] == "linear":
        x = s["x"].double()
        q, sx = _exact_quantize(x, c["scale"])
    else:
        q, sx = s["x"].double(), s["x_scale"].double()
    out_rows = torch.arange(c["n"], device="cuda") // BLOCK
    w = s["w"].double() * s["w_scale"].double()[out_rows][:, cols]
    y = torch.matmul(q * sx[:, cols], w.t().contiguous())
    if c["rms"]:
        y = y / torch.sqrt((x * x).sum(-1) / c["k"] + 1e-5)[:, None]
    if c["epilogue"] == "residual":
        y = y + s["residual"].double()
    elif c["epilogue"] == "silu_mul":
        gate, up = y[:, :c["n"] // 2], y[:, c["n"] // 2:]
        y = gate * torch.sigmoid(gate) * up
    return y
