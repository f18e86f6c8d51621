"""Operators of a latent cache that is shared and kept bounded, as cases that can be timed and checked.

* prefix: one decode step of a batch whose sequences share a long prefix: attention over the prefix's latents, computed
  once for all, joined with attention over each sequence's own latents, and the value up-projection;
* scores: attention weights added up by position over the heads, from attention logits;
* select: the positions that a bounded cache keeps: the first and the latest, and those of the largest scores between;
* compact: the cache's rows of the kept positions moved together, in place, the scores with them.

``run`` computes them in plain fp32 torch, or with ``own`` by the library's calls; ``exact`` restates them in fp64.
"""
import math
import os
import random
import sys

import torch

own = False

HEAD_DIM = 128
_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # the smallest call: two continuations of a short prompt, their first token
        dict(name="prefix_two", op="prefix", batch=2, heads=8, kv=8, prefix=300, own=1, lo=16, hi=64, rv=512, theta=1e4,
             ragged=False, dtype="f16"),
        # eight samples of one 4099-token prompt, grouped heads of odd ranks, their lengths differ (one has nothing yet)
        dict(name="prefix_samples8", op="prefix", batch=8, heads=32, kv=8, prefix=4099, own=333, lo=33, hi=127, rv=1228,
             theta=5e5, ragged=True, dtype="bf16"),
        # four requests behind one system prompt of 16384 tokens
        dict(name="prefix_gqa4", op="prefix", batch=4, heads=32, kv=8, prefix=16384, own=1024, lo=64, hi=128, rv=512,
             theta=5e5, ragged=False, dtype="bf16"),
        # the largest: batch 16 over 32768 shared positions
        dict(name="prefix_decode16", op="prefix", batch=16, heads=32, kv=32, prefix=32768, own=512, lo=8, hi=96, rv=1640,
             theta=1e4, ragged=False, dtype="f16"),
        # a decode step of batch 8 behind an 8192-token prompt: the step's weights onto the sums
        dict(name="scores_step8", op="scores", batch=8, heads=32, len=8449, dtype="f32", masked=0.0, onto=True),
        # batch 16, context 32768
        dict(name="scores_long16", op="scores", batch=16, heads=32, len=32768, dtype="f32", masked=0.0, onto=True),
        # a padded batch of 16-bit logits: half of the places masked, some rows with nothing left
        dict(name="scores_masked", op="scores", batch=3, heads=12, len=777, dtype="bf16", masked=0.5, onto=False),
        # batch 8 behind an 8192-token prompt, bounded to 2048 positions
        dict(name="select_step8", op="select", batch=8, len=8449, keep=2048, sinks=4, recent=256, seen=1.0),
        # one long context of which a quarter is kept; half of its positions never got any weight
        dict(name="select_long", op="select", batch=1, len=131072, keep=32768, sinks=16, recent=1024, seen=0.5),
        # a layer's quantised cache of batch 8 bounded to 2048 positions
        dict(name="compact_int8", op="compact", batch=8, kv=32, len=8449, keep=2048, lo=8, hi=96, rv=1640, format="int8_g64",
             dtype="f16"),
        # a layer's 16-bit cache of batch 4, 32768 positions to 8192
        dict(name="compact_dense", op="compact", batch=4, kv=32, len=32768, keep=8192, lo=8, hi=96, rv=1640, format="dense",
             dtype="f16"),
        # one short context of grouped heads of odd ranks
        dict(name="compact_small", op="compact", batch=1, kv=8, len=301, keep=128, lo=17, hi=101, rv=333, format="dense",
             dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prefix", "prefix", "prefix", "scores", "select", "compact"])
    if op == "prefix":
        heads, kv = rng.choice([(32, 32), (32, 8), (8, 8), (16, 2), (40, 8), (64, 8)])
        lo = rng.randint(1, 100)
        c = dict(op=op, batch=_log(rng, 1, 40), heads=heads, kv=kv, prefix=_log(rng, 1, 65536),
                 own=rng.choice([0, _log(rng, 1, 2048)]), lo=lo, hi=rng.randint(lo, 128), rv=_log(rng, 16, 2048),
                 theta=rng.choice([1e4, 5e5]), ragged=rng.random() < 0.4, dtype=rng.choice(["f16", "bf16"]))
        big = listed()[3]
        while _prefix_work(c)["flops"] > _prefix_work(big)["flops"] or _prefix_work(c)["bytes"] > _prefix_work(big)["bytes"]:
            c["prefix"] = max(1, c["prefix"] * 3 // 4)
            c["own"] = c["own"] * 3 // 4
        return c
    if op == "scores":
        c = dict(op=op, batch=_log(rng, 1, 32), heads=rng.choice([1, 8, 12, 32, 40, 64]), len=_log(rng, 1, 131072),
                 dtype=rng.choice(["f32", "f32", "f16", "bf16"]), masked=rng.choice([0.0, 0.0, 0.3, 0.9]),
                 onto=rng.random() < 0.7)
        c["len"] = max(1, min(c["len"], 16 * 32 * 32768 // (c["batch"] * c["heads"])))
        return c
    n = _log(rng, 2, 131072)
    if op == "select":
        keep = rng.randint(1, n)
        sinks = rng.randint(0, min(keep, 64))
        return dict(op=op, batch=_log(rng, 1, 32), len=n, keep=keep, sinks=sinks, recent=rng.randint(0, keep - sinks),
                    seen=rng.choice([1.0, 1.0, 0.5, 0.0]))
    lo = rng.randint(1, 100)
    c = dict(op=op, batch=_log(rng, 1, 16), kv=rng.choice([1, 4, 8, 32]), len=n, keep=1, lo=lo, hi=rng.randint(lo, 128),
             rv=_log(rng, 16, 2048), format=rng.choice(["dense", "int8_g64"]), dtype=rng.choice(["f16", "bf16"]))
    c["len"] = max(2, min(c["len"], 4 * 32768 * 4096 // (c["batch"] * (c["kv"] * 64 + c["rv"]))))
    c["keep"] = rng.randint(1, c["len"])
    return c


# ---------------------------------------------------------------- inputs (from the seed alone)
def _ceil(a, b):
    return -(-a // b)


def _ranks(c):
    """Each KV head's own rank."""
    r = random.Random("%d %d %d" % (c["kv"], c["lo"], c["hi"]))
    return [r.randint(c["lo"], c["hi"]) for _ in range(c["kv"])]


def _width(c):
    """Elements from one position's K row to the next: the largest rank in whole 16-byte pieces."""
    return 8 * _ceil(max(_ranks(c)), 8)


def _rand(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _k_latents(g, ranks, *shape):
    """[..., heads, positions, width] N(0, 1), zeros behind each head's rank."""
    x = _rand(g, *shape)
    cols = torch.arange(shape[-1], device="cuda")
    return x.mul_(cols < torch.tensor(ranks, device="cuda")[:, None, None])


def _kept(g, batch, n, keep):
    """Ascending positions [batch, keep], as a selection by scores leaves them."""
    return torch.rand(batch, n, generator=g, device="cuda").topk(keep, -1).indices.sort(-1).values.int()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c, s = case, dict(case=case)
    if c["op"] == "scores":
        b, h, n, dt = c["batch"], c["heads"], c["len"], _TYPES[c["dtype"]]
        x = _rand(g, b, h, n) * 2.5
        if c["masked"]:
            x.masked_fill_(torch.rand(b, 1, n, generator=g, device="cuda") < c["masked"], -math.inf)
            x[b - 1, h // 2:] = -math.inf                    # rows whose mask leaves nothing
        s["logits"] = x.to(dt)
        if c["onto"]:
            s["before"] = _rand(g, b, n).exp_()
        return s
    if c["op"] == "select":
        # lognormal sums of weights; positions that were never looked at hold exact zeros (ties)
        x = torch.exp(2 * _rand(g, c["batch"], c["len"]))
        s["scores"] = x * (torch.rand(c["batch"], c["len"], generator=g, device="cuda") < c["seen"])
        return s
    dt, ranks, width = _TYPES[c["dtype"]], _ranks(c), _width(c)
    if c["op"] == "compact":
        b, n, kv, rv = c["batch"], c["len"], c["kv"], c["rv"]
        if c["format"] == "dense":
            s["k"] = [_k_latents(g, ranks, b, kv, n, width).to(dt)]
            s["v"] = [_rand(g, b, n, rv).to(dt)]
        else:
            pitch = 16 * _ceil(width, 16)
            s["k"] = [(_k_latents(g, ranks, b, kv, n, pitch) * 40).clamp_(-127, 127).to(torch.int8),
                      _rand(g, b, kv, 8 * _ceil(n, 8)).half()]
            v = torch.randint(0, 256, (b, n, 16 * _ceil(rv, 32)), generator=g, device="cuda", dtype=torch.uint8)
            v[..., _ceil(rv, 2):] = 0
            s["v"] = [v, _rand(g, b, n, _ceil(rv, 64)).half(), _rand(g, b, n, _ceil(rv, 64)).half()]
        s["scores"] = torch.exp(_rand(g, b, n))
        s["positions"] = _kept(g, b, n, c["keep"])
        return s
    b, hq, kv, p, n, rv = c["batch"], c["heads"], c["kv"], c["prefix"], c["own"], c["rv"]
    per_rank = torch.tensor(ranks, device="cuda").rsqrt()[:, None, None]
    s["bk"] = (_rand(g, kv, width, HEAD_DIM) * per_rank).to(dt)                # rows behind a head's rank are not read
    s["prefix_k"] = _k_latents(g, ranks, kv, p, width).to(dt)
    s["prefix_v"] = _rand(g, p, rv).to(dt)
    s["uv"] = (_rand(g, kv * HEAD_DIM, rv) / math.sqrt(rv)).to(dt)
    s["q"] = (2 * _rand(g, b, hq, HEAD_DIM)).to(dt)       # rotated at its position behind the sequence's own first one
    if n:
        s["k"] = _k_latents(g, ranks, b, kv, n, width).to(dt)
        s["v"] = _rand(g, b, n, rv).to(dt)
        if c["ragged"]:
            length = torch.randint(0, n + 1, (b,), generator=g, device="cuda")
            length[0], length[-1] = n, 0
            s["mask"] = torch.where(torch.arange(n, device="cuda") < length[:, None], 0.0, -math.inf)
    if own:
        # the handle that a serving program makes once, when the shared prompt has been read
        starkv = _library()
        s["rope"] = starkv.RopeConfig(theta=c["theta"])
        s["prefix"] = starkv.SharedPrefix(_spec(starkv, c, s["prefix_k"][None], s["bk"]), s["prefix_v"][None], rope=s["rope"])
    return s


# ---------------------------------------------------------------- the plain form
def _inv_freq(theta):
    return 1.0 / (theta ** (torch.arange(0, HEAD_DIM, 2, dtype=torch.int64).float() / HEAD_DIM))


def _rotate(x, first, theta):
    """Rotary positions first, first + 1, ... of x [..., positions, 128], angles in 64 bits."""
    n = x.shape[-2]
    angle = torch.arange(first, first + n, device=x.device).double()[:, None] * _inv_freq(theta).double().to(x.device)
    cos, sin = angle.cos().to(x.dtype), angle.sin().to(x.dtype)
    a, b = x[..., :64], x[..., 64:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _plain_prefix(s, f=torch.float32):
    c = s["case"]
    b, hq, kv, p, n = c["batch"], c["heads"], c["kv"], c["prefix"], c["own"]
    gs, scale = hq // kv, 1 / math.sqrt(HEAD_DIM)
    q, bk = s["q"].to(f), s["bk"].to(f)
    keys = _rotate(torch.matmul(s["prefix_k"].to(f), bk), 0, c["theta"])                       # [kv, p, 128]
    far = _rotate(q.unsqueeze(2), p, c["theta"])[:, :, 0]                                      # p positions further
    far = far.view(b, kv, gs, HEAD_DIM).transpose(0, 1).reshape(kv, b * gs, HEAD_DIM)
    logits = torch.matmul(far, keys.transpose(1, 2).contiguous()) * scale                      # [kv, b gs, p]
    logits = logits.view(kv, b, gs, p).transpose(0, 1).reshape(b, hq, p)
    del keys
    if n:
        keys = _rotate(torch.matmul(s["k"].to(f), bk), 0, c["theta"])                          # [b, kv, n, 128]
        near = torch.matmul(q.view(b, kv, gs, HEAD_DIM), keys.transpose(2, 3).contiguous()) * scale
        near = near.view(b, hq, n)
        if "mask" in s:
            near = near + s["mask"].to(f)[:, None, :]
        logits = torch.cat((logits, near), -1)
    w = torch.exp(logits - logits.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    o = torch.matmul(w[..., :p].reshape(b * hq, p), s["prefix_v"].to(f)).view(b, hq, -1)
    if n:
        o = o + torch.matmul(w[..., p:].contiguous(), s["v"].to(f))
    o = o.view(b, kv, gs, -1).transpose(0, 1).reshape(kv, b * gs, -1)
    u = s["uv"].to(f).view(kv, HEAD_DIM, -1).transpose(1, 2).contiguous()
    return torch.matmul(o, u).view(kv, b, gs, HEAD_DIM).transpose(0, 1).reshape(b, hq, HEAD_DIM)


def _plain_scores(s):
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    w = torch.exp(x - torch.where(top > -math.inf, top, 0.0))
    total = w.sum(-1, keepdim=True)
    w = (w / torch.where(total > 0, total, 1.0)).sum(1)
    return s["before"].add_(w) if "before" in s else w


def _plain_select(s):
    c, x = s["case"], s["scores"].clone()
    x[:, :c["sinks"]] = math.inf
    x[:, c["len"] - c["recent"]:] = math.inf
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :c["keep"]]
    return order.sort(-1).values.int()


def _plain_compact(s):
    c, i = s["case"], s["positions"].long()
    keep = c["keep"]

    def move(t, dim):
        at = i.view(i.shape[0], *[1] * (dim - 1), keep, *[1] * (t.dim() - dim - 1))
        shape = list(t.shape)
        shape[dim] = keep
        t.narrow(dim, 0, keep).copy_(t.gather(dim, at.expand(shape)))

    move(s["k"][0], 2)
    move(s["v"][0], 1)
    if c["format"] != "dense":
        move(s["k"][1], 2)
        move(s["v"][1], 1)
        move(s["v"][2], 1)
    move(s["scores"], 1)
    s["scores"][:, keep:] = 0
    return s["k"] + s["v"] + [s["scores"]]


# ---------------------------------------------------------------- the library's calls
def _library():
    pkg = os.path.join(os.getcwd(), "star-kv_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import starkv
    return starkv


def _spec(starkv, c, x, bk, scale=None):
    """x [b, heads, positions, width] as the library's description of K latents."""
    ranks = _ranks(c)
    heads = range(len(ranks))
    more = {} if scale is None else dict(fmt=starkv.ops.FMT_INT8_SYM, scale=scale, scale_stride_b=scale.stride(0),
                                         scale_stride_h=scale.stride(1))
    return starkv.KLatentSpec(x, ranks, [h * x.stride(1) for h in heads], [x.stride(2)] * len(ranks), x.stride(0), bk,
                              [h * bk.stride(0) for h in heads], bk.stride(1), **more)


def _own_compact(starkv, s):
    c = s["case"]
    bk = s["k"][0].new_empty(1, 1, HEAD_DIM).expand(c["kv"], 1, HEAD_DIM)       # not read
    k = _spec(starkv, c, s["k"][0], bk, s["k"][1] if len(s["k"]) > 1 else None)
    v = s["v"][0] if c["format"] == "dense" else \
        starkv.VLatentSpec.int4_g64(s["v"][0][..., :_ceil(c["rv"], 2)], s["v"][1], s["v"][2], c["rv"])
    starkv.keep_positions(k, v, s["positions"], c["len"], scores=s["scores"])
    return s["k"] + s["v"] + [s["scores"]]


def run(state):
    s, c = state, state["case"]
    if not own:
        if c["op"] == "prefix":
            return _plain_prefix(s).to(_TYPES[c["dtype"]])
        return {"scores": _plain_scores, "select": _plain_select, "compact": _plain_compact}[c["op"]](s)
    starkv = _library()
    if c["op"] == "prefix":
        k = _spec(starkv, c, s["k"], s["bk"]) if c["own"] else None
        return starkv.prefix_decode_attention(s["q"], s["prefix"], k, s.get("v"), s["uv"], mask=s.get("mask"))
    if c["op"] == "scores":
        return starkv.attention_scores(s["logits"], s.get("before"))
    if c["op"] == "select":
        return starkv.select_positions(s["scores"], c["keep"], sinks=c["sinks"], recent=c["recent"])
    return _own_compact(starkv, s)


# ---------------------------------------------------------------- what a pass cannot do without
def _prefix_work(c):
    b, hq, kv, p, n, rv, r = c["batch"], c["heads"], c["kv"], c["prefix"], c["own"], c["rv"], sum(_ranks(c))
    rows = p + b * n
    data = 2 * (rows * (r + rv) + r * HEAD_DIM + kv * HEAD_DIM * rv + 2 * b * hq * HEAD_DIM)
    return {"bytes": data, "flops": 2 * rows * r * HEAD_DIM + 2 * b * hq * ((p + n) * (HEAD_DIM + rv) + HEAD_DIM * rv)}


def work(case):
    c = case
    if c["op"] == "prefix":
        return _prefix_work(c)
    b = c["batch"]
    if c["op"] == "scores":
        n = b * c["len"]
        return {"bytes": n * c["heads"] * (4 if c["dtype"] == "f32" else 2) + n * (8 if c["onto"] else 4),
                "flops": 5 * n * c["heads"]}
    if c["op"] == "select":
        return {"bytes": 4 * b * (c["len"] + c["keep"]), "flops": b * c["len"]}
    r = sum(_ranks(c))
    row = 2 * (r + c["rv"]) if c["format"] == "dense" else r + 2 * c["kv"] + _ceil(c["rv"], 2) + 4 * _ceil(c["rv"], 64)
    return {"bytes": b * (c["keep"] * (2 * row + 8) + 4 * c["len"]), "flops": b * c["keep"]}


# ---------------------------------------------------------------- the definitions in fp64
def _exact_prefix(c, s):
    """One key at the distance it has: the prefix's position j lies prefix - j before a sequence's own first one."""
    b, hq, kv, p, n = c["batch"], c["heads"], c["kv"], c["prefix"], c["own"]
    gs = hq // kv
    inv = _inv_freq(c["theta"]).double().cuda()

    def turned(x, positions):
        z = torch.complex(x[..., :64], x[..., 64:])
        z = z * torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), positions[:, None] * inv)
        return torch.cat((z.real, z.imag), -1)

    out = []
    value = s["uv"].double().view(kv, HEAD_DIM, -1)
    for h in range(kv):
        bk = s["bk"][h].double()
        q = s["q"][:, h * gs:(h + 1) * gs].double().reshape(b * gs, HEAD_DIM)
        shared = turned(s["prefix_k"][h].double() @ bk, torch.arange(-p, 0, device="cuda").double())
        x = (q @ shared.t().contiguous()).view(b, gs, p) / math.sqrt(HEAD_DIM)
        if n:
            mine = turned(s["k"][:, h].double() @ bk, torch.arange(n, device="cuda").double())
            y = (q.view(b, gs, HEAD_DIM) @ mine.transpose(1, 2).contiguous()) / math.sqrt(HEAD_DIM)
            if "mask" in s:
                y = y + s["mask"].double()[:, None]
            x = torch.cat((x, y), -1)
        w = torch.softmax(x, -1)
        o = w[..., :p].reshape(b * gs, p) @ s["prefix_v"].double()
        if n:
            o = o + (w[..., p:].contiguous() @ s["v"].double()).view(b * gs, -1)
        out.append((o @ value[h].t().contiguous()).view(b, gs, HEAD_DIM))
    return torch.cat(out, 1)


def exact(case, seed):
    c = case
    if c["op"] == "select":
        return None
    s = prepare(case, seed)
    if c["op"] == "prefix":
        return _exact_prefix(c, s)
    if c["op"] == "scores":
        x = s["logits"].double()
        lse = torch.logsumexp(x, -1, keepdim=True)
        w = torch.where(lse > -math.inf, torch.exp(x - torch.where(lse > -math.inf, lse, 0.0)), 0.0).sum(1)
        return w + s["before"].double() if "before" in s else w
    keep, rows = c["keep"], torch.arange(c["batch"], device="cuda")[:, None]
    i = s["positions"].long()

    def moved(t, heads):
        if not t.is_floating_point():
            return None
        t = t.double()
        if heads:
            t[:, :, :keep] = t.transpose(1, 2)[rows, i].transpose(1, 2)
        else:
            t[:, :keep] = t[rows, i]
        return t

    scores = moved(s["scores"], False)
    scores[:, keep:] = 0
    return [moved(t, True) for t in s["k"]] + [moved(t, False) for t in s["v"]] + [scores]
