"""GPU tests of a decoder whose projections run on e4m3 weights
(fuse_layers_(fp8=...)) and of the log probabilities of what it generates and
scores: the 8-bit operators, the latent attentions and token_logprobs in one
run, as a user of the model has them.

Every product and every log probability of the run is recorded with the inputs
it had and checked against its definition in 64 bits, with the bounds of
test_gpu_fp8.py and test_gpu_logprobs.py."""
import pytest
import torch

import test_gpu_fp8 as products
import test_gpu_logprobs as probabilities
from _util import KernelRecorder

pytestmark = pytest.mark.gpu

E8, F32 = torch.float8_e8m0fnu, torch.float32
F16, BF16 = torch.float16, torch.bfloat16
L, B, P, STEPS, V = 2, 2, 40, 4, 1000
KW = dict(n_layers=L, hidden=1024, heads=8, kv_heads=2, intermediate=2048 + 128, vocab=V, ranks=[48, 96], v_rank=256,
          batch=B, capacity=2 * (P + STEPS) + 3)


def _prompt(seed=6, n=P):
    return torch.randint(0, V, (B, n), generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


class Record:
    """Records the fp8_linear and token_logprobs calls that starkv.e2e makes."""

    def __init__(self, monkeypatch):
        import starkv.e2e as e2e
        self.products, self.probs = [], []
        linear, logprobs = e2e.fp8_linear, e2e.token_logprobs

        def rec_linear(x, w, ws, residual=None, silu_mul=False, rms_eps=None, out=None):
            c = dict(x=x.clone().reshape(-1, x.shape[-1]), w=w, ws=ws, n=w.shape[0], k=w.shape[1], scale=ws.dtype,
                     dtype=x.dtype, epilogue="silu_mul" if silu_mul else "none", out=x.dtype,
                     res=None if residual is None else residual.clone().reshape(-1, residual.shape[-1]))
            c["m"] = c["x"].shape[0]
            got = linear(x, w, ws, residual=residual, silu_mul=silu_mul, rms_eps=rms_eps, out=out)
            self.products.append((got.clone().reshape(c["m"], -1), c, rms_eps))
            return got

        def rec_logprobs(x, tokens=None, top=0):
            got = logprobs(x, tokens, top)
            self.probs.append((x.clone(), tokens.clone(), top, type(got)(*(t.clone() for t in got))))
            return got

        monkeypatch.setattr(e2e, "fp8_linear", rec_linear)
        monkeypatch.setattr(e2e, "token_logprobs", rec_logprobs)

    def check(self):
        torch.cuda.synchronize()
        for got, c, eps in self.products:
            products.check(got, c, rms_eps=eps)
        for x, tokens, top, got in self.probs:
            probabilities.check(x, tokens, top, got)


@pytest.mark.parametrize("dtype,scale,fmt", [(F16, E8, "int8_g64"), (BF16, E8, "int8_g64"), (F16, F32, "dense")],
                         ids=["f16-e8m0", "bf16-e8m0", "f16-f32"])
def test_generate_and_score(dtype, scale, fmt, monkeypatch):
    import starkv.e2e as e2e
    model = e2e.build_model(**KW, fmt=fmt, seed=3, dtype=dtype, fp8=scale)
    with KernelRecorder(e2e) as rec, monkeypatch.context() as mp:
        r = Record(mp)
        toks, logits, probs = e2e.generate(model, _prompt(), STEPS, logprobs=5)
        assert len(r.products) == 4 * L * (STEPS + 1) and len(r.probs) == STEPS + 1
        assert [c[1]["m"] for c in r.products[::4 * L]] == [B * P] + [B] * STEPS
        assert len(rec.calls) == L * (STEPS + 1)
        if dtype == F16:
            # the recorder's oracle keeps K and V unrounded, and its mean-rel 1e-3 is
            # for float16 outputs; bfloat16 prefill is gated in test_gpu_prefill.py
            # against an oracle that rounds as the kernel does
            assert rec.check() == L * (STEPS + 1)
        r.check()
        # greedy: each token is its row's most probable one
        assert toks.shape == probs.logprob.shape == probs.entropy.shape == (B, STEPS + 1)
        assert probs.top_ids.shape == (B, STEPS + 1, 5) and torch.equal(probs.top_logprobs[..., 0], probs.logprob)
        r.products.clear(), r.probs.clear()
        mp.setattr(e2e, "SCORE_LOGITS", 13 * V)                        # several pieces, the last one short
        held = [a.cache.length for a in e2e.attention_layers(model)]
        s = e2e.score(model, toks, top=3)
        assert held == [P + STEPS] * L == [a.cache.length for a in e2e.attention_layers(model)]
        assert s.logprob.shape == (B, STEPS) and s.top_ids.shape == (B, STEPS, 3)
        again = e2e.score(model, toks, top=3)
        assert all(torch.equal(a, b) for a, b in zip(s, again))
        e2e.score(model, _prompt(9), top=3)
        assert [p[0].shape[0] for p in r.probs] == [8] * 2 + [13] * 6
        r.check()
        one = e2e.score(model, toks[:, :1], top=3)
        assert one.logprob.shape == (B, 0) and one.top_ids.shape == (B, 0, 3)


def test_graph_replays_are_the_eager_steps():
    """decode_graphed's replays give, bit for bit, what the same steps give
    run one by one: tokens, logits and log probabilities."""
    import starkv.e2e as e2e
    model = e2e.build_model(**KW, fmt="int8_g64", seed=4, fp8=E8)
    atts = e2e.attention_layers(model)
    steps = 6
    toks, logits, probs = e2e.generate_graphed(model, _prompt(), steps, logprobs=4)
    assert toks.shape == probs.logprob.shape == (B, steps + 1) and probs.top_ids.shape == (B, steps + 1, 4)
    torch.cuda.synchronize()
    state = e2e.DecodeGraphState(B, atts[0].cache.cap, P, "cuda")
    tok = toks[:, :1]
    for a in atts:
        a.graph = state
    with torch.no_grad():
        for i in range(steps):
            h = model.model.embed_tokens(tok)
            for layer in model.model.layers:
                h = layer(h, attention_mask=None, position_ids=None, position_embeddings=None)
            last = model.lm_head(model.model.norm(h)[:, -1])
            tok = last.argmax(-1, keepdim=True)
            want = e2e.token_logprobs(last, tok[:, 0], 4)
            state.advance()
            assert torch.equal(logits[i + 1], last.float()) and torch.equal(toks[:, i + 1:i + 2], tok)
            for a, b in zip(probs, want):
                assert torch.equal(a[:, i + 1], b)
    for a in atts:
        a.graph = None
    state.check()
    # without log probabilities: the same tokens, two values as before
    for a in atts:
        a.cache.length = 0
    plain = e2e.generate_graphed(model, _prompt(), steps, keep_logits=False)
    assert len(plain) == 2 and torch.equal(plain[0], toks)
    for a in atts:
        a.cache.length = 0
    none = e2e.generate_graphed(model, _prompt(), 0, logprobs=0)
    assert none[2].logprob.shape == (B, 1) and torch.equal(none[2].logprob, probs.logprob[:, :1])


def test_layers_are_wired_as_the_16_bit_ones(monkeypatch):
    """With the products computed from the dequantised weights and unquantised
    activations, the 8-bit layers are the 16-bit layers of a model that holds
    those weights (norm weights and scales are powers of two: the fold is
    exact), within the mean-rel 1e-2 of the layers' 16-bit roundings."""
    import starkv.e2e as e2e
    model = e2e.build_model(**KW, fmt="dense", seed=5, fp8=E8)
    g = torch.Generator(device="cuda").manual_seed(1)
    with torch.no_grad():
        for layer in model.model.layers:
            for norm in (layer.input_layernorm, layer.post_attention_layernorm):
                norm.weight.copy_(torch.exp2(torch.randint(-1, 2, norm.weight.shape, generator=g, device="cuda").float()))
    toks, logits = e2e.generate(model, _prompt(), STEPS)               # requantises: the norms have changed

    def deq(q, s):
        return q.float() * s.float().repeat_interleave(128, 0)[:q.shape[0]].repeat_interleave(128, 1)[:, :q.shape[1]]

    plain = e2e.build_model(**KW, fmt="dense", seed=5)
    with torch.no_grad():
        for a, b in zip(model.model.layers, plain.model.layers):
            b.input_layernorm.weight.copy_(a.input_layernorm.weight)
            b.post_attention_layernorm.weight.copy_(a.post_attention_layernorm.weight)
            att, mlp = a.self_attn, a.mlp
            b.self_attn.qkv_weight.copy_(deq(*att.qkv_fp8) / a.input_layernorm.weight.float())
            b.self_attn.o_proj.weight.copy_(deq(*att.o_fp8))
            b.mlp.gate_up_weight.copy_(deq(*mlp.gate_up_fp8) / a.post_attention_layernorm.weight.float())
            b.mlp.down_proj.weight.copy_(deq(*mlp.down_fp8))
    want_toks, want = e2e.generate(plain, _prompt(), STEPS, forced=toks[:, :STEPS])

    def linear(x, w, ws, residual=None, silu_mul=False, rms_eps=None, out=None):
        xf = x.float()
        if rms_eps is not None:
            xf = xf * torch.rsqrt(xf.square().mean(-1, keepdim=True) + rms_eps)
        y = xf @ deq(w, ws).t().contiguous()
        if silu_mul:
            a, b = y.chunk(2, -1)
            y = torch.nn.functional.silu(a) * b
        if residual is not None:
            y = y + residual.float()
        return y.to(x.dtype) if out is None else out.copy_(y)

    for a in e2e.attention_layers(model):
        a.cache.length = 0
    monkeypatch.setattr(e2e, "fp8_linear", linear)
    _, got = e2e.generate(model, _prompt(), STEPS, forced=toks[:, :STEPS])
    for a, b in zip(got, want):
        rel = float((a.double() - b.double()).abs().mean() / b.double().abs().mean())
        print(f"   logits mean_rel={rel:.2e}", flush=True)
        assert rel <= 1e-2


def test_weights_loaded_later_reach_the_8bit_copies():
    import starkv.e2e as e2e
    want = e2e.build_model(**KW, fmt="int8_g64", seed=5, fp8=E8)
    toks, logits = e2e.generate(want, _prompt(8), STEPS)
    model = e2e.build_model(**KW, fmt="int8_g64", seed=4, fp8=E8)
    model.load_state_dict(want.state_dict())
    got_toks, got = e2e.generate(model, _prompt(8), STEPS)
    assert torch.equal(got_toks, toks) and all(torch.equal(a, b) for a, b in zip(got, logits))
    # back to 16 bits and to 8 again: fuse_layers_ decides
    e2e.fuse_layers_(model)
    assert model.model.layers[0].self_attn.qkv_fp8 is None and model.model.layers[0].self_attn.qkv_packed is not None
    e2e.fuse_layers_(model, fp8=E8)
    assert model.model.layers[0].self_attn.qkv_packed is None
    for a in e2e.attention_layers(model):
        a.cache.length = 0
    again, _ = e2e.generate(model, _prompt(8), STEPS)
    assert torch.equal(again, toks)


def test_score_after_a_shared_prefix():
    """Positions scored behind a prefix that the caches hold are those of the
    whole sequence (a 16-bit model: the latents and the masks are the same,
    the products' row counts are not), mean-rel 1e-3."""
    import starkv.e2e as e2e
    model = e2e.build_model(**KW, fmt="int8_g64", seed=7)
    tokens = _prompt(11, n=P)
    whole = e2e.score(model, tokens, top=2)
    assert all(a.cache.length == 0 for a in e2e.attention_layers(model))
    with torch.no_grad():
        model(input_ids=tokens[:, :17], position_ids=torch.arange(17, device="cuda")[None].expand(B, 17), use_cache=False)
    for seed in (12, 11):                                            # another continuation first
        part = e2e.score(model, tokens[:, 17:] if seed == 11 else _prompt(seed, n=9), top=2)
        assert all(a.cache.length == 17 for a in e2e.attention_layers(model))
    rel = float((part.logprob - whole.logprob[:, 17:]).abs().mean() / whole.logprob.abs().mean())
    print(f"   logprob mean_rel={rel:.2e}", flush=True)
    assert rel <= 1e-3


def test_one_token_prompts_and_texts():
    """A prompt of one token (every forward is a decode step), a text of two, one sequence."""
    import starkv.e2e as e2e
    kw = dict(KW, batch=1)
    model = e2e.build_model(**kw, fmt="int8_g64", seed=8, fp8=F32)
    prompt = _prompt(3)[:1, :1]
    toks, logits, probs = e2e.generate(model, prompt, 3, logprobs=0)
    assert toks.shape == probs.logprob.shape == (1, 4) and probs.top_ids.shape == (1, 4, 0)
    for i, row in enumerate(logits):
        probabilities.check(row, toks[:, i], 0, type(probs)(*(t[:, i] for t in probs)))
    for a in e2e.attention_layers(model):
        a.cache.length = 0
    s = e2e.score(model, torch.cat([prompt, toks[:, :1]], 1), top=64)
    assert s.logprob.shape == (1, 1) and s.top_ids.shape == (1, 1, 64)
    assert bool((s.top_logprobs[..., :-1] >= s.top_logprobs[..., 1:]).all())
