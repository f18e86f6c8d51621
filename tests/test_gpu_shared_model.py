"""A decoder whose sequences share one prompt, and one whose caches are bounded: the operators as a model uses them."""
import pytest
import torch

import starkv
from starkv import StarKVError, e2e

pytestmark = pytest.mark.gpu

L, B, P, STEPS, V = 2, 3, 50, 5, 500
KW = dict(n_layers=L, hidden=1024, heads=8, kv_heads=4, intermediate=1024, vocab=V, ranks=[24, 40, 64, 32], v_rank=192)


def tokens(n, b=1, seed=0):
    return torch.randint(0, V, (b, n), generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("fmt", ["dense", "int8_g64", "reference"])
def test_shared_prompt_matches_copies_of_it(fmt):
    """decode_graphed behind a shared prompt against the same steps over a copy of it in every cache.  Both round like the
    decode kernels: a layer's attention is off by at most 2^-7 of its 2-norm either way (tests/test_gpu_prefix.py), the
    residual stream carries the layers' errors on, so logits agree within 2 L 2^-7 = 2^-5 of theirs.  A prompt one token
    shorter is further off."""
    prompt, first = tokens(P, seed=3), tokens(1, B, seed=4)
    model = e2e.build_model(batch=B, capacity=16, fmt=fmt, **KW)
    last = e2e.share_prompt(model, prompt)
    assert last.shape == (1, V)
    assert all(a.prefix.length == P and a.cache.length == 0 for a in e2e.attention_layers(model))
    toks, logits = e2e.decode_graphed(model, first, STEPS)
    copies = e2e.build_model(batch=B, capacity=P + 16, fmt=fmt, **KW)
    forced = torch.cat((first, toks[:, :-1]), 1)
    _, want = e2e.generate(copies, prompt.expand(B, P), STEPS, forced=forced)
    off = lambda a, b: ((a.double() - b.double()).norm() / b.double().norm()).item()
    assert off(last.expand(B, V).float(), want[0]) < 2.0 ** -5
    for got, ref in zip(logits, want[1:]):
        assert off(got, ref) < 2.0 ** -5
    # a second prompt takes the first one's place
    e2e.share_prompt(model, prompt[:, :-1].contiguous())
    _, other = e2e.decode_graphed(model, first, 1)
    assert off(other[0], want[1]) > 2.0 ** -5
    e2e.drop_prompt(model)
    assert all(a.prefix is None and a.cache.length == 0 for a in e2e.attention_layers(model))


def test_shared_prompt_eager_steps_and_refusals():
    prompt, first = tokens(P, seed=5), tokens(1, B, seed=6)
    model = e2e.build_model(batch=B, capacity=8, fmt="int8_g64", **KW)
    e2e.share_prompt(model, prompt)
    _, graphed = e2e.decode_graphed(model, first, 3)
    e2e.share_prompt(model, prompt)
    tok = first
    for step in range(3):
        out = model(input_ids=tok, position_ids=torch.full((B, 1), step, device="cuda"), use_cache=False)
        rel = (out.logits[:, -1].float() - graphed[step]).norm() / graphed[step].norm()
        assert rel < 2.0 ** -5
        tok = out.logits[:, -1].argmax(-1, keepdim=True)
    with pytest.raises(StarKVError):
        e2e.generate(model, tokens(4, B), 1)
    with pytest.raises(StarKVError):
        e2e.share_prompt(model, tokens(4, B))
    with pytest.raises(StarKVError):
        e2e.generate_bounded(model, tokens(4, B), 1, keep=4)
    one = e2e.share_prompt(model, prompt[:, :1].contiguous())
    assert one.shape == (1, V) and torch.isfinite(one).all()


@pytest.mark.parametrize("fmt", ["dense", "int8_g64", "reference"])
def test_bounded_generation(fmt):
    """The same tokens as an unbounded cache while nothing had to go; afterwards the caches hold what LatentCache.bound
    says: every bound keeps the sinks, the recent positions, and the largest sums between."""
    cap, steps, keep = 24, 30, 12
    prompt = tokens(20, B, seed=7)
    model = e2e.build_model(batch=B, capacity=cap, fmt=fmt, **KW)
    seen = []
    bound = starkv.cache.LatentCache.bound

    def watch(self, n, scores, sinks, recent):
        before = scores.clone()
        p = bound(self, n, scores, sinks, recent)
        seen.append((before, p.clone(), scores.clone()))
        return p

    starkv.cache.LatentCache.bound = watch
    try:
        toks, logits = e2e.generate_bounded(model, prompt, steps, keep, sinks=2, recent=4)
    finally:
        starkv.cache.LatentCache.bound = bound
    assert toks.shape == (B, steps + 1) and len(logits) == steps + 1
    assert all(torch.isfinite(x).all() for x in logits)
    assert len(seen) == L * 3                             # after 4 steps, and every 12
    for before, p, after in seen:
        assert p.shape == (B, keep)
        for b in range(B):
            s = before[b].clone()
            s[:2], s[cap - 4:] = float("inf"), float("inf")
            want = torch.sort(torch.sort(s, descending=True, stable=True).indices[:keep]).values
            assert torch.equal(p[b].long(), want)
            assert torch.equal(after[b, :keep], before[b, want]) and (after[b, keep:] == 0).all()
    assert all(a.scores is None and a.cache.length <= cap for a in e2e.attention_layers(model))
    free = e2e.build_model(batch=B, capacity=cap + steps, fmt=fmt, **KW)
    plain, want = e2e.generate(free, prompt, 4)
    for got, ref in zip(logits[:5], want):
        assert torch.equal(got, ref)
    assert torch.equal(toks[:, :5], plain)


def test_bounded_refusals():
    model = e2e.build_model(batch=B, capacity=16, fmt="dense", **KW)
    for args in ((tokens(17, B), 1, 8), (tokens(4, B), 1, 16), (tokens(4, B), 1, 3)):
        with pytest.raises(StarKVError):
            e2e.generate_bounded(model, *args)
