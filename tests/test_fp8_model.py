"""Refusals of the decoder's 8-bit form and of score(), on the CPU."""
import pytest
import torch


def _model(intermediate=256, dtype=torch.float16):
    from starkv.e2e import build_model
    return build_model(n_layers=1, hidden=256, heads=2, kv_heads=1, intermediate=intermediate, vocab=64, ranks=[32],
                       v_rank=32, batch=1, capacity=8, fmt="dense", device="cpu", dtype=dtype, fused=False)


def test_fuse_layers_refuses_before_it_changes_anything():
    from starkv import StarKVError
    from starkv.e2e import build_model, fuse_layers_
    e8 = torch.float8_e8m0fnu
    for model, fp8 in ((_model(), torch.float8_e4m3fn), (_model(), torch.float16), (_model(intermediate=192), e8),
                       (_model(dtype=torch.float32), e8)):
        with pytest.raises(StarKVError, match="fuse_layers_"):
            fuse_layers_(model, fp8=fp8)
        assert not hasattr(model.model.layers[0].mlp, "gate_up_weight")
        assert not hasattr(model.model.layers[0], "starkv_fp8")
    with pytest.raises(StarKVError, match="fused"):
        build_model(n_layers=1, hidden=256, heads=2, kv_heads=1, intermediate=256, vocab=64, ranks=[32], v_rank=32,
                    batch=1, capacity=8, device="cpu", fused=False, fp8=e8)


def test_score_refuses():
    from starkv import StarKVError
    from starkv.e2e import decode_graphed, generate, generate_graphed, score
    model = _model()
    ids = torch.zeros(1, 4, dtype=torch.int64)
    for top in (-1, 65):                                 # before any forward: the caches stay where they are
        for call in (lambda: score(model, ids, top=top), lambda: generate(model, ids, 1, logprobs=top),
                     lambda: generate_graphed(model, ids, 1, logprobs=top),
                     lambda: decode_graphed(model, ids[:, :1], 1, logprobs=top)):
            with pytest.raises(StarKVError, match="alternatives"):
                call()
        assert model.model.layers[0].self_attn.cache.length == 0
    for tokens in (torch.zeros(4, dtype=torch.int64), torch.zeros(1, 0, dtype=torch.int64),
                   torch.zeros(1, 4, dtype=torch.int32)):
        with pytest.raises(StarKVError, match="score"):
            score(model, tokens)
