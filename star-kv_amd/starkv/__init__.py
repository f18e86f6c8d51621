"""starkv: MI355X (gfx950) decode and prefill attention over STAR-KV low-rank latent caches, shared
and bounded ones among them, with the 8-bit projections and token log probabilities of the models around it.

The compute lives in libstarkv.so (HIP kernels behind the C ABI of
include/starkv.h); this package binds it to torch tensors.
"""
from ._lib import StarKVError, lib
from .bounded import attention_scores, keep_positions, select_positions
from .fp8 import fp8_linear, fp8_matmul, fp8_quantize, fp8_quantize_weight
from .logprobs import TokenLogprobs, token_logprobs
from .ops import KLatentSpec, VLatentSpec, decode_attention, k_logits, prefill_attention, pv_latent, rope_apply
from .prefix import SharedPrefix, prefix_decode_attention
from .rope import RopeConfig, rope_table

__all__ = ["StarKVError", "lib", "KLatentSpec", "VLatentSpec", "decode_attention", "k_logits", "prefill_attention",
           "pv_latent", "rope_apply", "fp8_linear", "fp8_matmul", "fp8_quantize", "fp8_quantize_weight",
           "TokenLogprobs", "token_logprobs", "SharedPrefix", "prefix_decode_attention", "attention_scores",
           "select_positions", "keep_positions",
           "RopeConfig", "rope_table"]
