"""avelang_amd — MI355X-native (gfx950) gated-delta-net hot path.

Operators (FLA / Qwen3-Next argument lists):
    chunk_gated_delta_rule            chunked prefill (chunk 64, MFMA), differentiable
    chunk_gated_delta_rule_bwd        its gradients (q, k, v, g, beta, initial state)
    fused_recurrent_gated_delta_rule  token recurrence / decode (HBM-bound),
                                      optionally over a pool of state slots

Neighbours of the core in the Qwen3-Next layer (``layer_ops``):
    fused_gdn_gating (differentiable; fused_gdn_gating_bwd), l2norm_fwd,
    causal_conv1d_fn, causal_conv1d_update, rms_norm_gated

Linear attention with a decay for each head (``linear_attention``):
    chunk_linear_attn (differentiable; chunk_linear_attn_bwd),
    fused_recurrent_linear_attn
Layer norm (``norm``):
    layer_norm (differentiable; layer_norm_bwd)
What stands around a hybrid model's attention layers (``norm``, ``rotary``, ``paged_attention``):
    rms_norm (residual added; differentiable; rms_norm_bwd), rms_norm_quant (8 bits),
    rotary_embedding (differentiable), rotary_frequencies,
    PagedKVCache, paged_cache_write, paged_cache_read, paged_attention

All call hand-written HIP kernels through the C ABI in include/gdn.h, include/gdn_layer.h,
include/gdn_linear.h and include/gdn_attn.h (``libgdn.so``, built by ``python -m avelang_amd.build``).
"""
from .gated_delta_rule import (  # noqa: F401
    chunk_bwd_workspace_bytes,
    chunk_gated_delta_rule,
    chunk_gated_delta_rule_bwd,
    chunk_gated_delta_rule_fwd_save,
    chunk_gated_delta_rule_gated,
    chunk_workspace_bytes,
    fused_recurrent_gated_delta_rule,
    fused_recurrent_gated_delta_rule_gated,
)
from .layer_ops import (  # noqa: F401
    causal_conv1d_fn,
    causal_conv1d_update,
    fused_gdn_gating,
    fused_gdn_gating_bwd,
    l2norm_fwd,
    rms_norm_gated,
)
from .linear_attention import (  # noqa: F401
    chunk_linear_attn,
    chunk_linear_attn_bwd,
    chunk_linear_attn_fwd_save,
    fused_recurrent_linear_attn,
    linear_attn_workspace_bytes,
)
from .norm import (  # noqa: F401
    layer_norm,
    layer_norm_bwd,
    layer_norm_fwd_save,
    rms_norm,
    rms_norm_bwd,
    rms_norm_quant,
)
from .paged_attention import (  # noqa: F401
    PagedKVCache,
    paged_attention,
    paged_attention_workspace_bytes,
    paged_cache_read,
    paged_cache_write,
)
from .rotary import rotary_embedding, rotary_frequencies  # noqa: F401

__all__ = [
    "chunk_gated_delta_rule",
    "chunk_gated_delta_rule_bwd",
    "chunk_gated_delta_rule_fwd_save",
    "fused_recurrent_gated_delta_rule",
    "chunk_gated_delta_rule_gated",
    "fused_recurrent_gated_delta_rule_gated",
    "chunk_workspace_bytes",
    "chunk_bwd_workspace_bytes",
    "fused_gdn_gating",
    "fused_gdn_gating_bwd",
    "l2norm_fwd",
    "causal_conv1d_fn",
    "causal_conv1d_update",
    "rms_norm_gated",
    "chunk_linear_attn",
    "chunk_linear_attn_bwd",
    "chunk_linear_attn_fwd_save",
    "fused_recurrent_linear_attn",
    "linear_attn_workspace_bytes",
    "layer_norm",
    "layer_norm_bwd",
    "layer_norm_fwd_save",
    "rms_norm",
    "rms_norm_bwd",
    "rms_norm_quant",
    "rotary_embedding",
    "rotary_frequencies",
    "PagedKVCache",
    "paged_cache_write",
    "paged_cache_read",
    "paged_attention",
    "paged_attention_workspace_bytes",
]
