"""Tensors with a forward-mode tangent are refused (before anything else, so on the CPU too): no operator carries
one on, and an output without it would be taken for a constant."""
import pytest
import torch
from torch.autograd import forward_ad

import avelang_amd as ave

F32, BF = torch.float32, torch.bfloat16


def _t(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype)


def _cache():
    return ave.PagedKVCache(_t(2, 2, 16, 64), _t(2, 2, 16, 64))


I32 = dict(dtype=torch.int32)
QKV = dict(q=_t(1, 4, 2, 64), k=_t(1, 4, 2, 64), v=_t(1, 4, 2, 64))
GB = dict(g=_t(1, 4, 2, dtype=F32), beta=_t(1, 4, 2, dtype=F32))
AB = dict(a=_t(1, 4, 2), b=_t(1, 4, 2), A_log=_t(2), dt_bias=_t(2))
CALLS = [
    (ave.rms_norm, dict(x=_t(3, 64), weight=_t(64), residual=_t(3, 64)), {}),
    (ave.rms_norm_quant, dict(x=_t(3, 64), weight=_t(64), residual=_t(3, 64)), {}),
    (ave.rms_norm_bwd, dict(h=_t(3, 64), weight=_t(64), dy=_t(3, 64)), {}),
    (ave.rotary_embedding, dict(q=_t(4, 2, 64), k=_t(4, 2, 64)),
     dict(positions=torch.zeros(4, **I32), inv_freq=_t(32, dtype=F32))),
    (ave.paged_cache_write, dict(k=_t(4, 2, 64), v=_t(4, 2, 64)), dict(cache=_cache(), slots=torch.arange(4))),
    (ave.paged_attention, dict(q=_t(1, 1, 2, 64)),
     dict(cache=_cache(), block_table=torch.zeros(1, 1, **I32), lengths=torch.zeros(1, **I32))),
    (ave.layer_norm, dict(x=_t(3, 64), weight=_t(64), bias=_t(64)), {}),
    (ave.chunk_gated_delta_rule, dict(**QKV, **GB, initial_state=_t(1, 2, 64, 64, dtype=F32)), {}),
    (ave.fused_recurrent_gated_delta_rule, dict(**QKV, **GB), {}),
    (ave.chunk_gated_delta_rule_gated, dict(**QKV, a=AB["a"], b=AB["b"]), dict(A_log=AB["A_log"], dt_bias=AB["dt_bias"])),
    (ave.chunk_linear_attn, dict(**QKV, g=GB["g"]), {}),
    (ave.fused_recurrent_linear_attn, dict(**QKV, g=GB["g"]), {}),
    (ave.fused_gdn_gating, AB, {}),
    (ave.l2norm_fwd, dict(x=_t(3, 64)), {}),
    (ave.causal_conv1d_fn, dict(x=_t(1, 64, 8), weight=_t(64, 4)), {}),
    (ave.causal_conv1d_update, dict(x=_t(1, 64), conv_state=_t(1, 64, 3), weight=_t(64, 4)), {}),
    (ave.rms_norm_gated, dict(x=_t(3, 64), z=_t(3, 64), weight=_t(64)), {}),
]


@pytest.mark.parametrize("call,of,rest", CALLS, ids=lambda x: getattr(x, "__name__", ""))
def test_refused(call, of, rest):
    for name, t in of.items():
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(t, torch.ones_like(t))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(**{**of, name: dual}, **rest)
    with forward_ad.dual_level(), pytest.raises(ValueError, match="ROCm"):   # tensors without one go on
        call(**of, **rest)


def test_cache_tensors():
    with forward_ad.dual_level():
        k, v = (forward_ad.make_dual(_t(2, 2, 16, 64), torch.ones(2, 2, 16, 64).to(BF)) for _ in "kv")
        cache = ave.PagedKVCache(k, v)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ave.paged_cache_read(cache, torch.arange(3))
