"""Linear attention with a decay for each head and layer norm, in 64 bits.

The token recurrence
    S_t = e^{g_t} S_{t-1} + k_t v_t^T,   o_t = scale S_t^T q_t
and the norm's definition, written out in torch float64 on the CPU; the
gradients are autograd's of these same lines.
"""
import torch


def linear_attn(q, k, v, g, scale=None, h0=None, cu=None):
    """``(o, ht)`` in float64 from tensors of any type (q, k [B, T, Hqk, K],
    v [B, T, Hv, V], g [B, T, Hv] or [Hv], h0 [N, Hv, K, V], cu a list)."""
    q, k, v, g = (x.double() for x in (q, k, v, g))
    B, T, Hqk, K = q.shape
    Hv, V = v.shape[2:]
    scale = K ** -0.5 if scale is None else scale
    q, k = (x.repeat_interleave(Hv // Hqk, dim=2) for x in (q, k))
    a = (g.expand(B, T, Hv) if g.dim() == 1 else g).exp()
    if cu is None:
        spans = [(b, 0, T) for b in range(B)]
    else:
        spans = [(0, s, e) for s, e in zip(cu[:-1], cu[1:])]
    outs, states = [], []
    for n, (b, s, e) in enumerate(spans):
        S = torch.zeros(Hv, K, V, dtype=torch.float64) if h0 is None else h0[n].double()
        rows = []
        for t in range(s, e):
            S = a[b, t, :, None, None] * S + k[b, t, :, :, None] * v[b, t, :, None, :]
            rows.append(scale * (q[b, t, :, :, None] * S).sum(1))
        outs.append(torch.stack(rows) if rows else v.new_zeros(0, Hv, V))
        states.append(S)
    o = torch.stack(outs) if cu is None else torch.cat(outs)[None]
    return o, torch.stack(states)


def layer_norm(x, w=None, b=None, eps=1e-5):
    x = x.double()
    mid = x - x.mean(-1, keepdim=True)
    y = mid / ((mid * mid).mean(-1, keepdim=True) + eps).sqrt()
    if w is not None:
        y = y * w.double()
    return y if b is None else y + b.double()
