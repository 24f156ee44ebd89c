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


def linear_attn_chunked(q, k, v, g, do=None, dht=None, scale=None, h0=None, cu=None, chunk=64):
    """``(o, ht)``, and with do also ``(dq, dk, dv, dg, dh0)``, in float64 on q's
    device by the formulas of chunks written out, for lengths that the token
    loop and its autograd graph are too slow for."""
    q, k, v, g = (x.double() for x in (q, k, v, g))
    B, T, Hqk, K = q.shape
    Hv, V = v.shape[2:]
    rep, s = Hv // Hqk, K ** -0.5 if scale is None else scale
    per_head = g.dim() == 1
    g = g.expand(B, T, Hv) if per_head else g
    spans = [(b, 0, T) for b in range(B)] if cu is None else [(0, a, e) for a, e in zip(cu[:-1], cu[1:])]
    heads = lambda x: x.transpose(0, 1)   # noqa: E731  [tokens, H, ..] -> [H, tokens, ..]
    out = dict(o=torch.zeros_like(v), dq=torch.zeros(B, T, Hv, K, dtype=q.dtype, device=q.device),
               dk=torch.zeros(B, T, Hv, K, dtype=q.dtype, device=q.device), dv=torch.zeros_like(v),
               dg=torch.zeros(B, T, Hv, dtype=q.dtype, device=q.device))
    hts, dh0s = [], []
    for n, (b, start, end) in enumerate(spans):
        parts = []
        for a in range(start, end, chunk):
            at = slice(a, min(a + chunk, end))
            Q, Kc = (heads(x[b, at].repeat_interleave(rep, 1)) for x in (q, k))
            G = heads(g[b, at]).cumsum(1)
            gam = torch.exp(G[:, :, None] - G[:, None]).tril() * s
            parts.append((at, Q, Kc, heads(v[b, at]), G, G[:, -1:] - G, gam))
        S = torch.zeros(Hv, K, V, dtype=q.dtype, device=q.device) if h0 is None else h0[n].double()
        starts = []
        for at, Q, Kc, Vc, G, R, gam in parts:
            starts.append(S)
            P = gam * (Q @ Kc.mT.contiguous())
            out["o"][b, at] = heads(P @ Vc + s * G.exp()[..., None] * (Q @ S))
            S = G[:, -1].exp()[:, None, None] * S + Kc.mT.contiguous() @ (R.exp()[..., None] * Vc)
        hts.append(S)
        if do is None:
            continue
        D = torch.zeros_like(S) if dht is None else dht[n].double()
        for (at, Q, Kc, Vc, G, R, gam), S in reversed(list(zip(parts, starts))):
            O = heads(do[b, at].double())
            raw = O @ Vc.mT.contiguous()
            P, dP = gam * (Q @ Kc.mT.contiguous()), gam * raw
            iq = s * G.exp()[..., None] * (O @ S.mT.contiguous())
            ik = R.exp()[..., None] * (Vc @ D.mT.contiguous())
            out["dv"][b, at] = heads(P.mT.contiguous() @ O + R.exp()[..., None] * (Kc @ D))
            out["dk"][b, at] = heads(dP.mT.contiguous() @ Q + ik)
            out["dq"][b, at] = heads(dP @ Kc + iq)
            M = P * raw
            x, y = (Q * iq).sum(2) + M.sum(2) - M.sum(1), (Kc * ik).sum(2)
            out["dg"][b, at] = heads(G[:, -1:].exp() * (S * D).sum((1, 2))[:, None]
                                     + x.flip(1).cumsum(1).flip(1) + y.cumsum(1) - y)
            D = G[:, -1].exp()[:, None, None] * D + Q.mT.contiguous() @ (s * G.exp()[..., None] * O)
        dh0s.append(D)
    if do is None:
        return out["o"], torch.stack(hts)
    dq, dk = (out[x].reshape(B, T, Hqk, rep, K).sum(3) for x in ("dq", "dk"))
    dg = out["dg"].sum((0, 1)) if per_head else out["dg"]
    return out["o"], torch.stack(hts), dq, dk, out["dv"], dg, torch.stack(dh0s)
