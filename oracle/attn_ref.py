"""RMS norm, rotary positions, rows in 8 bits and attention over a cache, in 64 bits.

The definitions written out in torch float64 on the CPU; gradients are autograd's
of these same lines.
"""
import torch

MOST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def rms_norm(x, w=None, res=None, eps=1e-6, offset=0.0, rounded=True):
    """``(y, h)`` in float64; h = x + res rounded to res' type unless not ``rounded``
    (for gradients, which take the rounding as none)."""
    h = x.double()
    if res is not None:
        h = h + res.double()
        if rounded:
            h = h.to(res.dtype).double()
    y = h / ((h * h).mean(-1, keepdim=True) + eps).sqrt()
    return (y if w is None else y * (w.double() + offset)), h


def rotary(x, pos, freq, magnitude=1.0, near=False):
    """x [B, T, H, D] at pos [B, T] (or [T])."""
    x = x.double()
    r = 2 * freq.numel()
    t = (pos.double()[..., None] * freq.double())[..., None, :]
    a, b = (x[..., :r:2], x[..., 1:r:2]) if near else (x[..., :r // 2], x[..., r // 2:r])
    a, b = magnitude * (a * t.cos() - b * t.sin()), magnitude * (b * t.cos() + a * t.sin())
    y = torch.stack([a, b], -1).flatten(-2) if near else torch.cat([a, b], -1)
    return torch.cat([y, x[..., r:]], -1)


def codes(x, dtype):
    """``(codes, scale)`` of rows x: round(x M / max |x|) to nearest, ties to even, as
    float64 values (rows of 2^-100 at least, or zeros), scale fp32."""
    x = x.double()
    most = x.abs().amax(-1, keepdim=True)
    z = x * MOST[dtype] / torch.where(most > 0, most, 1.0)
    if dtype is torch.int8:
        step = torch.ones_like(z)
    else:   # three bits behind the leading one, no exponent under -6
        step = torch.exp2((torch.frexp(z)[1] - 4).clamp(min=-9).double())
    return (z / step).round() * step, (most[..., 0] / MOST[dtype]).float()


def rows_of(cache, scale, pages, n):
    """The first n cached rows [H, n, D] of the sequence whose pages are listed."""
    x = torch.stack([cache[p].double() * (1.0 if scale is None else scale[p].double()[..., None])
                     for p in pages]) if pages else cache[:0].double()
    H, D = cache.shape[1], cache.shape[3]
    return x.transpose(0, 1).reshape(H, -1, D)[:, :n]


def attention(q, k, v, scale, window=0):
    """q [L, Hq, D] the newest L of k, v [H, n, D]'s tokens: ``(o, lse, mean of |v|)``
    under the softmax, [L, Hq, D], [L, Hq], [L, Hq, D]; rows that see nothing 0, -inf."""
    q = q.double()
    L, Hq, D = q.shape
    H, n, _ = k.shape
    o, size = torch.zeros(L, Hq, D, dtype=torch.float64), torch.zeros(L, Hq, D, dtype=torch.float64)
    lse = torch.full((L, Hq), -torch.inf, dtype=torch.float64)
    for i in range(L):
        p = n - L + i
        lo = max(0, p - window + 1) if window else 0
        if p < 0:
            continue
        for h in range(Hq):
            kk, vv = k[h // (Hq // H), lo:p + 1], v[h // (Hq // H), lo:p + 1]
            s = scale * (kk * q[i, h]).sum(-1)
            lse[i, h] = torch.logsumexp(s, 0)
            w = (s - lse[i, h]).exp()
            o[i, h], size[i, h] = w @ vv, w @ vv.abs()
    return o, lse, size
