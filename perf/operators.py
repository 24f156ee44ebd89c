"""Linear attention with a decay for each head, and layer norm: calls as a serving or a training
program makes them, from one decoded token to packed prompts.

Linear attention (one state [K, V] per v-head, v-head h reads qk-head h // (Hv / Hqk)):
    S_t = e^{g_t} S_{t-1} + k_t v_t^T         o_t = K^{-1/2} S_t^T q_t
Layer norm over the last axis, with a weight and a bias of that axis or of the last two:
    y = (x - mean) / sqrt(var + eps) * weight + bias

``run`` calls the package's operators where ``own`` is set; else it computes the same in elementary
torch operations in fp32 (chunks of 64 tokens, all chunks' states at once through a matrix of the
decays between chunks; sums of log-decays in 64 bits).  ``exact`` walks the recurrence token by
token in 64 bits.

Case fields
    kind      prefill | decode | train | norm | norm_train
    seqs      sequences (batch rows; with ``packed`` the packed sequences of one row)
    tokens    tokens per sequence (with ``packed`` the largest length, ``least`` the smallest)
    hqk, hv   qk-heads and v-heads;  k, v: head sizes
    h0        an initial state is given (training: the final state's gradient too)
    slopes    one fixed decay per head instead of one per token and head
    rows, heads, d   norm: rows (heads = 0) or tokens of ``heads`` rows with parameters of their own
    x_type, w_type   norm: element types of the rows and of weight and bias
"""
import math

import torch
import torch.nn.functional as F

DEV = "cuda"
C = 64      # chunk of the plain form
EPS = 1e-5
own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    full = dict(hqk=16, hv=32, k=128, v=128)
    return [
        # a short ragged prompt
        dict(name="prefill_449", kind="prefill", seqs=1, tokens=449, packed=False, h0=False,
             slopes=False, **full),
        # a full prompt that continues a conversation: a state in, a state out
        dict(name="prefill_8k", kind="prefill", seqs=1, tokens=8192, packed=False, h0=True,
             slopes=False, **full),
        # 64 prompts of 128 .. 4096 tokens packed into one call, a fixed slope per head
        dict(name="prefill_packed_64", kind="prefill", seqs=64, tokens=4096, least=128, packed=True,
             h0=False, slopes=True, **full),
        # one GPU's heads of a layer split over eight, a ragged long document
        dict(name="prefill_shard_20k", kind="prefill", seqs=1, tokens=20011, packed=False, h0=True,
             slopes=False, hqk=2, hv=4, k=128, v=128),
        # one user's next token: the smallest call, all latency
        dict(name="decode_one", kind="decode", seqs=1, tokens=1, packed=False, h0=True,
             slopes=False, **full),
        # a full decode batch: streams the states of 256 sequences
        dict(name="decode_256", kind="decode", seqs=256, tokens=1, packed=False, h0=True,
             slopes=False, **full),
        # a training step of the operator: forward and every gradient, the decay's included
        dict(name="train_8k", kind="train", seqs=1, tokens=8192, packed=False, h0=False,
             slopes=False, **full),
        # training on packed documents of ragged length, four v-heads to a qk-head, the state
        # carried in and out
        dict(name="train_packed_6", kind="train", seqs=6, tokens=1500, least=100, packed=True,
             h0=True, slopes=False, hqk=4, hv=16, k=128, v=64),
        # the norm before a decoded token's projections
        dict(name="norm_one", kind="norm", rows=1, heads=0, d=2048, x_type="bf16", w_type="bf16"),
        # the norm of the attention's output in a prompt: every head's row by itself
        dict(name="norm_heads_8k", kind="norm", rows=8192, heads=32, d=128, x_type="bf16",
             w_type="f32"),
        # a training step of a layer's norm
        dict(name="norm_train_8k", kind="norm_train", rows=8192, heads=0, d=4096, x_type="bf16",
             w_type="f32"),
        # the same in 32 bits at odd sizes
        dict(name="norm_train_odd", kind="norm_train", rows=5003, heads=0, d=1001, x_type="f32",
             w_type="f32"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["prefill", "prefill", "decode", "train", "train", "norm", "norm_train"])
    if kind in ("norm", "norm_train"):
        heads = rng.choice([0, 0, 2, 8, 16, 32])
        d = _log_int(rng, 32, 512) if heads else _log_int(rng, 64, 8192)
        if rng.random() < 0.6:   # most models' rows are multiples of 16 elements
            d = -(-d // 16) * 16
        rows = _log_int(rng, 1, min(65536, (8192 * 4096) // (d * max(1, heads))))
        return dict(kind=kind, rows=rows, heads=heads, d=d, x_type=rng.choice(["bf16", "bf16", "f16", "f32"]),
                    w_type=rng.choice(["f32", "bf16"]))
    hqk, hv = rng.choice([(16, 32), (16, 32), (8, 16), (2, 4), (16, 16), (4, 16), (1, 8)])
    k, v = rng.choice([(128, 128), (128, 128), (128, 64), (64, 128), (64, 64)])
    c = dict(kind=kind, hqk=hqk, hv=hv, k=k, v=v, h0=rng.random() < 0.6, packed=False,
             slopes=rng.random() < 0.25)
    if kind == "decode":
        c.update(seqs=_log_int(rng, 1, 256), tokens=rng.choice([1, 1, 1, rng.randint(2, 6)]), h0=True)
        return c
    seqs = rng.choice([1, 1, 2, rng.randint(3, 8 if kind == "train" else 64)])
    if kind == "train":
        c.update(seqs=seqs, tokens=_log_int(rng, 2, 8192 // seqs), slopes=False)
    else:
        c.update(seqs=seqs, tokens=_log_int(rng, 1, min(65536 // seqs, 4096 if seqs > 2 else 65536)))
    if seqs > 2:
        c.update(packed=True, least=rng.randint(1, c["tokens"]))
    return c


def _lengths(case):
    if not case["packed"]:
        return [case["tokens"]] * case["seqs"]
    # a fixed spread of lengths between the least and the largest, in a mixed order
    n, lo, hi = case["seqs"], case["least"], case["tokens"]
    return [hi if i == 0 else lo + (hi - lo) * ((i * 29) % n) // n for i in range(n)]


# ------------------------------------------------------------------ inputs ----
def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))

    def randn(*shape):
        return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32)

    def rand(*shape):
        return torch.rand(shape, generator=gen, device=DEV, dtype=torch.float32)

    s = dict(case=dict(case))
    if case["kind"] in ("norm", "norm_train"):
        xt, wt = _TYPES[case["x_type"]], _TYPES[case["w_type"]]
        par = (case["heads"], case["d"]) if case["heads"] else (case["d"],)
        shape = (case["rows"],) + par
        # rows of different size and centre, as a residual stream or attention outputs have them
        s["x"] = (randn(*shape) * (0.5 + 2 * rand(*shape[:-1], 1)) + 0.3 * randn(*shape[:-1], 1)).to(xt)
        s["w"], s["b"] = (1 + 0.2 * randn(*par)).to(wt), (0.1 * randn(*par)).to(wt)
        if case["kind"] == "norm_train":
            s["dy"] = randn(*shape).to(xt)
            for n in ("x", "w", "b"):
                s[n].requires_grad_(True)
        return s

    bf = torch.bfloat16
    N, hqk, hv, K, V = (case[x] for x in ("seqs", "hqk", "hv", "k", "v"))
    lens = _lengths(case)
    B, T = (1, sum(lens)) if case["packed"] else (N, case["tokens"])
    # a layer's projections, and its decays: a rate exp(A_log) up to 16 per head times steps around
    # 1e-3 .. 1e-1 (memories from a few tokens to thousands), or one fixed slope per head
    s["q"], s["k"], s["v"] = (randn(B, T, h, d).to(bf) for h, d in ((hqk, K), (hqk, K), (hv, V)))
    if case["slopes"]:
        s["g"] = -torch.exp2(-8.0 * torch.arange(1, hv + 1, device=DEV, dtype=torch.float32) / hv)
        s["g"] = s["g"] * (0.9 + 0.2 * rand(hv))
    else:
        dt = torch.exp(rand(hv) * math.log(100.0) + math.log(0.001))
        bias = dt + torch.log(-torch.expm1(-dt))
        s["g"] = -(rand(hv) * 16 + 0.01) * F.softplus(0.5 * randn(B, T, hv) + bias)
    if case["h0"]:
        s["h0"] = 3 * randn(N, hv, K, V)
    if case["packed"]:
        # the program's plan of the batch: offsets, and each token's place in a padded layout
        cu = [0]
        for x in lens:
            cu.append(cu[-1] + x)
        s["cu"] = torch.tensor(cu, dtype=torch.int32, device=DEV)
        pad = -(-max(lens) // C) * C
        s["place"] = torch.cat([torch.arange(i * pad, i * pad + x) for i, x in enumerate(lens)]).to(DEV)
    if case["kind"] == "train":
        s["g"] = s["g"].to(bf)   # as a projection in bf16 gives it; its gradient comes in bf16 too
        s["do"] = randn(B, T, hv, V).to(bf)
        if case["h0"]:
            s["dht"] = randn(N, hv, K, V)
        for n in ("q", "k", "v", "g") + (("h0",) if case["h0"] else ()):
            s[n].requires_grad_(True)
    return s


# -------------------------------------------------------------------- call ----
def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        return _run_plain(s)


def _run_own(s):
    import avelang_amd as ave

    kind = s["case"]["kind"]
    if kind == "norm":
        return ave.layer_norm(s["x"], s["w"], s["b"], EPS)
    if kind == "norm_train":
        y = ave.layer_norm(s["x"], s["w"], s["b"], EPS)
        return (y.detach(),) + torch.autograd.grad(y, [s["x"], s["w"], s["b"]], s["dy"])
    if kind == "decode":
        return ave.fused_recurrent_linear_attn(s["q"], s["k"], s["v"], s["g"], initial_state=s["h0"],
                                               output_final_state=True, inplace_final_state=False)
    h0 = s.get("h0")
    if kind == "prefill":
        return ave.chunk_linear_attn(s["q"], s["k"], s["v"], s["g"], initial_state=h0,
                                     output_final_state=True, cu_seqlens=s.get("cu"))
    o, ht = ave.chunk_linear_attn(s["q"], s["k"], s["v"], s["g"], initial_state=h0,
                                  output_final_state=h0 is not None, cu_seqlens=s.get("cu"))
    if h0 is None:
        return (o.detach(),) + torch.autograd.grad(o, [s[n] for n in ("q", "k", "v", "g")], s["do"])
    return (o.detach(), ht.detach()) + torch.autograd.grad(
        [o, ht], [s[n] for n in ("q", "k", "v", "g", "h0")], [s["do"], s["dht"]])


# -------------------------------------------------------------- plain form ----
def _rows(s, x, heads, to):
    """[B, T, heads, D] as [N, Hv, Tpad, D] of type ``to``, zeros past a sequence's end."""
    case = s["case"]
    N, hv = case["seqs"], case["hv"]
    pad = -(-case["tokens"] // C) * C
    if case["packed"]:
        full = x.new_zeros(N * pad, heads, x.shape[-1], dtype=to)
        full[s["place"]] = x[0].to(to)
        full = full.reshape(N, pad, heads, -1)
    else:
        full = F.pad(x.to(to), (0, 0, 0, 0, 0, pad - case["tokens"]))
    return full.transpose(1, 2).repeat_interleave(hv // heads, dim=1)


def _back(s, x):
    """[N, H, Tpad, D] as the caller's [B, T, H, D]."""
    case = s["case"]
    x = x.transpose(1, 2)
    if case["packed"]:
        return x.reshape(-1, *x.shape[2:])[s["place"]][None]
    return x[:, :case["tokens"]]


def _decays(s):
    """Log-decays [N, Hv, Tpad] in 64 bits, 0 past a sequence's end."""
    g = s["g"]
    if g.dim() == 1:
        g = g.expand(*s["q"].shape[:2], g.shape[0])
    return _rows(s, g[..., None], s["case"]["hv"], torch.float64)[..., 0]


def _chunks(x, y, z, g, h):
    """o_i = sum_{j <= i} e^{G_i - G_j} (x_i . y_j) z_j + e^{G_i} x_i h, and the last state, for
    x, y [N, H, T, K], z [N, H, T, V], log-decays g [N, H, T] and h [N, H, K, V]."""
    N, H, T, K = x.shape
    n, V = T // C, z.shape[-1]
    x, y, z = (t.reshape(N, H, n, C, -1) for t in (x, y, z))
    G = g.reshape(N, H, n, C).cumsum(-1)
    last = G[..., -1]
    low = torch.ones(C, C, dtype=torch.bool, device=x.device).tril()
    gam = (G[..., :, None] - G[..., None, :]).masked_fill(~low, -math.inf).exp().float()
    o = (x @ y.transpose(-1, -2).contiguous() * gam) @ z
    del gam
    add = (y * (last[..., None] - G).exp().float()[..., None]).transpose(-1, -2).contiguous() @ z
    add = torch.cat([h[:, :, None], add], 2).reshape(N, H, n + 1, K * V)
    E = F.pad(last.cumsum(-1), (1, 0))
    low = torch.ones(n + 1, n + 1, dtype=torch.bool, device=x.device).tril()
    between = (E[..., :, None] - E[..., None, :]).masked_fill(~low, -math.inf).exp().float()
    state = (between @ add).reshape(N, H, n + 1, K, V)
    del add
    o += (x * G.exp().float()[..., None]) @ state[:, :, :n]
    return o.reshape(N, H, T, V), state[:, :, n].contiguous()


def _group_sum(case, x):
    """[N, Hv, T, D] summed over the v-heads of each qk-head."""
    N, hv, T, D = x.shape
    return x.reshape(N, case["hqk"], hv // case["hqk"], T, D).sum(2)


def _run_plain(s):
    case = s["case"]
    if case["kind"] in ("norm", "norm_train"):
        return _norm_plain(s)
    f32 = torch.float32
    bf = torch.bfloat16
    scale = case["k"] ** -0.5
    q, k = (_rows(s, s[n], case["hqk"], f32) for n in "qk")
    v = _rows(s, s["v"], case["hv"], f32)
    g = _decays(s)
    h0 = s.get("h0")
    if h0 is None:
        h0 = torch.zeros(case["seqs"], case["hv"], case["k"], case["v"], device=DEV)
    o, ht = _chunks(q * scale, k, v, g, h0)
    if case["kind"] != "train":
        return _back(s, o).to(bf), ht
    do = _rows(s, s["do"], case["hv"], f32)
    dht = s.get("dht", torch.zeros_like(h0))
    hT = h0.transpose(-1, -2).contiguous()
    dq = scale * _chunks(do, v, k, g, hT)[0]
    # the same sums backwards in time: a token's decay acts between it and the one before it
    back = F.pad(g.flip(-1)[..., :-1], (1, 0))
    kr, vr, qr, dr = (t.flip(2) for t in (k, v, q * scale, do))
    dv, dh = _chunks(kr, qr, dr, back, dht)
    dk = _chunks(vr, dr, qr, back, dht.transpose(-1, -2).contiguous())[0]
    dv, dk = dv.flip(2), dk.flip(2)
    # a sum of log-decays up to t multiplies what is read at t and divides what is written at t
    dG = (q * dq).sum(-1).double() - (k * dk).sum(-1).double()
    dg = dG.flip(-1).cumsum(-1).flip(-1) + (dht.double() * ht.double()).sum((-1, -2))[..., None]
    grads = (_back(s, _group_sum(case, dq)).to(bf), _back(s, _group_sum(case, dk)).to(bf),
             _back(s, dv).to(bf), _back(s, dg[..., None])[..., 0].to(bf))
    o = _back(s, o).to(bf)
    if "h0" not in s:
        return (o,) + grads
    return (o, ht) + grads + (dh * g[..., :1, None].exp().float(),)


def _norm_plain(s):
    x, w, b = s["x"].float(), s["w"].float(), s["b"].float()
    mid = x - x.mean(-1, keepdim=True)
    inv = torch.rsqrt((mid * mid).mean(-1, keepdim=True) + EPS)
    n = mid * inv
    y = (n * w + b).to(s["x"].dtype)
    if s["case"]["kind"] == "norm":
        return y
    dy = s["dy"].float()
    e = dy * w
    dx = inv * (e - e.mean(-1, keepdim=True) - n * (e * n).mean(-1, keepdim=True))
    return y, dx.to(s["x"].dtype), (dy * n).sum(0).to(s["w"].dtype), dy.sum(0).to(s["b"].dtype)


# ------------------------------------------------------------- what it costs ----
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def work(case):
    if case["kind"] in ("norm", "norm_train"):
        par = max(1, case["heads"]) * case["d"]
        n, xb, wb = case["rows"] * par, _BYTES[case["x_type"]], _BYTES[case["w_type"]]
        if case["kind"] == "norm":
            return dict(bytes=2 * n * xb + 2 * par * wb, flops=8.0 * n)
        # x and dy in, y and dx out; weight and bias in, their gradients out
        return dict(bytes=4 * n * xb + 4 * par * wb, flops=20.0 * n)
    N, hqk, hv, K, V = (case[x] for x in ("seqs", "hqk", "hv", "k", "v"))
    tok = sum(_lengths(case))
    qk, vo, state = 2 * tok * hqk * K * 2, tok * hv * V * 2, N * hv * K * V * 4
    g = 4 * hv if case["slopes"] else tok * hv * (2 if case["kind"] == "train" else 4)
    flops = 4.0 * K * V * tok * hv   # the rank-one update and S^T q of the recurrence
    if case["kind"] == "train":
        # q, k, v, g, do in; o and the gradients out; the states and their gradients
        return dict(bytes=2 * qk + 4 * vo + 2 * g + (4 * state if case["h0"] else 0), flops=3 * flops)
    return dict(bytes=qk + 2 * vo + g + state * (2 if case["h0"] else 1), flops=flops)


# ------------------------------------------------------------------ 64 bits ----
def _padded(case, x):
    """[B, T, H, D] as [T, N, H, D] in 64 bits, zeros past a sequence's end."""
    parts = x[0].double().split(_lengths(case)) if case["packed"] else x.double().unbind(0)
    return torch.nn.utils.rnn.pad_sequence(list(parts))


def _unpadded(case, x):
    if case["packed"]:
        return torch.cat([x[:n, i] for i, n in enumerate(_lengths(case))])[None]
    return x.transpose(0, 1)


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] in ("norm", "norm_train"):
            return _exact_norm(s)
        return _exact_steps(case, s)


def _exact_steps(case, s):
    rep = case["hv"] // case["hqk"]
    q, k = (_padded(case, s[n]).repeat_interleave(rep, 2) for n in "qk")
    v = _padded(case, s["v"])
    g = s["g"].double()
    if g.dim() == 1:
        g = g.expand(*s["q"].shape[:2], g.shape[0])
    g = _padded(case, g[..., None])   # [T, N, H, 1]
    scale = case["k"] ** -0.5
    T, N, H, K = q.shape
    V = v.shape[-1]
    S = s["h0"].double().clone() if "h0" in s else torch.zeros(N, H, K, V, dtype=torch.float64, device=DEV)
    a = g.exp()[..., None]
    o = torch.empty(T, N, H, V, dtype=torch.float64, device=DEV)
    train = case["kind"] == "train"
    if train:
        do, dq, dk, dv = _padded(case, s["do"]), torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    for t in range(T):
        S.mul_(a[t]).addcmul_(k[t][..., None], v[t][..., None, :])
        torch.matmul(q[t][..., None, :] * scale, S, out=o[t][..., None, :])
        if train:
            dq[t] = scale * (S * do[t][..., None, :]).sum(-1)
    if not train:
        return _unpadded(case, o), S
    ht = S
    dht = s["dht"].double() if "dht" in s else torch.zeros_like(S)
    D = dht.clone()
    for t in range(T - 1, -1, -1):
        D.addcmul_(scale * q[t][..., None], do[t][..., None, :])
        dk[t] = (D * v[t][..., None, :]).sum(-1)
        dv[t] = (D * k[t][..., None]).sum(-2)
        D.mul_(a[t])
    end = (dht * ht).sum((-1, -2))
    dg = ((q * dq).sum(-1) - (k * dk).sum(-1)).flip(0).cumsum(0).flip(0) + end
    dq, dk = (x.reshape(T, N, case["hqk"], rep, K).sum(3) for x in (dq, dk))
    out = [_unpadded(case, x) for x in (o, dq, dk, dv, dg)]
    return tuple(out) if "h0" not in s else (out[0], ht, *out[1:], D)


def _exact_norm(s):
    x, w, b = s["x"].double(), s["w"].double(), s["b"].double()
    var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
    xh = (x - mean) / torch.sqrt(var + EPS)
    y = xh * w + b
    if s["case"]["kind"] == "norm":
        return y
    dy = s["dy"].double()
    D = x.shape[-1]
    dxh = dy * w
    dx = (D * dxh - dxh.sum(-1, keepdim=True) - xh * (dxh * xh).sum(-1, keepdim=True)) / (D * torch.sqrt(var + EPS))
    return y, dx, (dy * xh).sum(0), dy.sum(0)
