"""Linear attention and layer norm on the CPU: the library's entry points and refusals, the
wrappers' refusals, workspace sizes, and the formulas that the kernels use against the token
recurrence, in 64 bits."""
import os
import re

import pytest
import torch

from avelang_amd import _native
from avelang_amd import linear_attention as L
from avelang_amd import norm as N
from oracle import linear_ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF = torch.bfloat16


def test_exports_are_the_headers():
    text = open(os.path.join(ROOT, "include", "gdn_linear.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    declared = set(re.findall(r"\b(gdn_\w+)\s*\(", text))
    assert declared == set(_native.EXPORTS_LINEAR)
    lib = _native.lib()
    assert all(hasattr(lib, n) for n in declared)


# Addresses that no call below reaches: every one is refused or has nothing to do.
P = [(i + 1) << 40 for i in range(16)]


def chunk(lib, **kw):
    a = dict(q=P[0], k=P[1], v=P[2], rows=(128, 128, 256), g=P[3], dt=0, head=0, h0=None, ht=None,
             o=P[4], cu=None, B=1, T=64, Hqk=2, Hv=4, K=64, V=64, N=1, states=None, ws=P[5],
             nbytes=1 << 40)
    a.update(kw)
    return lib.gdn_linear_chunk_fwd(a["q"], a["k"], a["v"], *a["rows"], a["g"], a["dt"], a["head"],
                                    a["h0"], a["ht"], a["o"], a["cu"], a["B"], a["T"], a["Hqk"],
                                    a["Hv"], a["K"], a["V"], a["N"], 0.1, a["states"], a["ws"],
                                    a["nbytes"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(K=96), -2), (dict(V=32), -2), (dict(Hv=3), -2), (dict(Hqk=0), -2), (dict(T=-1), -2),
    (dict(N=2), -3), (dict(cu=P[6], B=2, N=2), -3), (dict(q=None), -1), (dict(g=None), -1),
    (dict(o=None), -1), (dict(dt=7), -2), (dict(rows=(120, 128, 256)), -2),
    (dict(rows=(129, 128, 256)), -2), (dict(rows=(128, 128, 1 << 23)), -2), (dict(q=P[0] + 8), -2),
    (dict(o=P[0]), -5), (dict(o=P[4] + 2), -2), (dict(h0=P[7], ht=P[7] + 4096), -5),
    (dict(N=1 << 26, Hv=16, cu=P[6], rows=(128, 128, 1024)), -2),
    (dict(Hqk=1 << 15, Hv=1 << 15, rows=(1 << 21,) * 3), -2),
    (dict(T=70000, nbytes=16), -4), (dict(T=70000, ws=None), -4),
])
def test_chunk_refusals(kw, code):
    lib = _native.lib()
    assert chunk(lib, **kw) == code
    assert len(_native.last_error()) > 0


def test_nothing_to_do():
    lib = _native.lib()
    assert chunk(lib, T=0) == 0
    assert chunk(lib, B=0, N=0) == 0
    assert lib.gdn_layer_norm_fwd(None, None, None, None, None, 0, 1, 8, 1e-5, 0, 0, None) == 0
    assert lib.gdn_layer_norm_bwd(None, None, None, None, None, None, None, 0, 1, 8, 0, 0, None, 0,
                                  None) == 0


def test_backward_and_decode_refusals():
    lib = _native.lib()

    def bwd(dO=P[6], states=P[7], dg=P[11], nbytes=1 << 40, T=64, dq=P[8]):
        return lib.gdn_linear_chunk_bwd(P[0], P[1], P[2], 128, 128, 256, P[3], 0, 0, dO, None, states,
                                        dq, P[9], P[10], dg, None, None, 1, T, 2, 4, 64, 64, 1, 0.1,
                                        P[12], nbytes, None)
    assert bwd(dO=None) == -1 and bwd(states=None) == -1 and bwd(dg=None) == -1
    assert bwd(nbytes=8) == -4 and bwd(dq=P[8] + 4) == -2 and bwd(dO=P[6] + 2) == -2

    def rec(slots=1, idx=None, h0=P[4], ht=P[4], o=P[5], rows=(128, 128, 256)):
        return lib.gdn_linear_recurrent_fwd(P[0], P[1], P[2], *rows, P[3], 0, 0, h0, ht, o, None, idx,
                                            1, 1, 2, 4, 64, 64, 1, slots, 0.1, None)
    assert rec(slots=2) == -2 and rec(idx=P[6], slots=-1) == -2
    assert rec(idx=P[6], slots=4, ht=P[4] + 64) == -5 and rec(ht=P[4] + 64) == -5
    assert rec(o=None) == -1 and rec(o=P[5] + 2) == -2 and rec(rows=(8, 128, 256)) == -2


def test_norm_refusals():
    lib = _native.lib()

    def fwd(x=P[0], y=P[1], rows=4, heads=1, D=8, dt=0, wdt=0):
        return lib.gdn_layer_norm_fwd(x, None, None, y, None, rows, heads, D, 1e-5, dt, wdt, None)
    assert fwd(x=None) == -1 and fwd(y=None) == -1
    for kw in (dict(rows=-1), dict(heads=0), dict(D=0), dict(dt=3), dict(wdt=9), dict(rows=1 << 31),
               dict(heads=1 << 20, D=1 << 20)):
        assert fwd(**kw) == -2

    def bwd(stats=P[2], dw=P[5], nbytes=1 << 40):
        return lib.gdn_layer_norm_bwd(P[0], None, P[1], stats, P[3], dw, None, 4, 1, 8, 0, 0, P[6],
                                      nbytes, None)
    assert bwd(stats=None) == -1 and bwd(nbytes=8) == -4


def test_workspace_sizes():
    f = L.linear_attn_workspace_bytes
    assert f(1, 64, 2, 4, 64, 64, 1, False) == 0            # one walk, nothing kept
    assert f(1, 8192, 16, 32, 128, 128, 1, False) > 0
    assert f(1, 64, 2, 4, 64, 64, 1, True) > 0              # the table
    # a backward of an odd number of v-heads per qk-head keeps a part for each
    one = f(1, 4096, 4, 4, 64, 64, 1, False, backward=True)
    three = f(1, 4096, 4, 12, 64, 64, 1, False, backward=True)
    assert three - one > 4096 * 12 * 64 * 8 * 0.9
    assert f(1, 64, 0, 4, 64, 64, 1, False) == 0            # no such problem
    lib = _native.lib()
    assert lib.gdn_linear_states_bytes(1, 130, 4, 128, 64, 1, 0) == 3 * 4 * 128 * 64 * 2
    assert lib.gdn_linear_states_bytes(1, 130, 4, 128, 64, 3, 1) == 5 * 4 * 128 * 64 * 2
    assert lib.gdn_layer_norm_bwd_workspace_bytes(5, 1, 33, 0) >= 2 * 33 * 4


def _qkvg(dtype=BF, **kw):
    s = dict(q=(1, 8, 2, 64), k=(1, 8, 2, 64), v=(1, 8, 4, 64), g=(1, 8, 4))
    s.update(kw)
    return tuple(torch.zeros(s[n], dtype=dtype if n != "g" else torch.float32) for n in "qkvg")


@pytest.mark.parametrize("op", [L.chunk_linear_attn, L.fused_recurrent_linear_attn,
                                L.chunk_linear_attn_fwd_save])
def test_wrapper_refusals(op):
    bad = [
        (_qkvg(torch.float16), "bfloat16"), (_qkvg(k=(1, 8, 3, 64)), "k must have shape"),
        (_qkvg(v=(1, 7, 4, 64)), "v must have shape"), (_qkvg(v=(1, 8, 3, 64)), "multiple"),
        (_qkvg(q=(1, 8, 2, 32), k=(1, 8, 2, 32)), "head sizes"), (_qkvg(g=(1, 8, 2)), "g must have"),
        (_qkvg(q=(8, 2, 64)), "4-D"), (_qkvg(), "ROCm"), (_qkvg(g=(4,)), "ROCm"),
    ]
    for args, match in bad:
        with pytest.raises(ValueError, match=match):
            op(*args)
    q, k, v, g = _qkvg()
    with pytest.raises(ValueError, match="floating point"):
        op(q, k, v, g.long())
    with pytest.raises(ValueError, match="torch.Tensor"):
        op(None, k, v, g)
    with pytest.raises(ValueError, match="not supported when gradients"):
        L.chunk_linear_attn(q.requires_grad_(), k, v, g, out=v)


def test_norm_wrapper_refusals():
    x, w = torch.zeros(4, 3, 8), torch.zeros(8)
    for args, match in [((None,), "must be a tensor"), ((torch.zeros(4, 0),), "last axis"),
                        ((x.long(),), "float32, bfloat16"), ((x, w), "ROCm")]:
        with pytest.raises(ValueError, match=match):
            N.layer_norm(*args)
    with pytest.raises(ValueError, match="not supported when gradients"):
        N.layer_norm(x.requires_grad_(), w, w, out=x)


# ------------------------------------------------------------------ formulas ----
def _case(T=150, K=5, V=3, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen, dtype=torch.float64)  # noqa: E731
    return r(1, T, 1, K), r(1, T, 1, K), r(1, T, 1, V), -torch.exp(r(1, T, 1)), r(1, 1, K, V), r(1, T, 1, V), r(1, 1, K, V)


def _chunked(q, k, v, g, h0, do, dht, C=64):
    """o, ht and the gradients as the kernels form them, one head."""
    q, k, v, g, do = (x[0, :, 0] for x in (q, k, v, g, do))
    T, K = q.shape
    s = K ** -0.5
    S, o, starts = h0[0, 0], [], []
    spans = [(a, min(a + C, T)) for a in range(0, T, C)]

    def parts(a, b):
        G = g[a:b].cumsum(0)
        R = G[-1] - G
        gam = s * torch.exp(G[:, None] - G[None]).tril()
        return G, R, gam
    for a, b in spans:
        G, R, gam = parts(a, b)
        Pm = gam * (q[a:b] @ k[a:b].T)
        starts.append(S)
        o.append(Pm @ v[a:b] + s * G.exp()[:, None] * (q[a:b] @ S))
        S = G[-1].exp() * S + k[a:b].T @ (R.exp()[:, None] * v[a:b])
    D = dht[0, 0]
    dq, dk, dv, dg = (torch.empty_like(x) for x in (q, k, v, g))
    for (a, b), S0 in reversed(list(zip(spans, starts))):
        G, R, gam = parts(a, b)
        raw = do[a:b] @ v[a:b].T
        Pm, dP = gam * (q[a:b] @ k[a:b].T), gam * raw
        iq = s * G.exp()[:, None] * (do[a:b] @ S0.T)
        ik = R.exp()[:, None] * (v[a:b] @ D.T)
        dv[a:b] = Pm.T @ do[a:b] + R.exp()[:, None] * (k[a:b] @ D)
        dk[a:b], dq[a:b] = dP.T @ q[a:b] + ik, dP @ k[a:b] + iq
        M = Pm * raw
        x = (q[a:b] * iq).sum(1) + M.sum(1) - M.sum(0)
        y = (k[a:b] * ik).sum(1)
        dg[a:b] = G[-1].exp() * (S0 * D).sum() + x.flip(0).cumsum(0).flip(0) + y.cumsum(0) - y
        D = G[-1].exp() * D + q[a:b].T @ (s * G.exp()[:, None] * do[a:b])
    return torch.cat(o), S, dq, dk, dv, dg, D


def test_chunked_formulas_are_the_recurrence():
    q, k, v, g, h0, do, dht = _case()
    leaves = [x.clone().requires_grad_() for x in (q, k, v, g, h0)]
    o, ht = linear_ref.linear_attn(*leaves[:4], h0=leaves[4])
    want = torch.autograd.grad([o, ht], leaves, [do, dht])
    got = _chunked(q, k, v, g, h0, do, dht)
    # (64 bits throughout: a few thousand roundings of 2^-53)
    for x, ref in zip(got, (o[0, :, 0], ht[0, 0]) + tuple(w[0, :, 0] for w in want[:4]) + (want[4][0, 0],)):
        assert (x - ref).abs().max() <= 1e-11 * (1 + ref.abs().max())


def test_gradients_against_differences():
    """The oracle's gradients against central differences along random directions: an error of the
    third derivative's size times h^2 and of 2^-53 / h, under 1e-6 of the result at h = 1e-5."""
    q, k, v, g, h0, do, dht = _case(T=40, seed=3)
    xs = [q, k, v, g, h0]

    def f(vals):
        o, ht = linear_ref.linear_attn(*vals[:4], h0=vals[4])
        return ((o * do).sum() + (ht * dht).sum()).item()
    got = _chunked(*xs, do, dht)[2:]
    gen = torch.Generator().manual_seed(1)
    for i, x in enumerate(xs):
        d = torch.randn(x.shape, generator=gen, dtype=torch.float64)
        at = lambda e: [y + e * d if j == i else y for j, y in enumerate(xs)]  # noqa: E731
        num = (f(at(1e-5)) - f(at(-1e-5))) / 2e-5
        grad = got[i].reshape(x.shape)
        assert abs(num - (grad * d).sum().item()) <= 1e-6 * (grad.norm() * d.norm()).item()


def test_layer_norm_definition():
    x = torch.randn(7, 3, 20, dtype=torch.float64) * 3 + 1
    w, b = torch.randn(3, 20, dtype=torch.float64), torch.randn(3, 20, dtype=torch.float64)
    y = linear_ref.layer_norm(x)
    assert y.mean(-1).abs().max() < 1e-14
    ref = torch.nn.functional.layer_norm(x, (20,), eps=1e-5) * w + b
    assert (linear_ref.layer_norm(x, w, b) - ref).abs().max() < 1e-13
