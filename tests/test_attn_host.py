"""RMS norm, rotary positions, the paged cache and attention over it on the CPU: the library's entry
points, their refusals (before anything is enqueued) and the sizes of their workspaces."""
import math
import os
import re

import pytest
import torch

import avelang_amd as ave
from avelang_amd import _native

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32, BF, F16, E4M3, I8 = range(5)
# Addresses that no call below reaches: every one is refused or has nothing to do.
P = [(i + 1) << 40 for i in range(16)]


def test_exports_are_the_headers():
    text = open(os.path.join(ROOT, "include", "gdn_attn.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    declared = set(re.findall(r"\b(gdn_\w+)\s*\(", text))
    assert declared == set(_native.EXPORTS_ATTN)
    lib = _native.lib()
    assert all(hasattr(lib, n) for n in declared)


# ------------------------------------------------------------------ norms ----
def rms(x=P[0], res=P[1], w=P[2], y=P[3], h=P[4], scale=None, rows=4, D=64, dt=BF, rt=BF, wt=F32,
        out=BF):
    return _native.lib().gdn_rms_norm_fwd(x, res, w, y, h, scale, rows, D, 1e-6, 0.0, dt, rt, wt, out, None)


@pytest.mark.parametrize("kw,code", [
    (dict(rows=-1), -2), (dict(D=0), -2), (dict(dt=3), -2), (dict(wt=7), -2), (dict(rt=F16), -2),
    (dict(out=F16), -2), (dict(out=5), -2), (dict(rows=1 << 31), -2), (dict(D=(1 << 28) + 1), -2),
    (dict(rows=1 << 24, D=40000), -2), (dict(rows=1 << 29, D=8), -2),
    (dict(x=None), -1), (dict(y=None), -1), (dict(h=None), -1), (dict(out=E4M3), -1), (dict(out=I8), -1),
    (dict(y=P[0] + 2), -5), (dict(y=P[1] + 64), -5), (dict(h=P[3]), -5), (dict(h=P[0] + 8), -5),
    (dict(h=P[1] - 8), -5), (dict(out=E4M3, scale=P[6], y=P[0]), -5), (dict(rt=F32, h=P[0]), -5),
    (dict(rt=F32, y=P[1]), -5),
])
def test_rms_refusals(kw, code):
    assert rms(**kw) == code and len(_native.last_error()) > 0


def test_rms_backward_refusals():
    def bwd(h=P[0], dy=P[1], dh=P[2], dx=P[4], dr=None, dw=P[6], rows=4, D=64, dt=BF, ht=BF, wt=F32,
            ws=P[7], nbytes=1 << 40):
        return _native.lib().gdn_rms_norm_bwd(h, P[8], dy, dh, dx, dr, dw, rows, D, 1e-6, 0.0, dt, ht, wt,
                                              ws, nbytes, None)
    for kw in (dict(h=None), dict(dy=None), dict(dx=None)):
        assert bwd(**kw) == -1
    for kw in (dict(dx=P[0]), dict(dx=P[1] + 2), dict(dx=P[2]), dict(dr=P[4] + 4), dict(dr=P[0], ht=F32)):
        assert bwd(**kw) == -5
    assert bwd(rows=400, nbytes=8) == -4 and bwd(rows=400, ws=None) == -4
    assert bwd(dt=4) == -2 and bwd(ht=F16) == -2 and bwd(rows=-1) == -2 and bwd(D=1 << 28) == -2
    assert bwd(rows=1 << 24, D=40000, dw=None) == -2
    assert bwd(rows=0, dw=None) == 0 and rms(rows=0, x=None, y=None) == 0
    f = _native.lib().gdn_rms_norm_bwd_workspace_bytes
    assert f(0, 64, BF) == f(1, 64, BF) == 0 < f(400, 64, BF) <= f(4096, 64, BF) and f(5, 64, 9) == 0


# ----------------------------------------------------------------- rotary ----
def rotary(q=P[0], k=P[1], qo=P[2], ko=P[3], strides=(512, 256, 64, 256, 128, 64, 512, 256, 64, 256, 128, 64), B=1,
           T=2, Hq=4, Hk=2, D=64, pos=P[4], freq=P[5], R=64, dt=BF):
    from avelang_amd.rotary import _STRIDES
    return _native.lib().gdn_rotary(q, k, qo, ko, strides and _STRIDES(*strides), B, T, Hq, Hk, D, pos, 1, 0, freq,
                                    R, 1.0, 0, 0, dt, None)


@pytest.mark.parametrize("kw,code", [
    (dict(B=-1), -2), (dict(T=-1), -2), (dict(Hq=0), -2), (dict(Hk=-1), -2), (dict(D=63), -2), (dict(D=0), -2),
    (dict(D=514), -2), (dict(R=0), -2), (dict(R=66), -2), (dict(R=7), -2), (dict(dt=3), -2),
    (dict(Hq=(1 << 20) + 1), -2), (dict(B=1 << 16, T=1 << 16), -2), (dict(q=None), -1), (dict(qo=None), -1),
    (dict(ko=None), -1), (dict(pos=None), -1), (dict(freq=None), -1), (dict(strides=None), -1),
    (dict(strides=(-1,) * 12), -2), (dict(qo=P[0]), -5), (dict(qo=P[0], ko=P[1], strides=(512, 256, 64, 256, 128, 64,
                                                                                         512, 128, 64, 256, 128, 64)), -5),
    (dict(ko=P[2]), -5), (dict(qo=P[0] + 64), -5), (dict(ko=P[0] + 64), -5), (dict(qo=P[1]), -5),
])
def test_rotary_refusals(kw, code):
    assert rotary(**kw) == code and len(_native.last_error()) > 0


def test_rotary_nothing_and_frequencies():
    assert rotary(T=0, q=None, pos=None) == 0 and rotary(B=0) == 0
    f, m = ave.rotary_frequencies(8, 100.0)
    assert m == 1.0 and f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64))
    g, m = ave.rotary_frequencies(8, 100.0, factor=4.0)
    assert m == 1.0 and torch.equal(g, f / 4)
    g, m = ave.rotary_frequencies(64, factor=8.0, original=4096)
    f, _ = ave.rotary_frequencies(64)
    turns = 4096 * f / (2 * math.pi)
    assert m == 0.1 * math.log(8) + 1
    assert torch.equal(g[turns >= 32], f[turns >= 32]) and torch.equal(g[turns <= 1], f[turns <= 1] / 8)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and (g[mid] < f[mid]).all() and (g[mid] > f[mid] / 8).all()
    for kw in (dict(dim=7), dict(dim=0), dict(dim=8, base=0.0), dict(dim=8, factor=0.0), dict(dim=8, original=-1),
               dict(dim=8, factor=2.0, original=64, slow=3.0, fast=3.0)):
        with pytest.raises(ValueError):
            ave.rotary_frequencies(**kw)


# ------------------------------------------------------------------ cache ----
def write(k=P[0], v=P[1], st=(128, 64, 128, 64), slots=P[2], kc=P[3], vc=P[4], ks=P[5], vs=P[6], T=3, H=2, D=64,
          pages=4, page=16, dt=BF, ct=E4M3):
    return _native.lib().gdn_paged_write(k, v, *st, slots, 0, kc, vc, ks, vs, T, H, D, pages, page, dt, ct, None)


def read(k=P[0], v=P[1], slots=P[2], kc=P[3], vc=P[4], ks=P[5], vs=P[6], T=3, H=2, D=64, pages=4, page=16, dt=BF,
         ct=E4M3):
    return _native.lib().gdn_paged_read(kc, vc, ks, vs, slots, 0, k, v, T, H, D, pages, page, dt, ct, None)


@pytest.mark.parametrize("call", [write, read])
@pytest.mark.parametrize("kw,code", [
    (dict(T=-1), -2), (dict(H=0), -2), (dict(H=1 << 16), -2), (dict(D=96), -2), (dict(pages=-1), -2),
    (dict(page=0), -2), (dict(page=1 << 21), -2), (dict(ct=F32), -2), (dict(ct=9), -2), (dict(dt=F32), -2),
    (dict(dt=F16, ct=BF), -2), (dict(k=None), -1), (dict(v=None), -1), (dict(slots=None), -1), (dict(kc=None), -1),
    (dict(vs=None), -1), (dict(kc=P[3] + 8), -2),
])
def test_cache_refusals(call, kw, code):
    assert call(**kw) == code and len(_native.last_error()) > 0


def test_cache_nothing():
    assert write(st=(-1, 64, 128, 64)) == -2
    assert write(T=0, k=None, slots=None) == 0 and read(T=0, k=None) == 0 and write(pages=0, kc=None) == 0


def test_cache_object_refusals():
    bf = torch.zeros(2, 3, 16, 64, dtype=torch.bfloat16)
    i8, s = torch.zeros(2, 3, 16, 64, dtype=torch.int8), torch.zeros(2, 3, 16)
    c = ave.PagedKVCache(i8, i8.clone(), s, s.clone())
    assert c.sizes == (3, 64, 2, 16)
    odd = torch.zeros(2 * 3 * 16 * 64 + 1, dtype=torch.bfloat16)[1:].view(2, 3, 16, 64)
    for args in ((bf, bf[:1]), (bf, bf.half()), (bf.float(), bf.float()), (bf[0], bf[0]), (bf[..., :32], bf[..., :32]),
                 (bf.transpose(1, 2), bf.transpose(1, 2)), (bf, bf, s, s), (i8, i8), (i8, i8, s), (i8, i8, s, s[:1]),
                 (i8, i8, s, s.double()), (odd, bf), (bf, odd), (None, bf), (bf[:, :0], bf[:, :0])):
        with pytest.raises(ValueError, match="PagedKVCache"):
            ave.PagedKVCache(*args)
    # nothing of these runs on the CPU
    row = torch.zeros(1, 3, 64, dtype=torch.bfloat16)
    for call in (lambda: ave.paged_cache_write(c, row, row, torch.zeros(1, dtype=torch.int32)),
                 lambda: ave.paged_cache_read(c, torch.zeros(1, dtype=torch.int32)),
                 lambda: ave.paged_attention(row[None], c, torch.zeros(1, 1, dtype=torch.int32),
                                             torch.zeros(1, dtype=torch.int32)),
                 lambda: ave.rms_norm(row), lambda: ave.rms_norm_quant(row),
                 lambda: ave.rotary_embedding(row, None, torch.zeros(1, dtype=torch.int32), torch.ones(32))):
        with pytest.raises(ValueError, match="ROCm"):
            call()


# -------------------------------------------------------------- attention ----
def attn(q=P[0], st=(512, 512, 128), kc=P[1], vc=P[2], ks=P[3], vs=P[4], table=P[5], row=8, lens=P[6], o=P[7], N=2,
         L=1, Hq=4, H=2, D=128, pages=9, page=16, most=100, window=0, dt=BF, ct=E4M3, ws=P[9], nbytes=1 << 40):
    return _native.lib().gdn_paged_attn_fwd(q, *st, kc, vc, ks, vs, table, row, lens, o, None, N, L, Hq, H, D, pages,
                                            page, most, window, 0.1, dt, ct, ws, nbytes, None)


@pytest.mark.parametrize("kw,code", [
    (dict(N=-1), -2), (dict(L=0), -2), (dict(Hq=0), -2), (dict(H=0), -2), (dict(Hq=3), -2), (dict(D=80), -2),
    (dict(pages=0), -2), (dict(page=24), -2), (dict(page=0), -2), (dict(most=-1), -2), (dict(most=129), -2),
    (dict(most=(1 << 30) + 1), -2), (dict(row=6), -2), (dict(row=-1), -2), (dict(window=-1), -2), (dict(dt=F32), -2),
    (dict(ct=F32), -2), (dict(ct=F16), -2), (dict(L=1 << 20), -2), (dict(N=1 << 20, most=1 << 20, row=1 << 16), -2),
    (dict(st=(512, 512, 64 + 4)), -2), (dict(st=(-8, 512, 128)), -2), (dict(q=P[0] + 8), -2), (dict(o=P[7] + 2), -2),
    (dict(ks=P[3] + 4), -2), (dict(vc=P[2] + 8), -2), (dict(q=None), -1), (dict(o=None), -1), (dict(lens=None), -1),
    (dict(table=None), -1), (dict(kc=None), -1), (dict(ks=None), -1), (dict(o=P[0] + 16), -5), (dict(nbytes=64), -4),
    (dict(ws=None), -4), (dict(ws=P[9] + 4), -4),
])
def test_attention_refusals(kw, code):
    assert attn(**kw) == code and len(_native.last_error()) > 0


def test_attention_sizes():
    assert attn(N=0, q=None, o=None, ws=None, nbytes=0) == 0
    f = ave.paged_attention_workspace_bytes
    assert f(0, 1, 4, 2, 128, 100) == 0 and f(1, 1, 3, 2, 128, 100) == 0
    last = 0
    for n in (1, 100, 1000, 10000, 100000):   # one for the largest holds every smaller call
        assert f(3, 2, 8, 2, 128, n) >= last
        last = f(3, 2, 8, 2, 128, n)
    last = 0
    for n in (1, 2, 30, 31, 500, 4000):
        assert f(n, 1, 8, 2, 256, 5000) >= last
        last = f(n, 1, 8, 2, 256, 5000)
