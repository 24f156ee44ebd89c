"""Rotary positions against float64.

Bounds: a turn is rounded to fp32 once it is within half a turn (2^-25, 2^-22.3 of an angle), sine and
cosine to 2^-23; two products and a sum: 2^-21 of |a| + |b|, and half a step of the type.
"""
import pytest
import torch

import avelang_amd as ave
from oracle import attn_ref as R

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
FAR = torch.tensor([0, 1, 17, 4095, 131071, 1_000_003, 2 ** 31 - 1, -5], dtype=torch.int64)


def _bound(x, freq, mag, near, want, t):
    r = 2 * freq.numel()
    x = x.double().abs()
    a, b = (x[..., :r:2], x[..., 1:r:2]) if near else (x[..., :r // 2], x[..., r // 2:r])
    s = mag * (a + b)
    s = torch.stack([s, s], -1).flatten(-2) if near else torch.cat([s, s], -1)
    return torch.cat([s, torch.zeros_like(x[..., r:])], -1) * 2 ** -21 + want.abs() * torch.finfo(t).eps / 2 + 1e-9


def _case(B, T, hq, hk, D, r, t, seed=0):
    gen = torch.Generator().manual_seed(seed + D + r)
    q, k = (torch.randn((B, T, h, D), generator=gen).to(t) for h in (hq, hk))
    freq, mag = ave.rotary_frequencies(r, factor=8.0, original=4096)
    return q, k, freq, mag


@pytest.mark.parametrize("near", [False, True])
@pytest.mark.parametrize("t", [BF16, F16, F32])
@pytest.mark.parametrize("B,T,hq,hk,D,r", [(1, 1, 16, 2, 256, 64), (2, 5, 3, 1, 128, 128), (1, 8, 4, 4, 64, 32),
                                           (3, 7, 1, 1, 2, 2), (1, 3, 5, 2, 96, 20), (2, 4, 2, 1, 128, 68),
                                           (1, 2, 2, 1, 70, 6), (1, 6, 2, 2, 512, 512), (1, 300, 8, 2, 64, 64),
                                           (2, 1500, 6, 2, 128, 128), (1, 4000, 8, 1, 32, 16)])
def test_forward(rocm_device, B, T, hq, hk, D, r, t, near):
    q, k, freq, mag = _case(B, T, hq, hk, D, r, t)
    pos = FAR.repeat(-(-B * T // 8))[:B * T].view(B, T)
    got = ave.rotary_embedding(q.cuda(), k.cuda(), pos.cuda(), freq.cuda(), magnitude=mag, interleaved=near)
    for x, y in zip((q, k), got):
        want = R.rotary(x, pos, freq, mag, near)
        assert y.dtype == t and y.is_contiguous()
        assert ((y.cpu().double() - want).abs() <= _bound(x, freq, mag, near, want, t)).all()
        assert torch.equal(y.cpu()[..., r:], x[..., r:])


@pytest.mark.parametrize("near", [False, True])
@pytest.mark.parametrize("D,r", [(128, 128), (256, 64), (96, 20)])
def test_layouts(rocm_device, D, r, near):
    """Column slices, heads ahead of tokens, 3-D, int32 positions shared by the batch, in place."""
    B, T, hq, hk = 2, 9, 4, 2
    freq, mag = (x.cuda() if torch.is_tensor(x) else x for x in ave.rotary_frequencies(r))
    y = torch.randn(B, T, (hq + 2 * hk) * D + 6, device="cuda").bfloat16()[..., 3:-3]
    q, k, _ = (x.unflatten(-1, (-1, D)) for x in y.split([hq * D, hk * D, hk * D], -1))
    pos = torch.arange(T, device="cuda", dtype=torch.int32) * 1000
    call = lambda q, k, p, **kw: ave.rotary_embedding(q, k, p, freq, interleaved=near, **kw)  # noqa: E731
    want = call(q.contiguous(), k.contiguous(), pos.long()[None].expand(B, T))
    for a, b in zip(call(q, k, pos), want):
        assert torch.equal(a, b)
    qt, kt = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k))
    assert all(torch.equal(a, b) for a, b in zip(call(qt, kt, pos), want))
    for i in range(B):
        got = call(q[i], k[i], pos)
        assert got[0].dim() == 3 and all(torch.equal(a, b[i]) for a, b in zip(got, want))
    assert torch.equal(call(q, None, pos), want[0])
    rest = y.clone()
    got = call(q, k, pos, inplace=True)
    assert got[0] is q and torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(y[..., (hq + hk) * D:], rest[..., (hq + hk) * D:])
    qt2 = qt.clone(memory_format=torch.preserve_format)
    assert torch.equal(call(qt2, None, pos, inplace=True), want[0])


@pytest.mark.parametrize("near", [False, True])
@pytest.mark.parametrize("t", [BF16, F32])
def test_gradients(rocm_device, near, t):
    q, k, freq, mag = _case(2, 11, 4, 2, 128, 96, t)
    pos = FAR.repeat(3)[:22].view(2, 11)
    gen = torch.Generator().manual_seed(1)
    dq, dk = (torch.randn(x.shape, generator=gen).to(t) for x in (q, k))
    qd, kd = q.cuda().requires_grad_(), k.cuda().requires_grad_()
    out = ave.rotary_embedding(qd, kd, pos.cuda(), freq.cuda(), magnitude=mag, interleaved=near)
    got = torch.autograd.grad(out, [qd, kd], [dq.cuda(), dk.cuda()], retain_graph=True)
    for x, g, d in ((q, got[0], dq), (k, got[1], dk)):
        xd = x.double().requires_grad_()
        want, = torch.autograd.grad(R.rotary(xd, pos, freq, mag, near), [xd], d.double())
        assert g.dtype == t and ((g.cpu().double() - want).abs() <= _bound(d, freq, mag, near, want, t)).all()
    # one output unused, strided gradients
    only, = torch.autograd.grad(out[1], [kd], dk.cuda().transpose(1, 2).contiguous().transpose(1, 2), retain_graph=True)
    assert torch.equal(only, got[1])
    assert torch.autograd.grad(out[1].sum(), [qd], allow_unused=True, retain_graph=True)[0] is None
    # the operator is linear: differences of any size are its gradient's, but for rounding
    if t is F32:
        with torch.no_grad():
            e = torch.randn(q.shape, generator=gen).cuda()
            f = lambda x: (ave.rotary_embedding(x, None, pos.cuda(), freq.cuda(), magnitude=mag, interleaved=near).double() * dq.cuda().double()).sum()  # noqa: E731
            diff = (f(qd + e) - f(qd - e)) / 2
            assert (diff - (got[0].double() * e.double()).sum()).abs() <= 2 ** -20 * (dq.cuda().abs() * e.abs()).double().sum() * 8


def test_empty(rocm_device):
    freq = ave.rotary_frequencies(64, device="cuda")[0]
    q = torch.empty(2, 0, 4, 64, device="cuda", requires_grad=True)
    y = ave.rotary_embedding(q, None, torch.empty(0, device="cuda", dtype=torch.int64), freq)
    assert y.shape == q.shape and torch.autograd.grad(y.sum(), [q])[0].shape == q.shape
    with pytest.raises(ValueError, match="inplace"):
        ave.rotary_embedding(q, None, torch.empty(0, device="cuda", dtype=torch.int64), freq, inplace=True)


def test_in_place_is_seen(rocm_device):
    """Autograd refuses a backward that needs a tensor that was turned in place since."""
    w = torch.randn(4, 1, 64, device=rocm_device, requires_grad=True)
    x = torch.randn(4, 1, 64, device=rocm_device)
    y = (w * x).sum()
    pos, f = torch.arange(4, device=rocm_device), torch.ones(32, dtype=torch.float64, device=rocm_device)
    ave.rotary_embedding(x, None, pos, f, inplace=True)
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()
    with torch.inference_mode():
        z = torch.randn(4, 1, 64, device=rocm_device)
        want = ave.rotary_embedding(z, None, pos, f)
        assert torch.equal(ave.rotary_embedding(z, None, pos, f, inplace=True), want)
