"""RMS norm with the residual's addition, in its own type, in 8 bits and in training, against float64.

Bounds: a row's sum of squares goes through at most 48 fp32 additions a value (32 in a lane, 16 between
lanes), the root halves its error and a handful of roundings follow: 2^-18 of a result, and half a step of
its type.  Gradients: 2^-17 of the terms that are added.
"""
import pytest
import torch

import avelang_amd as ave
from oracle import attn_ref as R

pytestmark = pytest.mark.gpu
F32, BF16, F16, E4M3, I8 = torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.int8
TYPES = [(BF16, BF16), (BF16, F32), (BF16, None), (F16, F16), (F16, None), (F32, F32), (F32, None)]
ROWS_D = [(1, 1), (3, 7), (5, 64), (2, 127), (9, 130), (1, 513), (33, 1024), (4, 1001), (3, 2048), (2, 2049),
          (3, 4100), (2, 8190), (2, 8193), (3, 20001)]


def _inputs(rows, D, xt, rt, wt, seed=0):
    gen = torch.Generator().manual_seed(seed + 7 * D + rows)
    r = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    x = (r(rows, D) * (0.2 + 3 * torch.rand((rows, 1), generator=gen))).to(xt)
    res = None if rt is None else (2 * r(rows, D)).to(rt)
    return x, res, (0.3 * r(D)).to(wt)


def _cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


def _half(t):
    return torch.finfo(t).eps / 2


def _least(t):
    """Half the step of t's subnormal values (fp16: 2^-25, as its values under 2^-14 lie 2^-24 apart)."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def _added(x, res):
    return x if res is None else (x.float() + res.float()).to(res.dtype)


@pytest.mark.parametrize("xt,rt", TYPES)
@pytest.mark.parametrize("rows,D", ROWS_D)
def test_forward(rocm_device, rows, D, xt, rt):
    wt = BF16 if D % 2 else F32
    x, res, w = _inputs(rows, D, xt, rt, wt)
    got = ave.rms_norm(*_cuda(x, w), residual=_cuda(res)[0], offset=1.0)
    h = _added(x, res)
    if rt is not None:
        got, gh = got
        assert gh.dtype == rt and torch.equal(gh.cpu(), h)
    want, _ = R.rms_norm(h, w, offset=1.0)
    assert got.dtype == xt
    off = (got.cpu().double() - want).abs()
    assert (off <= want.abs() * (_half(xt) + 2 ** -18) + 2.0 ** -24).all(), off.max()


@pytest.mark.parametrize("xt,rt", TYPES)
@pytest.mark.parametrize("code", [E4M3, I8])
@pytest.mark.parametrize("rows,D", ROWS_D)
def test_eight_bits(rocm_device, rows, D, xt, rt, code):
    x, res, w = _inputs(rows, D, xt, rt, F32, seed=1)
    c, scale, *h = ave.rms_norm_quant(*_cuda(x, w), residual=_cuda(res)[0], dtype=code)
    assert c.dtype == code and scale.shape == (rows,) and len(h) == (rt is not None)
    y, _ = R.rms_norm(_added(x, res), w)
    most = y.abs().amax(-1)
    scale = scale.cpu().double()
    assert ((scale - most / R.MOST[code]).abs() <= scale * 2 ** -17).all()
    # half a step of the code, of a value that fp32 holds to 2^-17
    back = c.cpu().float().double() * scale[:, None]
    step = torch.maximum(y.abs() / 16, scale[:, None] * 2 ** -10) if code is E4M3 else scale[:, None] / 2
    assert ((back - y).abs() <= step * (1 + 2 ** -12) + most[:, None] * 2 ** -16).all()


@pytest.mark.parametrize("xt,rt", TYPES)
@pytest.mark.parametrize("rows,D", ROWS_D + [(700, 300), (2100, 64)])
def test_gradients(rocm_device, rows, D, xt, rt):
    wt = F16 if D % 2 else F32
    x, res, w = _inputs(rows, D, xt, rt, wt, seed=2)
    gen = torch.Generator().manual_seed(D)
    dy = torch.randn(rows, D, generator=gen).to(xt)
    leaves = [t.requires_grad_() for t in _cuda(x, w, res) if t is not None]
    dev = dict(zip("xwr", leaves))
    if rt is None:
        y, grads = ave.rms_norm(dev["x"], dev["w"], offset=0.5), [dy]
        dh, out = None, [y]
    else:
        dh = torch.randn(rows, D, generator=gen).to(rt)
        out, grads = ave.rms_norm(dev["x"], dev["w"], residual=dev["r"], offset=0.5), [dy, dh]
    got = torch.autograd.grad(out, leaves, _cuda(*grads))
    # the formula's gradients at the h that the forward holds
    h = _added(x, res).double().requires_grad_()
    wd = w.double().requires_grad_()
    y, _ = R.rms_norm(h, wd, offset=0.5)
    gh, gw = torch.autograd.grad(y, [h, wd], dy.double())
    gh = gh + (0 if dh is None else dh.double())
    with torch.no_grad():
        rstd = 1 / ((h * h).mean(-1, keepdim=True) + 1e-6).sqrt()
        hh, e = h * rstd, dy.double() * (wd + 0.5)
        terms = rstd * (e.abs() + hh.abs() * (e * hh).abs().mean(-1, keepdim=True)) + (0 if dh is None else dh.double().abs())
        sums = (dy.double() * hh).abs().sum(0)
    for g, t in ((got[0], xt),) + (((got[2], rt),) if rt is not None else ()):
        assert g.dtype == t
        assert ((g.cpu().double() - gh).abs() <= terms * 2 ** -17 + gh.abs() * _half(t) + _least(t) + 1e-12).all()
    assert got[1].dtype == wt
    # (a column's sum: rows of a group one after the other, at most 2100 / 1024 here, 512 groups in 32 steps)
    assert ((got[1].cpu().double() - gw).abs() <= sums * 2 ** -17 + gw.abs() * _half(wt) + 2.0 ** -25).all()


def test_gradients_are_differences(rocm_device):
    """Central differences of the fp32 forward along random directions."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    x, w, res, dy, dh = (torch.randn(s, generator=gen, device="cuda") for s in ((4, 96), (96,), (4, 96), (4, 96), (4, 96)))
    leaves = [t.requires_grad_() for t in (x, w, res)]
    got = torch.autograd.grad(ave.rms_norm(x, w, residual=res), leaves, [dy, dh])

    def value(x, w, res):
        y, h = ave.rms_norm(x, w, residual=res)
        return (y.double() * dy.double()).sum() + (h.double() * dh.double()).sum()
    with torch.no_grad():
        for i, g in enumerate(got):
            d = torch.randn(leaves[i].shape, generator=gen, device="cuda")
            e = 2.0 ** -8
            a = [t + e * d if j == i else t for j, t in enumerate(leaves)]
            b = [t - e * d if j == i else t for j, t in enumerate(leaves)]
            diff = (value(*a) - value(*b)) / (2 * e)
            # 768 values of size 1 held to 2^-22, over 2 e: 0.024; e^2 / 6 = 2.5e-6 of a third derivative
            # of a few hundred at most
            assert (diff - (g.double() * d.double()).sum()).abs() <= 0.03


def test_unused_outputs(rocm_device):
    x, w, res = (torch.randn(s, device="cuda", requires_grad=True) for s in ((3, 64), (64,), (3, 64)))
    y, h = ave.rms_norm(x.bfloat16(), w, residual=res)
    g = torch.autograd.grad(h.sum(), [x, w, res], retain_graph=True)
    assert torch.equal(g[0], torch.ones_like(x)) and not g[1].any() and torch.equal(g[2], torch.ones_like(x))
    gy = torch.autograd.grad(y.float().sum(), [x, res])
    assert torch.equal(gy[0], gy[1].bfloat16().float())
    with pytest.raises(ValueError, match="not supported when gradients"):
        ave.rms_norm(x, w, out=torch.empty_like(x))


def test_only_what_is_wanted(rocm_device):
    x = torch.randn(5, 96, device="cuda")
    w = torch.randn(96, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(ave.rms_norm(x, w).sum(), [w])
    x2 = x.clone().requires_grad_()
    y = ave.rms_norm(x2, w.detach())
    gx, = torch.autograd.grad(y.sum(), [x2])
    x3 = x.clone().requires_grad_()
    full = torch.autograd.grad(ave.rms_norm(x3, w).sum(), [x3, w])
    assert torch.equal(g, full[1]) and torch.equal(gx, full[0])


@pytest.mark.parametrize("D", [64, 1001, 4096, 20001])
def test_special_rows(rocm_device, D):
    """Zeros, tiny rows, infinities and NaN stay in their own rows."""
    x = torch.randn(6, D, device="cuda", generator=torch.Generator("cuda").manual_seed(D))
    x[1], x[2, D // 2], x[3, 0] = 0, torch.inf, torch.nan
    x[4] = 1e-38
    clean = ave.rms_norm(x[[0, 5]])
    y = ave.rms_norm(x)
    assert torch.equal(y[[0, 5]], clean) and not y[1].any() and y[3].isnan().all() and y[2, D // 2].isnan()
    assert y[4].isfinite().all()
    for code in (E4M3, I8):
        c, s = ave.rms_norm_quant(x, dtype=code)
        c0, s0 = ave.rms_norm_quant(x[[0, 5]], dtype=code)
        assert torch.equal(c[[0, 5]].view(I8), c0.view(I8)) and torch.equal(s[[0, 5]], s0)
        assert s[1] == 0 and not c[1].view(I8).any() and s[2].isnan() and s[3].isnan()
        assert s[4].isfinite() and c[4].float().isfinite().all()
    # a row under 2^-100: stored as if its largest value were that
    w = torch.full((D,), 2.0 ** -110, device="cuda")
    c, s = ave.rms_norm_quant(torch.ones(1, D, device="cuda"), w, eps=0.0)
    assert s[0] == 2.0 ** -100 / 448 and (c.float() == 0.4375).all()   # 448 / 1024


def test_in_place_and_out(rocm_device):
    for D in (130, 2048, 20001):
        x, res, w = _cuda(*_inputs(5, D, BF16, BF16, BF16))
        y, h = ave.rms_norm(x, w, residual=res)
        x1, r1 = x.clone(), res.clone()
        a, b = ave.rms_norm(x1, w, residual=r1, out=x1, residual_out=r1)
        assert a is x1 and b is r1 and torch.equal(a, y) and torch.equal(b, h)
        x1, out = x.clone(), torch.empty_like(x)
        a, b = ave.rms_norm(x1, w, residual=res, out=out, residual_out=x1)
        assert torch.equal(a, y) and torch.equal(b, h)
        r1 = res.clone()
        c, s, b = ave.rms_norm_quant(x, w, residual=r1, residual_out=r1)
        c2, s2, _ = ave.rms_norm_quant(x, w, residual=res)
        assert torch.equal(c.view(I8), c2.view(I8)) and torch.equal(s, s2) and torch.equal(r1, h)


def test_strides_offsets_and_empty(rocm_device):
    """Slices, transposes, rows at odd elements; no rows at all."""
    big = torch.randn(40, 4 * 130 + 1, device="cuda").bfloat16()
    w = torch.randn(130, device="cuda")
    for x in (big[:, 1:131], big[::3, 131:261], big[:, :520].view(40, 4, 130).transpose(0, 1),
              big.view(-1)[3:3 + 13 * 130].view(13, 130)):
        assert torch.equal(ave.rms_norm(x, w), ave.rms_norm(x.contiguous().clone(), w))
        c, s = ave.rms_norm_quant(x, w)
        assert s.shape == x.shape[:-1]
        assert torch.equal(c.view(I8), ave.rms_norm_quant(x.contiguous().clone(), w)[0].view(I8))
    e = torch.empty(0, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    y, h = ave.rms_norm(e, w, residual=e.detach())
    ge, gw = torch.autograd.grad([y, h], [e, w], [y.detach(), h.detach()])
    assert ge.shape == (0, 64) and not gw.any()
    assert ave.rms_norm_quant(e.detach())[1].shape == (0,)


def test_backward_takes_saved_tensors_as_they_come(rocm_device):
    x, w = torch.randn(6, 200, device="cuda", requires_grad=True), torch.randn(200, device="cuda", requires_grad=True)
    want = torch.autograd.grad(ave.rms_norm(x, w).sum(), [x, w])
    with torch.autograd.graph.save_on_cpu():
        y = ave.rms_norm(x, w)
    got = torch.autograd.grad(y.sum(), [x, w])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_same_bits_every_time(rocm_device):
    x, dy = (torch.randn(5000, 700, device="cuda").bfloat16() for _ in "xy")
    w = torch.randn(700, device="cuda")
    first = ave.rms_norm_bwd(x, w, dy)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(ave.rms_norm_bwd(x, w, dy), first))
    x.requires_grad_()
    w.requires_grad_()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(ave.rms_norm(x, w), [x, w], dy), first))


@pytest.mark.parametrize("of", ["x", "residual"])
def test_in_place_is_seen(rocm_device, of):
    """Autograd refuses a backward that needs a tensor that was written over since."""
    w = torch.randn(4, 64, device=rocm_device, requires_grad=True)
    x, r = torch.randn(4, 64, device=rocm_device), torch.randn(4, 64, device=rocm_device)
    y = (w * (x if of == "x" else r)).sum()
    if of == "x":
        ave.rms_norm(x, out=x)
    else:
        ave.rms_norm(x, residual=r, residual_out=r)
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()
    with torch.inference_mode():
        z = torch.randn(4, 64, device=rocm_device)
        want = ave.rms_norm(z)
        assert torch.equal(ave.rms_norm(z, out=z), want)


@pytest.mark.parametrize("t", [BF16, F32])
@pytest.mark.parametrize("D", [96, 250, 1000, 2500, 8000])
@pytest.mark.parametrize("rows", [1, 2, 3, 8, 9, 16, 17, 32, 33])
def test_few_rows_gradients(rocm_device, rows, D, t):
    """One workgroup's rows and one more: the weight's gradient with and without a second launch."""
    gen = torch.Generator().manual_seed(rows * D)
    x, dy = (torch.randn(rows, D, generator=gen).to(t) for _ in "xy")
    w = torch.randn(D, generator=gen).to(BF16 if rows % 2 else F32)
    dx, dw, _ = ave.rms_norm_bwd(x.cuda(), w.cuda(), dy.cuda(), eps=1e-5, offset=1.0)
    leaves = [v.double().requires_grad_() for v in (x, w)]
    h, weight = leaves
    y = h * (h.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * (weight + 1)
    want = torch.autograd.grad(y, leaves, dy.double())
    # sums in fp32: under (D / 64 + 16) steps of 2^-24 of the terms' sizes; rows up to 2^3 large
    eps = 2.0 ** -24 * (D / 64 + 32)
    ax = want[0].abs() * torch.finfo(t).eps / 2 + eps * 8 * (1 + want[0].abs().amax(-1, keepdim=True))
    xh = (h / (h.square().mean(-1, keepdim=True) + 1e-5).sqrt()).detach()
    aw = want[1].abs() * torch.finfo(w.dtype).eps / 2 + 4 * eps * (dy.double() * xh).abs().sum(0)
    assert ((dx.cpu().double() - want[0]).abs() <= ax).all()
    assert ((dw.cpu().double() - want[1]).abs() <= aw).all()
