"""Layer norm, forward and backward, against its definition in 64 bits.

Tolerances.  y and dx are computed in fp32 and rounded once: half a step of
their type (2^-8 bf16, 2^-11 fp16) of their value, and 2^-19 of the size of the
terms they are the sum of for fp32's own roundings (a few dozen on a path of
tree sums).  dweight and dbias are fp32 sums over the rows, split into at least
a few dozen partial sums: 2^-18 in the norm before their own rounding.
"""
import pytest
import torch

from oracle import linear_ref

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half(t):
    return torch.finfo(t).eps / 2


def make(shape, par, xt, wt, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    x = (r(*shape) * (0.5 + r(*shape[:-1], 1).abs()) + r(*shape[:-1], 1)).to(xt)
    return x, (1 + 0.2 * r(*par)).to(wt), (0.1 * r(*par)).to(wt), r(*shape).to(xt)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [1, 2, 7, 8, 64, 100, 128, 250, 256, 500, 1001, 2048, 2500, 4096, 8192,
                               8200, 20001])
@pytest.mark.parametrize("xt,wt", [("bf16", "f32"), ("f32", "f32"), ("f16", "bf16"), ("bf16", "bf16")])
def test_norm(rocm_device, D, xt, wt):
    import avelang_amd as ave
    xt, wt = TYPES[xt], TYPES[wt]
    for rows, heads in ((5, 0), (3, 4)) if D <= 8200 else ((3, 0),):
        par = (heads, D) if heads else (D,)
        x, w, b, dy = make((rows,) + par, par, xt, wt, seed=D)
        leaves = [t.double().requires_grad_() for t in (x, w, b)]
        ref = linear_ref.layer_norm(*leaves)
        want = torch.autograd.grad(ref, leaves, dy.double())
        mine = [t.to(rocm_device).requires_grad_() for t in (x, w, b)]
        y = ave.layer_norm(*mine)
        assert y.dtype == xt
        # the terms' sizes: a row's centre far from 0 costs the centred values that much more
        xd, e = x.double(), dy.double() * w.double()
        var, mean = torch.var_mean(xd, -1, correction=0, keepdim=True)
        rstd = (var + 1e-5).rsqrt()
        xh = ((xd - mean) * rstd).abs()
        off = xh + rstd * (xd.abs() + mean.abs())
        size = off * w.double().abs() + b.double().abs()
        assert ((y.detach().cpu().double() - ref).abs() <= half(xt) * ref.abs() + 2 ** -19 * size + half(xt) * 1e-4).all()
        with torch.no_grad():
            assert torch.equal(ave.layer_norm(*mine), y)
        got = torch.autograd.grad(y, mine, dy.to(rocm_device))
        assert all(g.dtype == t and g.shape == r.shape for g, r, t in zip(got, want, (xt, wt, wt)))
        m = lambda z: z.mean(-1, keepdim=True)  # noqa: E731
        size = rstd * (e.abs() + m(e.abs()) + off * m(e.abs() * xh) + xh * m(e.abs() * off))
        assert ((got[0].cpu().double() - want[0]).abs() <= half(xt) * want[0].abs() + 2 ** -19 * size + half(xt) * 1e-4).all()
        for g, r, t, terms in zip(got[1:], want[1:], (wt, wt), (dy.double() * off, dy.double())):
            assert (g.cpu().double() - r).norm() <= half(t) * r.norm() + 2 ** -18 * terms.norm()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 3, 1000, 20000])
@pytest.mark.parametrize("heads,D", [(0, 48), (0, 1000), (5, 33), (32, 128)])
def test_many_rows(rocm_device, rows, heads, D):
    """The sums over the rows, and twice the same bits."""
    import avelang_amd as ave
    if rows * max(1, heads) * D > 3e7:
        rows = 2001
    par = (heads, D) if heads else (D,)
    x, w, b, dy = make((rows,) + par, par, torch.bfloat16, torch.float32, seed=rows)
    leaves = [t.double().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(linear_ref.layer_norm(*leaves), leaves, dy.double())
    t = [z.to(rocm_device) for z in (x, w, b, dy)]
    y, stats = ave.layer_norm_fwd_save(*t[:3])
    got = ave.layer_norm_bwd(t[0], t[1], t[3], stats)
    for g, r, h in zip(got, want, (2 ** -8, 0, 0)):
        assert (g.cpu().double() - r).norm() <= (h + 2 ** -18) * r.norm()
    again = ave.layer_norm_bwd(t[0], t[1], t[3], stats)
    assert all(torch.equal(g, a) for g, a in zip(got, again))


@pytest.mark.gpu
def test_rows_apart_and_parameters_left_out(rocm_device):
    """A row of NaN or infinity stays in its row; constant rows; no weight, no bias; odd bases;
    views; empty; out on x."""
    import avelang_amd as ave
    x, w, b, dy = (t.to(rocm_device) for t in make((40, 96), (96,), torch.bfloat16, torch.float32))
    want = ave.layer_norm(x, w, b)
    bad = x.clone()
    bad[3, 5], bad[7, 0], bad[9] = float("nan"), float("inf"), 2.0
    got = ave.layer_norm(bad, w, b)
    keep = [i for i in range(40) if i not in (3, 7, 9)]
    assert torch.equal(got[keep], want[keep]) and got[3].isnan().all() and got[7].isnan().all()
    assert torch.equal(got[9], b.to(x.dtype))
    for ww, bb in ((None, None), (w, None), (None, b)):
        r = linear_ref.layer_norm(x.cpu(), None if ww is None else ww.cpu(), None if bb is None else bb.cpu())
        xs = x.clone().requires_grad_()
        y = ave.layer_norm(xs, ww, bb)
        assert ((y.detach().cpu().double() - r).abs() <= 2 ** -8 * r.abs() + 2 ** -15).all()
        y.backward(dy)
        assert xs.grad.isfinite().all()
    flat = torch.empty(40 * 96 + 1, dtype=x.dtype, device=rocm_device)
    odd = flat[1:].view(40, 96)
    odd.copy_(x)
    assert torch.equal(ave.layer_norm(odd, w, b), want)
    wide = torch.empty(40, 200, dtype=x.dtype, device=rocm_device)
    wide[:, 7:103] = x
    assert torch.equal(ave.layer_norm(wide[:, 7:103], w, b), want)
    assert ave.layer_norm(x[:0], w, b).shape == (0, 96)
    e = x[:0].clone().requires_grad_()
    ww = w.clone().requires_grad_()
    ave.layer_norm(e, ww, b).sum().backward()
    assert (ww.grad == 0).all()
    buf = x.clone()
    assert ave.layer_norm(buf, w, b, out=buf) is buf and torch.equal(buf, want)


@pytest.mark.gpu
def test_norm_graph(rocm_device):
    import avelang_amd as ave
    x, w, b, dy = (t.to(rocm_device) for t in make((500, 300), (300,), torch.float32, torch.float32))

    def work():
        y, stats = ave.layer_norm_fwd_save(x, w, b)
        return (y,) + ave.layer_norm_bwd(x, w, dy, stats)
    work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
    for _ in range(3):
        x.copy_(torch.randn_like(x))
        dy.copy_(torch.randn_like(dy))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(held, work()))
