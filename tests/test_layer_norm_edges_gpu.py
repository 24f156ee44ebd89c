"""Layer norm's backward at its edges: rows that are constant and large, several rows per workgroup
of long rows.

Tolerances: as in the tests of ordinary rows.  y and dx are computed in fp32 and rounded once, half a
step of their type and 2^-19 of the terms they are the sum of; dweight and dbias are fp32 sums over
the rows, 2^-18 in the norm before their own rounding.
"""
import pytest
import torch

from oracle import linear_ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [1, 5, 8, 13, 100, 250, 1000, 2001, 2100, 8200, 20001])
@pytest.mark.parametrize("xt", [torch.float32, torch.bfloat16])
def test_constant_rows(rocm_device, D, xt):
    """x = 2^120 / D's power of two: xh is 0, dx = (dy w - its mean) / sqrt(eps) and finite, however
    large the mean; the other rows and the sums over the rows as ever."""
    import avelang_amd as ave
    gen = torch.Generator().manual_seed(D)
    x = torch.randn((3, D), generator=gen).to(xt)
    # (the row's sum stays within fp32 and exact: its mean is x itself)
    x[1] = 2.0 ** (127 - max(1, (D - 1).bit_length()) - 1)
    w = (1 + 0.2 * torch.randn(D, generator=gen))
    dy = torch.randn((3, D), generator=gen).to(xt)
    leaves = [t.double().requires_grad_() for t in (x, w)]
    want = torch.autograd.grad(linear_ref.layer_norm(*leaves, eps=1e-30), leaves, dy.double())
    mine = [t.to(rocm_device).requires_grad_() for t in (x, w)]
    got = torch.autograd.grad(ave.layer_norm(*mine, eps=1e-30), mine, dy.to(rocm_device))
    half = torch.finfo(xt).eps / 2
    dx, dw = (g.double().cpu() for g in got)
    assert dx.isfinite().all() and dw.isfinite().all()
    e = dy.double() * w.double()
    assert ((dx[1] - want[0][1]).abs() <= (half * want[0][1].abs() + 2 ** -19 * 1e15 * (e[1].abs() + e[1].abs().mean()))).all()
    if D > 5:   # (shorter rows' terms cancel to eps' share)
        assert (dx[[0, 2]] - want[0][[0, 2]]).norm() <= (half + 2 ** -18) * want[0][[0, 2]].norm()
        assert (dw - want[1]).norm() <= 2 ** -18 * want[1].norm()


@pytest.mark.parametrize("rows,D,xt", [(1500, 4096, torch.bfloat16), (1601, 8192, torch.bfloat16),
                                       (1301, 8000, torch.float32), (1100, 2049, torch.float32),
                                       (5000, 2048, torch.float16)])
@pytest.mark.parametrize("heads", [0, 3])
def test_several_rows_per_workgroup(rocm_device, rows, D, xt, heads):
    """More rows than the groups that walk them: each takes two and more, the next on its way."""
    import avelang_amd as ave
    gen = torch.Generator(device=rocm_device).manual_seed(rows)
    r = lambda *s: torch.randn(s, generator=gen, device=rocm_device)  # noqa: E731
    par = (heads, D) if heads else (D,)
    x = (r(rows, *par) * (0.5 + r(rows, *par[:-1], 1).abs()) + r(rows, *par[:-1], 1)).to(xt)
    w, b, dy = 1 + 0.2 * r(*par), 0.1 * r(*par), r(rows, *par).to(xt)
    leaves = [t.double().requires_grad_() for t in (x, w, b)]
    ref = linear_ref.layer_norm(*leaves)
    want = torch.autograd.grad(ref, leaves, dy.double())
    mine = [t.clone().requires_grad_() for t in (x, w, b)]
    y = ave.layer_norm(*mine)
    got = torch.autograd.grad(y, mine, dy)
    half = torch.finfo(xt).eps / 2
    assert (y.detach().double() - ref.detach()).norm() <= (half + 2 ** -18) * ref.detach().norm()
    for g, want_g, h in zip(got, want, (half, 0, 0)):
        assert (g.double() - want_g).norm() <= (h + 2 ** -18) * want_g.norm()
    again = torch.autograd.grad(ave.layer_norm(*mine), mine, dy)
    assert all(torch.equal(g, a) for g, a in zip(got, again))
