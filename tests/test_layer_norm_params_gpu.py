"""Layer norm with parameters of every type beside rows of every type: fp32 rows of more than one vector
per lane with fp16 parameters once read the parameters of another address.

Bounds as in test_layer_norm_gpu: 2^-18 of the terms for fp32's sums, half a step of the type.
"""
import pytest
import torch

import avelang_amd as ave
from oracle import linear_ref

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.mark.parametrize("xt", TYPES)
@pytest.mark.parametrize("wt", TYPES)
@pytest.mark.parametrize("rows,D", [(3, 64), (5, 300), (1, 513), (4, 1001), (2, 2049), (3, 5000), (2, 8192)])
def test_parameters_of_every_type(rocm_device, rows, D, xt, wt):
    gen = torch.Generator().manual_seed(D)
    x = torch.randn((rows, D), generator=gen).to(TYPES[xt])
    w, b = (torch.randn(D, generator=gen).to(TYPES[wt]) for _ in "wb")
    dy = torch.randn((rows, D), generator=gen).to(TYPES[xt])
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    y = ave.layer_norm(*leaves)
    got = torch.autograd.grad(y, leaves, dy.cuda())
    ref = [t.double().requires_grad_() for t in (x, w, b)]
    want = linear_ref.layer_norm(*ref)
    grads = torch.autograd.grad(want, ref, dy.double())
    size = [6 * w.abs().double() + b.abs().double(), 30 * dy.abs().double() + 30, 6 * dy.abs().double().sum(0),
            dy.abs().double().sum(0)]
    for a, r, s, t in zip((y, *got), (want, *grads), size, (xt, xt, wt, wt)):
        assert a.dtype == TYPES[t]
        assert ((a.detach().cpu().double() - r.detach()).abs()
                <= s * 2 ** -18 + r.detach().abs() * torch.finfo(TYPES[t]).eps / 2 + 2.0 ** -25).all()
