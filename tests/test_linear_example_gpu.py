"""The example's block: its parts together, as a program runs them.

Tolerances: a bf16 output differs by at most 2^-8 of its value per rounding;
the two ways to the same tokens round o, the head norm and the projection
each once, their operands once more: 2^-6 in the norm.
"""
import importlib.util
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    spec = importlib.util.spec_from_file_location(
        "decay_attention", os.path.join(ROOT, "examples", "decay_attention.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.gpu
@pytest.mark.parametrize("slopes", [False, True])
def test_prompt_then_tokens(rocm_device, slopes):
    torch.manual_seed(1)
    block = _example().DecayAttention(256, 2, 4, 64, 128, slopes=slopes, device=rocm_device)
    x = torch.randn(2, 140, 256, device=rocm_device).bfloat16()
    with torch.no_grad():
        whole, end = block(x)
        y, state = block(x[:, :133])
        out = [y]
        for t in range(133, 140):
            y, state = block(x[:, t:t + 1], state, decode=True)
            out.append(y)
    out = torch.cat(out, 1)
    assert ((out - whole).float().norm() <= 2 ** -6 * whole.float().norm())
    assert (state - end).norm() <= 2 ** -6 * end.norm()


@pytest.mark.gpu
def test_training_step(rocm_device):
    """Every parameter gets a gradient that lowers the loss along it."""
    torch.manual_seed(2)
    block = _example().DecayAttention(256, 2, 4, 64, 64, device=rocm_device)
    x = torch.randn(1, 200, 256, device=rocm_device).bfloat16()
    cu = torch.tensor([0, 70, 200], dtype=torch.int32, device=rocm_device)

    def loss():
        return (block(x, cu_seqlens=cu)[0].float() - 1).square().mean()
    first = loss()
    first.backward()
    with torch.no_grad():
        for n, p in block.named_parameters():
            assert p.grad is not None and p.grad.isfinite().all() and p.grad.norm() > 0, n
        size = torch.sqrt(sum(p.grad.float().square().sum() for p in block.parameters()))
        for p in block.parameters():
            p -= (0.05 * p.grad.float() / size).to(p.dtype)
        assert loss() < first
