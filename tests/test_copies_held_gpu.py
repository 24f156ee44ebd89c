"""Copies of strided arguments live until the launch that reads them: another thread of the same stream cannot be
given their memory, and fill it, between the call's reading of their addresses and its launch."""
import sys

import pytest
import torch

import avelang_amd as ave

pytestmark = pytest.mark.gpu


def _busy(monkeypatch, module, name, size, value):
    """Ahead of every launch, as another thread may: fresh int32 tensors of ``size``, filled with a value in range."""
    module = sys.modules["avelang_amd." + module]
    stream, held = getattr(module, name), []

    def busy(dev):
        held.extend(torch.full((size,), value, dtype=torch.int32, device=dev) for _ in range(4))
        return stream(dev)

    monkeypatch.setattr(module, name, busy)


def test_paged_attention_lengths(rocm_device, monkeypatch):
    cache = ave.PagedKVCache.zeros(12, 16, 2, 64)
    for x in (cache.k, cache.v):
        x.normal_()
    table = torch.arange(12, dtype=torch.int32, device=rocm_device).view(3, 4)
    lens = torch.tensor([60, 7, 33], dtype=torch.int32, device=rocm_device)
    q = torch.randn(3, 1, 4, 64, device=rocm_device).bfloat16()
    want = ave.paged_attention(q, cache, table, lens)
    strided = torch.stack([lens, lens], 1)[:, 0]
    _busy(monkeypatch, "paged_attention", "_stream", 3, 1)
    assert torch.equal(ave.paged_attention(q, cache, table, strided), want)
