"""Copies of strided arguments live until the launch that reads them: another thread of the same stream cannot be
given their memory, and fill it, between the call's reading of their addresses and its launch."""
import sys

import pytest
import torch

import avelang_amd as ave
from avelang_amd import workloads as W

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


def _every_other(t):
    return torch.stack([t, t], -1)[..., 0]


@pytest.mark.parametrize("T", [1, 70])
def test_gating_parameters(rocm_device, T):
    """Both strided: neither's copy takes the other's place."""
    t = W.make(2, T, 2, 4, 128, 128, seed=5).torch(rocm_device)
    a, b = (torch.randn(2, T, 4, device=rocm_device) for _ in "ab")
    A_log, bias = torch.rand(4, device=rocm_device), torch.randn(4, device=rocm_device)
    call = ave.chunk_gated_delta_rule_gated if T > 1 else ave.fused_recurrent_gated_delta_rule_gated
    h0 = torch.randn(2, 4, 128, 128, device=rocm_device)
    want, _ = call(t["q"], t["k"], t["v"], a, b, A_log, bias, initial_state=h0)
    got, _ = call(t["q"], t["k"], t["v"], a, b, _every_other(A_log), _every_other(bias), initial_state=h0)
    assert torch.equal(got, want)


@pytest.mark.parametrize("rows", [False, True])
def test_state_slots(rocm_device, monkeypatch, rows):
    """(With both entries 1, which the busy thread leaves, the kernel would refuse the slots and write NaN.)"""
    t = W.make(2, 1, 2, 4, 128, 128, seed=6).torch(rocm_device)
    pool = torch.randn(4, 4, 128, 128, device=rocm_device)
    idx = torch.tensor([3, 0], dtype=torch.int32, device=rocm_device)
    q, k, v = t["q"], t["k"], t["v"]
    if rows:   # columns of one projection
        q, k, v = torch.cat([x.flatten(2) for x in (q, k, v)], -1).split([256, 256, 512], -1)
        q, k, v = q.view(2, 1, 2, 128), k.view(2, 1, 2, 128), v.view(2, 1, 4, 128)
    args = q, k, v, t["g"], t["beta"]
    one, two = pool.clone(), pool.clone()
    want, _ = ave.fused_recurrent_gated_delta_rule(*args, initial_state=one, output_final_state=True,
                                                   ssm_state_indices=idx)
    strided = _every_other(idx)
    _busy(monkeypatch, "gated_delta_rule", "_stream_ptr", 2, 1)
    got, _ = ave.fused_recurrent_gated_delta_rule(*args, initial_state=two, output_final_state=True,
                                                  ssm_state_indices=strided)
    assert torch.equal(got, want) and torch.equal(one, two)
