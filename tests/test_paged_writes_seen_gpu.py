"""What the paged operators write in place is seen by autograd, where it has kept it."""
import pytest
import torch

import avelang_amd as ave

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code", [torch.bfloat16, torch.int8])
def test_cache(rocm_device, code):
    cache = ave.PagedKVCache.zeros(3, 16, 2, 64, code)
    rows = torch.randn(5, 2, 64, device=rocm_device).bfloat16()
    held = [t for t in (cache.k, cache.v, cache.k_scale, cache.v_scale) if t is not None]
    w = [torch.ones(t.shape, device=rocm_device, requires_grad=True) for t in held]
    for x, t in zip(w, held):
        loss = t * x
        version = t._version
        ave.paged_cache_write(cache, rows, rows, torch.arange(5, device=rocm_device))
        assert t._version > version
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.sum().backward()
    version = cache.k._version
    ave.paged_cache_read(cache, torch.arange(5, device=rocm_device))
    assert cache.k._version == version


def test_out(rocm_device):
    cache = ave.PagedKVCache.zeros(3, 16, 2, 64)
    i32 = dict(dtype=torch.int32, device=rocm_device)
    q = torch.randn(2, 1, 4, 64, device=rocm_device).bfloat16()
    args = q, cache, torch.zeros(2, 1, **i32), torch.ones(2, **i32)
    out = torch.zeros_like(q)
    w = torch.ones_like(q, requires_grad=True)
    loss = (out * w).sum()
    ave.paged_attention(*args, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_inference_tensors(rocm_device):
    with torch.inference_mode():
        cache = ave.PagedKVCache.zeros(3, 16, 2, 64, torch.float8_e4m3fn)
        rows = torch.randn(2, 2, 64, device=rocm_device).bfloat16()
        i32 = dict(dtype=torch.int32, device=rocm_device)
        q, out = (torch.randn(2, 1, 4, 64, device=rocm_device).bfloat16() for _ in "qo")
        args = q, cache, torch.zeros(2, 1, **i32), torch.ones(2, **i32)
    for mode in (True, False):
        with torch.inference_mode(mode):
            ave.paged_cache_write(cache, rows, rows, torch.arange(2, device=rocm_device))
            assert ave.paged_attention(*args, out=out) is out
