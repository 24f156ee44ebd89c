"""A workspace for the largest call of a program serves its smaller ones."""
import random
import re

import pytest
import torch

from avelang_amd import _native
from avelang_amd import linear_attention as L

HEADS = [(16, 32, 128, 128), (2, 4, 128, 64), (16, 16, 64, 128), (4, 16, 64, 64), (1, 8, 128, 128),
         (3, 9, 64, 64), (128, 384, 64, 128), (600, 600, 64, 64)]


def _need(B, T, Hqk, Hv, K, V, N, packed, backward):
    """What the entry point asks for: from its refusal of a workspace too small for anything."""
    lib = _native.lib()
    p = [(i + 1) << 42 for i in range(14)]
    rows, cu = (Hqk * K, Hqk * K, Hv * V), p[4] if packed else None
    if backward:
        rc = lib.gdn_linear_chunk_bwd(p[0], p[1], p[2], *rows, p[3], 0, 0, p[5], None, p[6], p[7], p[8],
                                      p[9], p[10], None, cu, B, T, Hqk, Hv, K, V, N, 0.1, p[11], 1, None)
    else:
        rc = lib.gdn_linear_chunk_fwd(p[0], p[1], p[2], *rows, p[3], 0, 0, None, None, p[5], cu, B, T,
                                      Hqk, Hv, K, V, N, 0.1, None, p[11], 1, None)
    if rc == -2:   # too many tokens altogether
        return 0
    assert rc == -4
    return int(re.search(r"needs (\d+) bytes", _native.last_error()).group(1))


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("heads", HEADS)
def test_sizes_grow(heads, backward):
    """Every pair of sizes: more tokens, more sequences never ask for less; and a call never needs
    more than what its own sizes are told (packed calls and gradients need some in any case)."""
    f = L.linear_attn_workspace_bytes
    rng = random.Random(heads[1])
    Ts = sorted({1, 63, 64, 65, 100, 127, 128, 129, 512, 576, 1024, 1088, 2048, 2112, 6144, 6208, 8192}
                | {int(2 ** rng.uniform(0, 15)) for _ in range(40)})
    Ns = sorted({1, 2, 3, 4, 7, 8, 15, 16, 17, 31, 32, 33, 63, 64, 100, 256, 511, 512, 513, 1000})
    for packed in (False, True):
        size = {(T, n): f(1 if packed else n, T, *heads, n, packed, backward) for T in Ts for n in Ns}
        for i, T in enumerate(Ts):
            for j, n in enumerate(Ns):
                assert i == 0 or size[T, n] >= size[Ts[i - 1], n]
                assert j == 0 or size[T, n] >= size[T, Ns[j - 1]]
                if packed or backward:
                    assert size[T, n] >= _need(1 if packed else n, T, *heads, n, packed, backward)


def test_prompt_sizes():
    """One prompt's need is not monotone by itself (fewer, longer segments from some length on)."""
    f = lambda T: L.linear_attn_workspace_bytes(1, T, 16, 32, 128, 128, 1, False)  # noqa: E731
    sizes = [f(T) for T in range(1, 20000, 37)]
    assert sizes == sorted(sizes) and f(64) == 0 and f(1 << 20) < 40 << 20
    need = lambda T: _need(1, T, 16, 32, 128, 128, 1, False, False)  # noqa: E731
    assert need(512) > need(576)
    assert all(f(T) >= need(T) for T in range(65, 20000, 61))


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [False, True])
def test_one_workspace_for_all(rocm_device, packed):
    import avelang_amd as ave
    heads = (2, 4, 64, 64)
    Ts = [1, 64, 65, 130, 300, 449, 512, 576, 1000, 2000]
    size = max(Ts)
    ws = [torch.empty(L.linear_attn_workspace_bytes(1, size, *heads, 3 if packed else 1, packed, b),
                      dtype=torch.uint8, device=rocm_device) for b in (False, True)]
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(s, generator=gen).to(rocm_device)  # noqa: E731
    for T in Ts:
        q, k, v, do = (r(1, T, h, 64).bfloat16() for h in (2, 2, 4, 4))
        g = -r(1, T, 4).abs()
        cu = torch.tensor([0, T // 3, T // 3, T], device=rocm_device) if packed else None
        h0 = r(3 if packed else 1, 4, 64, 64)
        kw = dict(initial_state=h0, cu_seqlens=cu)
        a = ave.chunk_linear_attn(q, k, v, g, output_final_state=True, **kw)
        b = ave.chunk_linear_attn(q, k, v, g, output_final_state=True, workspace=ws[0], **kw)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        a = ave.chunk_linear_attn_bwd(q, k, v, g, do, **kw)
        b = ave.chunk_linear_attn_bwd(q, k, v, g, do, workspace=ws[1], **kw)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
