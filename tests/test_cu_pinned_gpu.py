"""cu_seqlens in pinned host memory, a serving loop's staging buffer, refilled as soon as the call
returns: the call keeps the offsets that it was given.

Tolerances: none, the same bits as with offsets that nobody touches.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("op", ["chunk_linear_attn", "fused_recurrent_linear_attn", "chunk_gated_delta_rule",
                                "fused_recurrent_gated_delta_rule"])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_refilled_at_once(rocm_device, op, dtype):
    import avelang_amd as ave
    gen = torch.Generator().manual_seed(4)
    r = lambda *s: torch.randn(s, generator=gen).to(rocm_device)  # noqa: E731
    q, k, v = (0.1 * r(1, 200, h, 64) for h in (2, 2, 4))
    args = [x.bfloat16() for x in (q, k, v)] + [-r(1, 200, 4).abs()]
    if "delta" in op:
        args.append(r(1, 200, 4).sigmoid())
    state = r(3, 4, 64, 64)
    first, second = (torch.tensor(c, dtype=dtype) for c in ([0, 30, 130, 200], [0, 100, 150, 200]))

    def call(cu):
        return getattr(ave, op)(*args, initial_state=state.clone(), output_final_state=True, cu_seqlens=cu)
    want = [call(c.to(rocm_device)) for c in (first, second)]
    big = torch.randn(8192, 8192, device=rocm_device).bfloat16()
    staging = torch.empty(4, dtype=dtype, pin_memory=True)
    torch.cuda.synchronize()
    for _ in range(10):   # some 10 ms ahead of the copies
        big @ big
    got = []
    for c in (first, second):
        staging.copy_(c)
        got.append(call(staging))
    staging.zero_()
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(x, y))


def test_captured(rocm_device):
    """In a graph every replay reads the buffer as it is then."""
    import avelang_amd as ave
    gen = torch.Generator().manual_seed(5)
    q, k, v = (torch.randn((1, 200, h, 64), generator=gen).to(rocm_device).bfloat16() for h in (2, 2, 4))
    g = -torch.rand((1, 200, 4), generator=gen).to(rocm_device)
    offsets = [torch.tensor(c, dtype=torch.int32) for c in ([0, 30, 130, 200], [0, 100, 150, 200])]
    want = [ave.chunk_linear_attn(q, k, v, g, output_final_state=True, cu_seqlens=c) for c in offsets]
    staging = torch.empty(4, dtype=torch.int32, pin_memory=True).copy_(offsets[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ave.chunk_linear_attn(q, k, v, g, output_final_state=True, cu_seqlens=staging)
    for i in (0, 1, 0, 1):
        staging.copy_(offsets[i])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(held, want[i]))
