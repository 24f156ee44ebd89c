"""Linear attention token by token under a device cu_seqlens that breaks its contract: every
sequence is empty, o is zero and the states stay, as in the chunked form.

Tolerances: none.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

BAD = {"decreasing": [0, 100, 50, 230], "short_total": [0, 70, 100, 200], "nonzero_start": [5, 70, 70, 230],
       "overshoot": [0, 70, 300, 230], "beyond": [0, 70, 100, 300]}


@pytest.mark.parametrize("case", sorted(BAD))
@pytest.mark.parametrize("heads,K,V", [((2, 4), 64, 128), ((1, 512), 64, 64)])   # tiles; whole states
def test_violation_empties_every_sequence(rocm_device, case, heads, K, V):
    import avelang_amd as ave
    gen = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(s, generator=gen).to(rocm_device)  # noqa: E731
    q, k, v = (r(1, 230, h, d).bfloat16() for h, d in ((heads[0], K), (heads[0], K), (heads[1], V)))
    g, h0 = -r(heads[1]).abs(), r(3, heads[1], K, V)
    cu = torch.tensor(BAD[case], dtype=torch.int32, device=rocm_device)
    out = torch.full_like(v, 7.0)
    o, ht = ave.fused_recurrent_linear_attn(q, k, v, g, initial_state=h0, output_final_state=True,
                                            inplace_final_state=False, cu_seqlens=cu, out=out)
    assert o is out and not o.any() and torch.equal(ht, h0)
    pool, idx = r(5, heads[1], K, V), torch.tensor([3, 9, 0], dtype=torch.int32, device=rocm_device)
    before = pool.clone()
    out.fill_(7.0)
    ave.fused_recurrent_linear_attn(q, k, v, g, initial_state=pool, output_final_state=True, cu_seqlens=cu,
                                    ssm_state_indices=idx, out=out)
    assert not out.any() and torch.equal(pool, before)
    # and what keeps the contract is as ever
    cu = torch.tensor([0, 100, 100, 230], dtype=torch.int32, device=rocm_device)
    a = ave.fused_recurrent_linear_attn(q, k, v, g, initial_state=h0, output_final_state=True,
                                        inplace_final_state=False, cu_seqlens=cu)
    b = ave.fused_recurrent_linear_attn(q, k, v, g, initial_state=h0, output_final_state=True,
                                        inplace_final_state=False, cu_seqlens=cu.cpu())
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and a[0].any()


@pytest.mark.parametrize("B,T,cu", [(2, 0, None), (0, 5, None), (1, 0, [0, 0, 0])])
@pytest.mark.parametrize("per_head", [False, True])
def test_no_tokens(rocm_device, B, T, cu, per_head):
    """Nothing to read: the states stay, and the decays' gradients over no tokens are zero."""
    import avelang_amd as ave
    N = B if cu is None else 2
    z = lambda *s: torch.zeros(s, device=rocm_device, dtype=torch.bfloat16)  # noqa: E731
    q, k, v = z(B, T, 2, 64), z(B, T, 2, 64), z(B, T, 4, 64)
    g = -torch.ones(4, device=rocm_device) if per_head else torch.zeros(B, T, 4, device=rocm_device)
    h0, dht = (torch.randn(N, 4, 64, 64, device=rocm_device) for _ in range(2))
    c = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=rocm_device)
    for op, kw in ((ave.chunk_linear_attn, {}), (ave.fused_recurrent_linear_attn, dict(inplace_final_state=False))):
        o, ht = op(q, k, v, g, initial_state=h0, output_final_state=True, cu_seqlens=c, **kw)
        assert o.shape == v.shape and torch.equal(ht, h0)
    dq, dk, dv, dg, dh0 = ave.chunk_linear_attn_bwd(q, k, v, g, v, dht, initial_state=h0, cu_seqlens=c)
    assert dq.shape == q.shape and dv.shape == v.shape and torch.equal(dh0, dht)
    assert dg.shape == g.shape and not dg.any()
