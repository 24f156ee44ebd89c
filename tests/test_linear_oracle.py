"""The oracle's formulas of chunks against its token recurrence and that one's autograd gradients,
in 64 bits: a few thousand roundings of 2^-53."""
import pytest
import torch

from oracle import linear_ref


@pytest.mark.parametrize("heads", [(1, 1), (2, 4), (1, 3)])
@pytest.mark.parametrize("lens,slopes,h0", [(None, False, True), (None, True, False),
                                            ([1, 0, 64, 70, 130], False, True), ([65, 3], True, True)])
def test_chunks_are_the_recurrence(heads, lens, slopes, h0):
    gen = torch.Generator().manual_seed(heads[1])
    r = lambda *s: torch.randn(s, generator=gen, dtype=torch.float64)  # noqa: E731
    B, T, K, V = (2, 150, 5, 3) if lens is None else (1, sum(lens), 5, 3)
    N = B if lens is None else len(lens)
    cu = None if lens is None else [sum(lens[:i]) for i in range(N + 1)]
    g = -r(heads[1]).exp() / 8 if slopes else -torch.exp(r(B, T, heads[1]))
    leaves = [r(B, T, heads[0], K), r(B, T, heads[0], K), r(B, T, heads[1], V), g]
    if h0:
        leaves.append(r(N, heads[1], K, V))
    leaves = [x.requires_grad_() for x in leaves]
    do, dht = r(B, T, heads[1], V), r(N, heads[1], K, V)
    o, ht = linear_ref.linear_attn(*leaves[:4], h0=leaves[4] if h0 else None, cu=cu)
    want = (o, ht) + torch.autograd.grad([o, ht], leaves, [do, dht])
    with torch.no_grad():
        got = linear_ref.linear_attn_chunked(*leaves[:4], do, dht, h0=leaves[4] if h0 else None, cu=cu)
    for x, ref in zip(got, want):
        assert x.shape == ref.shape and (x - ref).abs().max() <= 1e-11 * (1 + ref.abs().max())
