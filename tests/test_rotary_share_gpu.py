"""Rotary positions in place, q and k in one buffer: turned where they share nothing, refused where they do."""
import random

import pytest
import torch

import avelang_amd as ave

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", range(60))
def test_one_buffer(rocm_device, seed):
    rng = random.Random(seed)
    B, T, D = rng.randint(1, 3), rng.randint(1, 6), rng.choice([2, 6, 16])

    def layout(heads):
        """Strides of batch, token and head, one inside the other in any order, with gaps."""
        order, strides, at = rng.sample(range(3), 3), [0] * 3, D + rng.choice([0, 0, D, 2 * D, 3])
        for j in order:
            strides[j] = at
            at = at * (B, T, heads)[j] + rng.choice([0, 0, D, 5])
        return strides

    hq, hk = rng.randint(1, 4), rng.randint(1, 3)
    qs = layout(hq)
    ks = qs if rng.random() < 0.6 else layout(hk)
    buf = torch.randn(20000, device=rocm_device).bfloat16()
    views = lambda t: (t.as_strided((B, T, hq, D), (*qs, 1), q0), t.as_strided((B, T, hk, D), (*ks, 1), k0))  # noqa: E731
    q0, k0 = rng.randint(0, 60), rng.randint(0, 400)
    mine = [set(x.flatten().tolist()) for x in views(torch.arange(20000))]
    q, k = views(buf)
    pos, f = torch.arange(T, device=rocm_device) * 31, ave.rotary_frequencies(D, device=rocm_device)[0]
    want, before = ave.rotary_embedding(q, k, pos, f), buf.clone()
    if len(mine[0]) < B * T * hq * D or len(mine[1]) < B * T * hk * D or mine[0] & mine[1]:
        with pytest.raises(ValueError, match="of their own|share no element"):
            ave.rotary_embedding(q, k, pos, f, inplace=True)
        assert torch.equal(buf, before)
        return
    ave.rotary_embedding(q, k, pos, f, inplace=True)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    rest = torch.ones(20000, dtype=torch.bool)
    rest[list(mine[0] | mine[1])] = False
    assert torch.equal(buf.cpu()[rest], before.cpu()[rest])
