"""The oracle of the attention layers' operators: gradients against differences, 8-bit codes against
their type's own values, all in 64 bits."""
import torch

from oracle import attn_ref as R


def _r(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


def test_rms_norm_gradients_are_differences():
    x, w, res = (t.requires_grad_() for t in (_r(3, 7), _r(7, seed=1), _r(3, 7, seed=2)))
    assert torch.autograd.gradcheck(lambda *a: R.rms_norm(*a, offset=1.0, rounded=False), (x, w, res))


def test_rotary_gradients_are_differences():
    f = 1e4 ** (-torch.arange(0, 6, 2, dtype=torch.float64) / 6)
    pos = torch.tensor([[0, 5, 1000]])
    for near in (False, True):
        x = _r(1, 3, 2, 8).requires_grad_()
        assert torch.autograd.gradcheck(lambda x: R.rotary(x, pos, f, 1.2, near), (x,))
        # turned back it is itself, times the magnitude's square
        y = R.rotary(R.rotary(x, pos, f, 1.2, near), -pos, f, 1.2, near)
        assert torch.allclose(y[..., :6], 1.44 * x[..., :6]) and torch.equal(y[..., 6:], x[..., 6:])


def test_codes_are_the_types_values():
    x = torch.cat([_r(64, 128), torch.zeros(1, 128, dtype=torch.float64)]).to(torch.bfloat16)
    for dtype in R.MOST:
        c, scale = R.codes(x, dtype)
        assert torch.equal(c.float().to(dtype).double(), c)        # values of the type, the largest among them
        assert torch.equal(c.abs().amax(-1)[:-1], torch.full((64,), R.MOST[dtype], dtype=torch.float64))
        assert not c[-1].any() and scale[-1] == 0
        half = torch.maximum(c.abs() / 16, torch.tensor(2.0 ** -10)) if dtype is not torch.int8 else torch.full_like(c, 0.5)
        assert ((c * x.double().abs().amax(-1, keepdim=True) / R.MOST[dtype] - x.double()).abs()
                <= half * scale.double()[:, None] * 1.0000001).all()


def test_attention_is_softmax():
    q, k, v = _r(3, 4, 8), _r(2, 9, 8, seed=1), _r(2, 9, 8, seed=2)
    o, lse, size = R.attention(q, k, v, 0.3)
    kk, vv = k.repeat_interleave(2, 0), v.repeat_interleave(2, 0)
    s = 0.3 * q.transpose(0, 1) @ kk.mT
    s = s.masked_fill(torch.ones(3, 9, dtype=torch.bool).triu(7), -torch.inf)
    assert torch.allclose(o.transpose(0, 1), s.softmax(-1) @ vv)
    assert torch.allclose(lse.T, s.logsumexp(-1)) and (size >= o.abs() - 1e-15).all()
    # the newest token alone sees all, a window of one only itself, fewer tokens than rows none
    assert torch.allclose(R.attention(q, k, v, 0.3, window=1)[0], vv[:, 6:].transpose(0, 1))
    o, lse, _ = R.attention(q, k[:, :1], v[:, :1], 0.3)
    assert not o[:2].any() and torch.isinf(lse[:2]).all() and torch.allclose(o[2], vv[:, 0])
