"""Attention over a paged cache where weights and values differ by many powers of two, against float64.

Bounds as in test_paged_attention_gpu.py, without an absolute part but half of fp16's smallest step: with A the
mean of |v| under the softmax 2^-13 A, 2^-11 A more for a bf16 output over 8 bits, and half a step of the
output's type.  P (over 8 bits times V's scale) is brought to at least 2^14 where it is largest in its row, so that
fp16's smallest half step, 2^-25, is 2^-39 of that: for n tokens 2^-39 of the largest P times the sum of |v| (of
|codes|), which is no more than 2^-39 n times the largest |v| (over 8 bits, where every row has a code of M in some
column, than 2^-39 n times the largest A of the row).  A score's fp32 sum errs by some 2^-24 (D / 32 + 32) of sum |q k| scale: that of a token whose key
is its query's multiple is the score itself, 16 at most here, so 2^-15 of every weight.
"""
import pytest
import torch

import avelang_amd as ave
from oracle import attn_ref as R
from test_paged_attention_gpu import BF16, CODES, E4M3, F16, I8, _case

pytestmark = pytest.mark.gpu
C8 = [(BF16, E4M3), (F16, E4M3), (BF16, I8), (F16, I8)]


def _check(got, q, cache, table, lens, window=0, rows=slice(None)):
    D, page = q.shape[-1], cache.k.shape[2]
    c = [None if x is None else x.cpu() for x in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    one = cache.k.element_size() == 1 and q.dtype is BF16
    for i, n in enumerate(lens.tolist()):
        pages = table[i, :-(-n // page)].tolist()
        k, v = R.rows_of(c[0], c[2], pages, n), R.rows_of(c[1], c[3], pages, n)
        o, _, size = (x[rows] for x in R.attention(q[i].cpu(), k, v, D ** -0.5, window))
        off = (got[i].cpu().double()[rows] - o).abs()
        bound = size * (2 ** -13 + (2 ** -11 if one else 0)) + o.abs() * torch.finfo(q.dtype).eps / 2
        bound += 2 ** -25 if q.dtype is F16 else 0
        bound += 2 ** -39 * n * (size.amax(-1, keepdim=True) if c[2] is not None else v.abs().max())
        assert (off <= bound).all(), (i, n, (off / bound).max())


def _token(cache, table, i, t):
    """(page, row) of sequence i's token t."""
    page = cache.k.shape[2]
    return int(table[i, t // page]), t % page


def _place(cache, table, i, t, k, v):
    """Rows k, v [H, D] as sequence i's token t."""
    page, row = _token(cache, table, i, t)
    ave.paged_cache_write(cache, k[None], v[None], torch.tensor([page * cache.k.shape[2] + row]))


@pytest.mark.parametrize("t,code", CODES)
@pytest.mark.parametrize("D,H,N,most", [(64, 2, 600, 300), (128, 8, 30, 880), (64, 1, 1, 9000)])
def test_a_token_that_takes_nearly_all(rocm_device, D, H, N, most, t, code):
    """The first token takes 99.9 % of the softmax and has a small value: what is left is the other tokens'."""
    lens = [most - (7 * i) % (most // 2) for i in range(N)]
    q, cache, table, n = _case(lens, 1, H, H, D, 16, t, code, seed=21)
    q.mul_(0.1)
    for i, m in enumerate(lens):
        # (the others' scores are about 0: q is short)
        k = q[i, 0].float()
        k = k * (torch.log(torch.tensor(999.0 * m)) * D ** 0.5 / k.square().sum(-1, keepdim=True))
        _place(cache, table, i, 0, k.to(t), 1e-3 * torch.randn(H, D, device="cuda").to(t))
    _check(ave.paged_attention(q, cache, table, n), q, cache, table, n)


@pytest.mark.parametrize("code", [F16, I8])
@pytest.mark.parametrize("size", [1e3, 2.0 ** 18, 1e6, 1e8])
def test_large_scores(rocm_device, size, code):
    """Scores of such a size: one token takes all of the softmax, or tokens of the same key share it."""
    q, cache, table, n = _case([300, 1, 40], 1, 4, 2, 64, 16, F16, code, seed=30)
    for sign in (1, -1):
        k = sign * q[:, 0, ::2].float()
        scale = size / k.square().sum(-1).amin().item()
        for i, ln in enumerate(n.tolist()):
            for at in range(ln):
                page, row = _token(cache, table, i, at)
                if at % 3 == 0:
                    _place(cache, table, i, at, k[i].half(), torch.full((2, 64), 2.0, device="cuda").half())
                else:   # (a third of the key: far below, or far above, the others)
                    _place(cache, table, i, at, (k[i] / 3).half(), torch.full((2, 64), 1.0, device="cuda").half())
        o = ave.paged_attention(q, cache, table, n, scale)
        # heads 0 and 2 have their own query in the keys; a sequence of one token sees that alone
        want = torch.tensor([2.0, 2.0, 2.0] if sign > 0 else [1.0, 2.0, 1.0], device="cuda")
        assert ((o[:, 0, ::2].float() - want[:, None, None]).abs() <= 2 ** -10).all()


@pytest.mark.parametrize("t,code", C8)
@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("lens", [[200, 40, 4], [3000, 700, 9]])
@pytest.mark.parametrize("power", [16, 80, 126, None])
def test_a_large_value_that_is_not_seen(rocm_device, power, lens, D, t, code):
    """A draft's scale of v, 2^power or infinite, is nothing to the rows ahead of it, nor to those whose window has
    left it behind."""
    q, cache, table, n = _case(lens, 4, 4, 2, D, 16, t, code, seed=4)
    base = ave.paged_attention(q, cache, table, n)
    near = ave.paged_attention(q, cache, table, n, window=2)
    big = torch.inf if power is None else 2.0 ** power
    for i, ln in enumerate(lens):
        page, row = _token(cache, table, i, ln - 3)   # row 1 of 4: seen by rows 1 to 3, in a window of 2 by 1 and 2
        cache.v_scale[page, 1, row] = big
    o = ave.paged_attention(q, cache, table, n)
    assert torch.equal(o[:, :1], base[:, :1]) and torch.equal(o[:, :, :2], base[:, :, :2])
    o = ave.paged_attention(q, cache, table, n, window=2)
    assert torch.equal(o[:, ::3], near[:, ::3]) and torch.equal(o[:, :, :2], near[:, :, :2])
    if power is None:
        assert not o[:, 1:3, 2:].isfinite().any()
    elif t is BF16 and power <= 80:
        _check(o, q, cache, table, n, 2, slice(1, 3))


@pytest.mark.parametrize("t,code", C8)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens", [[129, 40, 4], [4000, 700, 33]])
@pytest.mark.parametrize("power", [10, 30])
def test_a_large_value_of_no_weight(rocm_device, power, lens, D, t, code):
    """A token with a value 2^power times the others', and a weight of 2^-80 of theirs or less."""
    q, cache, table, n = _case(lens, 1, 2, 2, D, 16, t, code, seed=6)
    for i, ln in enumerate(lens):
        for at in {0, ln // 2, ln - 1}:
            k = q[i, 0].float()
            k = k * (-80 * D ** 0.5 / k.square().sum(-1, keepdim=True))
            _place(cache, table, i, at, k.to(t), torch.randn(2, D, device="cuda").to(t))
            page, row = _token(cache, table, i, at)
            cache.v_scale[page, :, row] *= 2.0 ** power
    _check(ave.paged_attention(q, cache, table, n), q, cache, table, n)


@pytest.mark.parametrize("code", [E4M3, I8])
@pytest.mark.parametrize("D,H,lens", [(128, 2, [1, 40, 300, 9000]), (256, 1, [5000]), (64, 2, [250] * 560)])
@pytest.mark.parametrize("top", [125, -100])
def test_far_scales(rocm_device, top, D, H, lens, code):
    """Values up to 2^top: neither their sum over the tokens nor a factor on its way leaves fp32's range."""
    q, cache, table, n = _case(lens, 1, 2 * H, H, D, 16, BF16, code, seed=7)
    page = cache.k.shape[2]
    for i, ln in enumerate(lens):   # (the rows that tokens have; the others stay NaN)
        for p in range(-(-ln // page)):
            cache.v_scale[int(table[i, p]), :, :min(page, ln - p * page)].mul_(2.0 ** (top - 3))   # |v| < 8
    _check(ave.paged_attention(q, cache, table, n), q, cache, table, n)
