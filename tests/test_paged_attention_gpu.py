"""Attention of the newest tokens over a paged cache against float64.

Bounds, with A the mean of |v| under the softmax: a score's fp32 sum errs by some 2^-24 (D / 32 + 32) of
sum |q k| scale, under 2^-14 for rows like these; P is held in two parts (2^-16 of it in bf16, 2^-22 in
fp16) or, for a bf16 output over 8 bits, in one fp16 part: 2^-13 A, with one part 2^-11 A + 2^-13 A, and half a
step of the output's type.  (fp16 has 11 significant bits, so one rounding is off by up to half of 2^-10 of the
value, 2^-11.  Where few tokens are seen nothing averages: of a row that sees a single one, o is the rounded
P = scale of v over a power of two, times v's code, and off by up to 2^-11 of A = |v| itself.)
"""
import pytest
import torch

import avelang_amd as ave
from oracle import attn_ref as R

pytestmark = pytest.mark.gpu
BF16, F16, E4M3, I8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.int8
CODES = [(BF16, BF16), (F16, F16), (BF16, E4M3), (F16, E4M3), (BF16, I8), (F16, I8)]


def _case(lens, L, Hq, H, D, page, t, code, seed=0, spare=3):
    """q, cache, table, lengths on the GPU; rows that no sequence has hold NaN."""
    gen = torch.Generator().manual_seed(seed + len(lens) + L)
    need = [-(-max(n, 0) // page) for n in lens]
    pages = sum(need) + spare
    table = torch.full((len(lens), max(need + [1])), -7, dtype=torch.int32)
    order = torch.randperm(pages, generator=gen).int()
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    cache = ave.PagedKVCache.zeros(pages, page, H, D, code)
    for x in (cache.k, cache.v):
        if code is I8:
            x.fill_(99)
        else:
            x.view(torch.uint8).fill_(0x7f if code is E4M3 else 0xff)   # NaN
    if cache.k_scale is not None:
        cache.k_scale.fill_(torch.nan)
        cache.v_scale.fill_(torch.nan)
    k, v = (torch.randn((sum(max(n, 0) for n in lens), H, D), generator=gen) for _ in "kv")
    k = (k + torch.randn((1, H, D), generator=gen)).to(t)
    v = (v + 0.5).to(t)
    slots = torch.cat([table[i, torch.arange(max(n, 0)) // page].long() * page + torch.arange(max(n, 0)) % page
                       for i, n in enumerate(lens)])
    if slots.numel():
        ave.paged_cache_write(cache, k.cuda(), v.cuda(), slots.cuda())
    q = torch.randn((len(lens), L, Hq, D), generator=gen).to(t)
    return q.cuda(), cache, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()


def _check(got, lse, q, cache, table, lens, scale=None, window=0, cap=None):
    D, page = q.shape[-1], cache.k.shape[2]
    c = [None if x is None else x.cpu() for x in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    one = cache.k.element_size() == 1 and q.dtype is BF16
    for i, n in enumerate(lens.tolist()):
        n = max(0, n if cap is None else min(n, cap))
        pages = table[i, :-(-n // page)].tolist()
        k, v = R.rows_of(c[0], c[2], pages, n), R.rows_of(c[1], c[3], pages, n)
        o, want, size = R.attention(q[i].cpu(), k, v, D ** -0.5 if scale is None else scale, window)
        off = (got[i].cpu().double() - o).abs()
        bound = size * (2 ** -13 + (2 ** -11 if one else 0)) + o.abs() * torch.finfo(q.dtype).eps / 2 + 1e-7
        assert (off <= bound).all(), (i, n, (off / bound).max())
        if lse is not None:
            x = lse[i].cpu().double()
            none = want == -torch.inf
            assert torch.equal(x == -torch.inf, none)
            assert ((x - want).abs()[~none] <= 2 ** -13 + 2 ** -22 * want.abs()[~none]).all()


@pytest.mark.parametrize("t,code", CODES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lens,L,Hq,H,page", [
    ([1], 1, 1, 1, 16), ([449], 1, 16, 2, 16), ([0, 5, 16, 17, 0, 31, 33, 128], 1, 4, 2, 16),
    ([3, 0, 130, 1, 64], 4, 6, 2, 32), ([700, 129], 5, 8, 1, 48), ([90], 3, 32, 2, 16), ([257, 40], 9, 8, 1, 64)])
def test_against_float64(rocm_device, lens, L, Hq, H, page, D, t, code):
    q, cache, table, n = _case(lens, L, Hq, H, D, page, t, code)
    o, lse = ave.paged_attention(q, cache, table, n, return_lse=True)
    assert o.dtype == t and lse.shape == q.shape[:3]
    _check(o, lse, q, cache, table, n)
    assert torch.equal(ave.paged_attention(q, cache, table, n), o)


@pytest.mark.parametrize("t,code", [(BF16, BF16), (F16, I8), (BF16, E4M3)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("window", [1, 2, 16, 33, 200, 10 ** 9])
def test_window(rocm_device, window, D, t, code):
    q, cache, table, n = _case([1, 300, 40, 515, 2], 3, 4, 2, D, 16, t, code, seed=5)
    o, lse = ave.paged_attention(q, cache, table, n, 0.11, window=window, return_lse=True)
    _check(o, lse, q, cache, table, n, 0.11, window)


@pytest.mark.parametrize("t,code", CODES)
def test_long_and_uneven(rocm_device, t, code):
    """Lengths that are cut over many workgroups beside ones that share one."""
    lens = [9000, 1, 130, 0, 4097, 64, 5, 2000] + [7] * 300 + [3333]
    q, cache, table, n = _case(lens, 1, 4, 2, 128, 16, t, code, seed=8)
    o, lse = ave.paged_attention(q, cache, table, n, return_lse=True)
    _check(o, lse, q, cache, table, n)


@pytest.mark.parametrize("t,code", CODES)
@pytest.mark.parametrize("D,most", [(128, 18), (64, 100), (128, 400), (256, 100), (128, 1100)])
def test_many_short(rocm_device, D, most, t, code):
    """More sequences than workgroups, of a few units each or of one, a wave to each or in shares."""
    lens = [(7 * i) % most + (i % 5 != 0) for i in range(530)]
    q, cache, table, n = _case(lens, 1, 4, 2, D, 16, t, code, seed=3)
    o, lse = ave.paged_attention(q, cache, table, n, return_lse=True)
    _check(o, lse, q, cache, table, n)


@pytest.mark.parametrize("t,code", [(BF16, BF16), (F16, I8), (BF16, E4M3)])
@pytest.mark.parametrize("L,window", [(3, 0), (2, 40)])
def test_many_short_drafts(rocm_device, L, window, t, code):
    lens = [(11 * i) % 150 for i in range(520)]
    q, cache, table, n = _case(lens, L, 8, 2, 64, 16, t, code, seed=6)
    o, lse = ave.paged_attention(q, cache, table, n, window=window, return_lse=True)
    _check(o, lse, q, cache, table, n, None, window)
    # a draft's value that is not finite stays out of the rows ahead of it
    if code in (BF16, F16):
        base = ave.paged_attention(q, cache, table, n)
        at = [i for i, ln in enumerate(lens) if ln >= L]
        for i in at:
            cache.v[int(table[i, (lens[i] - 1) // 16]), 1, (lens[i] - 1) % 16, 7] = torch.nan
        o = ave.paged_attention(q, cache, table, n)
        assert torch.equal(o[at][:, :-1], base[at][:, :-1]) and o[at][:, -1, 4:, 7].isnan().all()


@pytest.mark.parametrize("t,code", CODES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("L,Hq,window", [(1, 8, 0), (3, 8, 0), (5, 8, 33), (9, 8, 0), (20, 4, 70)])
def test_few_units(rocm_device, L, Hq, window, D, t, code):
    """Sequences of two units at most, which one workgroup takes whole."""
    q, cache, table, n = _case([256, 0, 129, 128, 1, 2, 17, 255, 200], L, Hq, 2, D, 16, t, code, seed=9)
    o, lse = ave.paged_attention(q, cache, table, n, window=window, return_lse=True)
    _check(o, lse, q, cache, table, n, None, window)


@pytest.mark.parametrize("t,code", CODES)
@pytest.mark.parametrize("D,N", [(64, 61), (128, 61), (256, 30)])
def test_whole_sequences(rocm_device, D, N, t, code):
    """Several units each, as many sequences as leave nothing to share out."""
    lens = [(197 * i) % 880 + 1 for i in range(N)]
    q, cache, table, n = _case(lens, 1, 16, 8, D, 16, t, code, seed=4)
    o, lse = ave.paged_attention(q, cache, table, n, return_lse=True)
    _check(o, lse, q, cache, table, n)


@pytest.mark.parametrize("t,code", [(BF16, BF16), (F16, E4M3), (BF16, I8)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("L,window", [(1, 0), (3, 0), (5, 300), (12, 0)])
def test_shares(rocm_device, L, window, D, t, code):
    """Shares of several units that begin and end inside sequences, beside many short ones."""
    lens = [7300, 1, 130, 0, 3097] + [9 + i % 150 for i in range(120)] + [2500]
    q, cache, table, n = _case(lens, L, 16, 4, D, 16, t, code, seed=12)
    o, lse = ave.paged_attention(q, cache, table, n, window=window, return_lse=True)
    _check(o, lse, q, cache, table, n, None, window)


@pytest.mark.parametrize("L,Hq,H", [(16, 8, 2), (64, 4, 1), (40, 16, 2)])
def test_many_rows(rocm_device, L, Hq, H):
    """More rows to a kv-head than the waves of one workgroup take."""
    q, cache, table, n = _case([100, 17, 3, 700], L, Hq, H, 64, 32, BF16, BF16, seed=2)
    o, lse = ave.paged_attention(q, cache, table, n, return_lse=True)
    _check(o, lse, q, cache, table, n)


@pytest.mark.parametrize("t,code", [(BF16, BF16), (F16, F16), (BF16, E4M3), (BF16, I8)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_values_that_are_not_finite(rocm_device, D, t, code):
    """Draft tokens' infinities and NaN stay out of the rows that do not see them, and reach those that do."""
    lens = [200, 40, 4]
    q, cache, table, n = _case(lens, 4, 4, 2, D, 16, t, code, seed=4)
    base = ave.paged_attention(q, cache, table, n)
    for i, ln in enumerate(lens):
        p = ln - 2   # position of row 2 of 4: seen by rows 2 and 3
        page, row = int(table[i, p // 16]), p % 16
        for x, s in ((cache.v, cache.v_scale), (cache.k, cache.k_scale)):
            if s is not None:
                s[page, 1, row] = torch.nan
            else:
                x[page, 1, row, :3] = torch.tensor([torch.nan, torch.inf, -torch.inf]).to(t)
    o = ave.paged_attention(q, cache, table, n)
    assert torch.equal(o[:, :2], base[:, :2]) and torch.equal(o[:, :, :2], base[:, :, :2])
    assert o[:, 2:, 2:].isnan().all()
    # only v: its own columns alone
    if code in (BF16, F16):
        q, cache, table, n = _case(lens, 4, 4, 2, D, 16, t, code, seed=4)
        for i, ln in enumerate(lens):
            cache.v[int(table[i, (ln - 2) // 16]), 1, (ln - 2) % 16, 5] = torch.inf
        o = ave.paged_attention(q, cache, table, n)
        keep = torch.arange(D, device="cuda") != 5
        assert torch.equal(o[..., keep], base[..., keep]) and not o[:, 2:, 2:, 5].isfinite().any()


def test_broken_pages_and_lengths(rocm_device):
    """A page outside the cache, lengths below 0 and past the table."""
    q, cache, table, n = _case([100, 60, 500], 1, 4, 2, 128, 16, BF16, BF16)
    good = ave.paged_attention(q, cache, table, n)
    for bad in (-1, cache.k.shape[0], 2 ** 31 - 1, -2 ** 31):
        t = table.clone()
        t[2, 3] = bad
        o = ave.paged_attention(q, cache, t, n)
        assert torch.equal(o[:2], good[:2]) and o[2].isnan().all()
    m = torch.tensor([-3, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")
    table[1] = table[2]
    o, lse = ave.paged_attention(q, cache, table, m, max_length=450, return_lse=True)
    assert not o[0].any() and not o[2].any() and (lse[0] == -torch.inf).all()
    _check(o[1:2], lse[1:2], q[1:2], cache, table[1:2], torch.tensor([450]))


def test_strides(rocm_device):
    q, cache, table, n = _case([100, 60, 37], 2, 4, 2, 128, 16, BF16, I8)
    want = ave.paged_attention(q, cache, table, n)
    wide = torch.zeros(3, 2, 4 * 128 + 24, device="cuda").bfloat16()
    wide[..., 8:520] = q.flatten(2)
    assert torch.equal(ave.paged_attention(wide[..., 8:520].unflatten(-1, (4, 128)), cache, table, n), want)
    odd = torch.zeros(3, 2, 4 * 128 + 3, device="cuda").bfloat16()
    odd[..., 3:] = q.flatten(2)
    assert torch.equal(ave.paged_attention(odd[..., 3:].unflatten(-1, (4, 128)), cache, table, n), want)
    qt = q.transpose(1, 2).contiguous().transpose(1, 2)
    big = torch.full((6, 40), -1, dtype=torch.int32, device="cuda")
    big[::2, :table.shape[1]] = table
    assert torch.equal(ave.paged_attention(qt, cache, big[::2], n), want)
    assert torch.equal(ave.paged_attention(q, cache, big[::2, :table.shape[1]], n), want)
    assert torch.equal(ave.paged_attention(q, cache, table.T.contiguous().T, torch.stack([n, n], 1)[:, 0]), want)
    for i in range(3):   # one sequence alone: strides of an axis of one
        one = ave.paged_attention(q[i:i + 1], cache, table[i:i + 1], n[i:i + 1])
        assert (one[0].float() - want[i].float()).abs().max() <= 2 ** -7 * want.abs().max()
    out = torch.empty_like(q)
    ws = torch.empty(ave.paged_attention_workspace_bytes(3, 2, 4, 2, 128, table.shape[1] * 16), dtype=torch.uint8,
                     device="cuda")
    assert ave.paged_attention(q, cache, table, n, out=out, workspace=ws) is out and torch.equal(out, want)


def test_nothing(rocm_device):
    cache = ave.PagedKVCache.zeros(2, 16, 2, 64)
    q = torch.randn(3, 1, 4, 64, device="cuda").bfloat16()
    i32 = dict(dtype=torch.int32, device="cuda")
    o, lse = ave.paged_attention(q, cache, torch.empty(3, 0, **i32), torch.zeros(3, **i32), return_lse=True)
    assert not o.any() and (lse == -torch.inf).all()
    assert ave.paged_attention(q[:0], cache, torch.empty(0, 2, **i32), torch.zeros(0, **i32)).shape == (0, 1, 4, 64)


def test_far_pages(rocm_device):
    """Pages past 2^32 bytes of a cache."""
    pages, page = 9000, 1024
    cache = ave.PagedKVCache.zeros(pages, page, 1, 256)    # 4.7e9 bytes each
    gen = torch.Generator("cuda").manual_seed(1)
    for p in (0, 4, pages - 1):
        cache.k[p].normal_(generator=gen)
        cache.v[p].normal_(generator=gen)
    q = torch.randn(1, 1, 4, 256, device="cuda", generator=gen).bfloat16()
    far = torch.tensor([[pages - 1, 4, 0]], dtype=torch.int32, device="cuda")
    n = torch.tensor([2 * page + 77], dtype=torch.int32, device="cuda")
    o = ave.paged_attention(q, cache, far, n)
    near = ave.PagedKVCache(*(x[[pages - 1, 4, 0]] for x in (cache.k, cache.v)))
    assert torch.equal(o, ave.paged_attention(q, near, torch.tensor([[0, 1, 2]], dtype=torch.int32).cuda(), n))
    _check(o, None, q, near, torch.tensor([[0, 1, 2]]), n)


def test_captured(rocm_device):
    """Captured once, replayed as the lengths grow, beside eager calls; another stream."""
    q, cache, table, n = _case([400, 77, 200, 1], 1, 8, 2, 128, 16, BF16, E4M3)
    ave.paged_attention(q, cache, table, n)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = ave.paged_attention(q, cache, table, n)
    for lens in ([400, 77, 200, 1], [3, 50, 0, 1], [399, 1, 1, 0]):
        n.copy_(torch.tensor(lens))
        q.normal_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, ave.paged_attention(q, cache, table, n))
        _check(o, None, q, cache, table, n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        p = ave.paged_attention(q, cache, table, n)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o, p)
