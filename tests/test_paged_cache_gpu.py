"""The paged cache: rows written in their type or in 8 bits and read back, bit for bit what rounding the
exact quotients gives."""
import pytest
import torch

import avelang_amd as ave
from oracle import attn_ref as R

pytestmark = pytest.mark.gpu
BF16, F16, E4M3, I8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.int8
CODES = [(BF16, BF16), (F16, F16), (BF16, E4M3), (F16, E4M3), (BF16, I8), (F16, I8)]


def _rows(T, H, D, t, seed=0):
    gen = torch.Generator().manual_seed(seed + T)
    size = torch.exp2(torch.randint(-20, 10, (T, H, 1), generator=gen).float())
    return tuple((torch.randn((T, H, D), generator=gen) * size).to(t) for _ in "kv")


def _bits(t):
    return t.view(torch.uint8 if t.element_size() == 1 else torch.int16)


@pytest.mark.parametrize("t,code", CODES)
@pytest.mark.parametrize("T,H,D,page", [(1, 1, 64, 1), (1, 2, 256, 16), (37, 3, 128, 16), (300, 8, 64, 48),
                                        (515, 2, 128, 7), (2000, 1, 256, 128)])
def test_write_and_read(rocm_device, T, H, D, page, t, code):
    k, v = _rows(T, H, D, t)
    if T > 20:
        k[3], v[5, 0] = 0, 0
    pages = -(-T // page) + 2
    cache = ave.PagedKVCache.zeros(pages, page, H, D, code)
    mark = 0x55 if code in R.MOST else 0x5555
    for x in (cache.k, cache.v):
        _bits(x).fill_(mark)
    gen = torch.Generator().manual_seed(D)
    slots = torch.randperm(pages * page, generator=gen)[:T]
    if T > 9:   # padding tokens: before the cache and behind it
        slots[7], slots[9] = -1, pages * page
    ave.paged_cache_write(cache, k.cuda(), v.cuda(), slots.cuda())
    used = (slots >= 0) & (slots < pages * page)
    at, rows = slots[used], torch.arange(pages * page)
    free = rows[~torch.isin(rows, at)]
    for x, c, s in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        c = _bits(c).cpu().transpose(1, 2).reshape(pages * page, H, D)
        assert (c[free] == mark).all()
        if code not in R.MOST:
            assert torch.equal(c[at], _bits(x)[used])
            continue
        want, scale = R.codes(x[used], code)
        assert torch.equal(c[at].view(code).double(), want)
        s = s.cpu().transpose(1, 2).reshape(-1, H)
        assert torch.equal(s[at], scale) and not s[free].any()
    for dt in {t, BF16 if code in R.MOST else t}:
        got = ave.paged_cache_read(cache, slots.int().cuda(), dt)
        for x, y in zip((k, v), got):
            assert y.dtype == dt and not y[~used.cuda()].any()
            if code not in R.MOST:
                assert torch.equal(y.cpu()[used], x[used])
            else:
                want, scale = R.codes(x[used], code)
                assert torch.equal(y.cpu()[used], (want.float() * scale[..., None]).to(dt))


@pytest.mark.parametrize("code", [E4M3, I8])
def test_ties_and_extremes(rocm_device, code):
    """Quotients that lie on a border between codes, at every size of row."""
    D, M = 64, R.MOST[code]
    rows = []
    for e in (-99, -30, 0, 60, 127):
        for most in (1.0, 1.75, 1.09375, 1.9921875):   # 1.75 = 7/4: the exact quotients of many bf16 values are ties
            x = torch.linspace(-1, 1, D, dtype=torch.float64) * most
            x[0] = most
            rows.append(x * 2.0 ** e)
    mid = (torch.arange(64, dtype=torch.float64) + 0.5) / M * 1.75   # half codes of a row whose largest is 1.75
    mid[0] = 1.75
    rows.append(mid)
    k = torch.stack(rows).to(BF16)[:, None]
    T = len(rows)
    cache = ave.PagedKVCache.zeros(T, 1, 1, D, code)
    ave.paged_cache_write(cache, k.cuda(), k.cuda(), torch.arange(T).cuda())
    want, scale = R.codes(k, code)
    assert torch.equal(cache.k.cpu().double()[:, :, 0], want) and torch.equal(cache.k_scale.cpu()[:, :, 0], scale)


@pytest.mark.parametrize("code", [E4M3, I8])
def test_small_and_broken_rows(rocm_device, code):
    k = torch.randn(5, 1, 64).to(BF16)
    k[0], k[1, 0, 3], k[2, 0, 5] = 1e-35, torch.inf, torch.nan
    k[3] = 0
    cache = ave.PagedKVCache.zeros(1, 16, 1, 64, code)
    ave.paged_cache_write(cache, k.cuda(), k.cuda(), torch.arange(5).cuda())
    s = cache.k_scale.cpu()[0, 0]
    assert s[0] == torch.tensor(2.0 ** -100) / R.MOST[code] and s[3] == 0
    assert s[1].isnan() and s[2].isnan()
    back = ave.paged_cache_read(cache, torch.arange(5).cuda())[0].cpu()
    assert back[1].isnan().all() and back[2].isnan().all() and not back[3].any()
    # half a step of a row whose largest value is 2^-100 (and back's own rounding)
    half = s[0].double() * (2 ** -10 if code is E4M3 else 0.5)
    assert ((back[0].double() - k[0].double()).abs() <= half + k[0].double() * 2 ** -8).all()
    want, scale = R.codes(k[4:], code)
    assert torch.equal(back[4:], (want.float() * scale[..., None]).to(BF16))


def test_layouts(rocm_device):
    """Column slices, [B, T] slots on the CPU, heads ahead of tokens, an odd start."""
    B, T, H, D = 2, 6, 2, 128
    y = torch.randn(B, T, 2 * H * D + 5, device="cuda").bfloat16()[..., 5:]
    k, v = (x.unflatten(-1, (H, D)) for x in y.split(H * D, -1))
    slots = torch.randperm(B * T).view(B, T)
    a, b, c = (ave.PagedKVCache.zeros(2, 16, H, D, I8) for _ in "abc")
    ave.paged_cache_write(a, k.contiguous(), v.contiguous(), slots.cuda())
    ave.paged_cache_write(b, k, v, slots)
    t = lambda x: x[0].transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    for i in range(B):
        x = [z[i].transpose(0, 1).contiguous().transpose(0, 1) for z in (k, v)]
        ave.paged_cache_write(c, *x, slots[i].int().cuda())
    for p in (b, c):
        assert torch.equal(a.k, p.k) and torch.equal(a.v, p.v) and torch.equal(a.k_scale, p.k_scale)
    got = ave.paged_cache_read(a, slots)
    assert got[0].shape == (B, T, H, D)
    ave.paged_cache_write(a, k[:0], v[:0], slots[:0])
    assert ave.paged_cache_read(a, slots[0, :0])[1].shape == (0, H, D)


def test_far_slots(rocm_device):
    """Rows past 2^32 bytes of a cache."""
    pages = 70000
    cache = ave.PagedKVCache.zeros(pages, 256, 1, 256, I8)    # 4.6e9 bytes each
    k, v = _rows(4, 1, 256, BF16)
    slots = torch.tensor([0, pages * 256 - 1, 2 ** 24 + 1, 2 ** 24 - 1])
    ave.paged_cache_write(cache, k.cuda(), v.cuda(), slots.cuda())
    for x, y in zip((k, v), ave.paged_cache_read(cache, slots.cuda())):
        want, scale = R.codes(x, I8)
        assert torch.equal(y.cpu(), (want.float() * scale[..., None]).to(BF16))


def test_captured(rocm_device):
    """A captured write and read, replayed over other rows."""
    H, D, T = 2, 128, 33
    cache = ave.PagedKVCache.zeros(8, 16, H, D, E4M3)
    k, v = (x.cuda() for x in _rows(T, H, D, BF16))
    slots = torch.randperm(128)[:T].cuda()
    g = torch.cuda.CUDAGraph()
    ave.paged_cache_write(cache, k, v, slots)
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        ave.paged_cache_write(cache, k, v, slots)
        out = ave.paged_cache_read(cache, slots)
    for i in range(3):
        k2, v2 = (x.cuda() for x in _rows(T, H, D, BF16, seed=9 + i))
        k.copy_(k2)
        v.copy_(v2)
        slots.copy_(torch.randperm(128)[:T])
        g.replay()
        torch.cuda.synchronize()
        other = ave.PagedKVCache.zeros(8, 16, H, D, E4M3)
        ave.paged_cache_write(other, k2, v2, slots)
        assert all(torch.equal(a, b) for a, b in zip(out, ave.paged_cache_read(other, slots)))


@pytest.mark.parametrize("t,code", [(BF16, E4M3), (F16, I8), (BF16, I8), (F16, E4M3), (BF16, BF16)])
@pytest.mark.parametrize("T,H,D", [(33001, 1, 256), (13121, 5, 128), (43713, 3, 64)])
def test_many_rows(rocm_device, T, H, D, t, code):
    """Sizes at which a group of lanes takes two rows: padding among them, the last one alone."""
    k, v = _rows(T, H, D, t)
    page = 48
    pages = -(-T // page) + 1
    cache = ave.PagedKVCache.zeros(pages, page, H, D, code)
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(D))[:T]
    slots[5::1009], slots[11::1511] = -3, pages * page + 7
    ave.paged_cache_write(cache, k.cuda(), v.cuda(), slots.cuda())
    used = (slots >= 0) & (slots < pages * page)
    rows = torch.arange(pages * page)
    free = rows[~torch.isin(rows, slots[used])]
    got = ave.paged_cache_read(cache, slots.cuda(), t)
    for x, c, s, y in ((k, cache.k, cache.k_scale, got[0]), (v, cache.v, cache.v_scale, got[1])):
        c = _bits(c).cpu().transpose(1, 2).reshape(pages * page, H, D)
        assert not c[free].any() and not y[~used.cuda()].any()
        if code not in R.MOST:
            assert torch.equal(c[slots[used]], _bits(x)[used]) and torch.equal(y.cpu()[used], x[used])
            continue
        want, scale = R.codes(x[used], code)
        assert torch.equal(c[slots[used]].view(code).double(), want)
        assert torch.equal(s.cpu().transpose(1, 2).reshape(-1, H)[slots[used]], scale)
        assert torch.equal(y.cpu()[used], (want.float() * scale[..., None]).to(t))
