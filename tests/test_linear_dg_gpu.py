"""The decay's gradient, and what the saved states hold.

dg is a sum of products of random signs, which shows every operand's rounding: the saved states' is
at most 2^-9 of a value (nine bits after the leading one; both parts of D 2^-16, everything else
fp32).  Independent roundings add up by their root mean square, under half the largest: 2^-10 in the
norm, and dg's own rounding to its type beside it.  dq is rounded once and holds dP rounded once,
2^-8 each: 2^-8 in the norm.
"""
import pytest
import torch

from oracle import linear_ref

BF = torch.bfloat16
pytestmark = pytest.mark.gpu


def make(dev, B, T, Hqk, Hv, K, V, g_dtype=torch.float32, N=None, seed=0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen, device=dev)  # noqa: E731
    return dict(q=r(B, T, Hqk, K).to(BF), k=r(B, T, Hqk, K).to(BF), v=r(B, T, Hv, V).to(BF),
                g=(-torch.exp(2 * r(B, T, Hv) - 3)).to(g_dtype), h0=3 * r(N or B, Hv, K, V),
                do=r(B, T, Hv, V).to(BF), dht=r(N or B, Hv, K, V))


def far(x, ref):
    assert x.shape == ref.shape and torch.isfinite(x).all()
    return ((x.double() - ref).norm() / ref.norm()).item()


SHAPES = [(1, 1, 16, 32, 128, 128), (1, 4, 16, 32, 64, 64), (1, 5, 32, 32, 128, 128), (3, 40, 4, 16, 64, 128),
          (1, 110, 4, 16, 128, 64), (2, 196, 2, 8, 64, 64), (1, 1294, 16, 32, 64, 64), (1, 1753, 16, 16, 128, 64),
          (1, 1400, 16, 32, 128, 128), (1, 449, 1, 3, 128, 128), (1, 6200, 16, 32, 128, 128)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("h0", [True, False])
@pytest.mark.parametrize("g_dtype", [torch.float32, BF])
def test_decay_gradient(rocm_device, shape, h0, g_dtype):
    import avelang_amd as ave
    if shape[1] < 40 and not h0:   # (nothing has been rounded yet)
        return
    t = make(rocm_device, *shape, g_dtype=g_dtype)
    h0 = t["h0"] if h0 else None
    want = linear_ref.linear_attn_chunked(t["q"], t["k"], t["v"], t["g"], t["do"], t["dht"], h0=h0)[5]
    dg = ave.chunk_linear_attn_bwd(t["q"], t["k"], t["v"], t["g"], t["do"], t["dht"], initial_state=h0)[3]
    own = far(want.to(g_dtype), want)
    assert dg.dtype == g_dtype and far(dg, want) <= (own ** 2 + 2.0 ** -20) ** 0.5


def test_packed(rocm_device):
    import avelang_amd as ave
    lens = [700, 0, 65, 1, 934]
    cu = [sum(lens[:i]) for i in range(6)]
    t = make(rocm_device, 1, 1700, 16, 32, 128, 128, N=5)
    want = linear_ref.linear_attn_chunked(t["q"], t["k"], t["v"], t["g"], t["do"], t["dht"], h0=t["h0"], cu=cu)[5]
    dg = ave.chunk_linear_attn_bwd(t["q"], t["k"], t["v"], t["g"], t["do"], t["dht"], initial_state=t["h0"],
                                   cu_seqlens=torch.tensor(cu, device=rocm_device))[3]
    assert far(dg, want) <= 2 ** -10


@pytest.mark.parametrize("T", [70, 1400])
@pytest.mark.parametrize("scale", ["channels", "huge", "tiny"])
def test_states_of_any_size(rocm_device, scale, T):
    """Neighbouring value channels of sizes 1 to 4096, states of 2^60 and of 2^-60: each channel's
    share of dq and dg is as good as the others' (do makes them alike)."""
    import avelang_amd as ave
    t = make(rocm_device, 1, T, 4, 8, 128, 128, seed=1)
    size = {"channels": 16.0 ** (torch.arange(128, device=rocm_device) % 4), "huge": torch.full((128,), 2.0 ** 60),
            "tiny": torch.full((128,), 2.0 ** -60)}[scale].to(rocm_device)
    t["v"], t["do"] = (t["v"] * size).to(BF), (t["do"] / size).to(BF)   # (powers of two: exact)
    t["h0"], t["dht"] = t["h0"] * size, t["dht"] / size
    want = linear_ref.linear_attn_chunked(t["q"], t["k"], t["v"], t["g"], t["do"], t["dht"], h0=t["h0"])
    dq, _, _, dg, _ = ave.chunk_linear_attn_bwd(t["q"], t["k"], t["v"], t["g"], t["do"], t["dht"],
                                                initial_state=t["h0"])
    assert far(dq, want[2]) <= 2 ** -8 and far(dg, want[5]) <= 2 ** -10


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_states_that_are_not_finite(rocm_device, bad):
    """They are saved as such: their head's gradients show it, no other's do."""
    import avelang_amd as ave
    t = make(rocm_device, 1, 100, 4, 4, 64, 128, seed=2)
    args = (t["q"], t["k"], t["v"], t["g"], t["do"])
    want = ave.chunk_linear_attn_bwd(*args, initial_state=t["h0"])
    t["h0"][0, 1, 5, 77] = bad
    got = ave.chunk_linear_attn_bwd(*args, initial_state=t["h0"])
    keep = [0, 2, 3]
    for x, y in zip(got, want):
        d = 1 if x.shape[1] == 4 else 2   # (dh0 [N, Hv, ..])
        at = torch.tensor(keep, device=rocm_device)
        assert torch.equal(x.index_select(d, at), y.index_select(d, at))
    assert not got[0][0, :, 1].isfinite().all() and not got[3][0, :, 1].isfinite().all()


@pytest.mark.parametrize("T", [1, 2, 4, 9, 16])
@pytest.mark.parametrize("heads", [(16, 32), (16, 16), (4, 12)])
@pytest.mark.parametrize("K,V", [(128, 128), (64, 64), (128, 64), (64, 128)])
@pytest.mark.parametrize("end", [False, True])
def test_few_tokens(rocm_device, T, heads, K, V, end):
    """Gradients that are sums of a few terms show their own rounding alone: P and dP enter in two
    parts within a tile of 16 tokens, and so does the final state's gradient (2^-16 of them left,
    2^-12 allowed)."""
    import avelang_amd as ave
    t = make(rocm_device, 2, T, *heads, K, V, seed=T)
    dht = t["dht"] if end else None
    want = linear_ref.linear_attn_chunked(t["q"], t["k"], t["v"], t["g"], t["do"], dht)
    got = ave.chunk_linear_attn_bwd(t["q"], t["k"], t["v"], t["g"], t["do"], dht)
    for x, ref in zip(got[:3], want[2:5]):
        assert far(x, ref) <= (far(ref.to(BF), ref) ** 2 + 2.0 ** -24) ** 0.5
