"""Linear attention in the forms that large calls take: several chunks per segment in the forward and
in the gradients, walks of 32 columns per wave, packed sequences cut into segments; against the
oracle's formulas of chunks in 64 bits.

Tolerances.  A rounding to bf16 is off by at most 2^-8 of its value.  o, dq, dk and dv are rounded
once at the end and hold operands that were rounded once, spread over many terms of either sign: 2^-8
in the norm.  States and dh0 are fp32 sums of terms in three bf16 parts (2^-24 each): a dozen such
roundings, 2^-20.  dg adds up products with one operand that was rounded, 2^-8, and in bf16 its own
rounding, together 2^-7.
"""
import pytest
import torch

from oracle import linear_ref

BF = torch.bfloat16
pytestmark = pytest.mark.gpu


def make(dev, B, T, Hqk, Hv, K, V, g="token", g_dtype=torch.float32, N=None, seed=0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen, device=dev)  # noqa: E731
    N = N or B
    gt = -torch.exp2(-8.0 * torch.arange(1, Hv + 1, device=dev) / Hv) if g == "head" else -torch.exp(2 * r(B, T, Hv) - 3)
    return dict(q=r(B, T, Hqk, K).to(BF), k=r(B, T, Hqk, K).to(BF), v=r(B, T, Hv, V).to(BF), g=gt.to(g_dtype),
                h0=3 * r(N, Hv, K, V), do=r(B, T, Hv, V).to(BF), dht=r(N, Hv, K, V))


def cu_of(lens):
    return None if lens is None else [sum(lens[:i]) for i in range(len(lens) + 1)]


def far(x, ref):
    assert x.shape == ref.shape and torch.isfinite(x).all()
    return ((x.double() - ref).norm() / ref.norm()).item()


def chunks_of(B, T, lens):
    return sum(-(-n // 64) for n in (lens or [T] * B))


# B, T, Hqk, Hv, K, V, lengths, chunks of all v-heads per CU from which a CU holds two workgroups
FORWARD = [(1, 6200, 16, 32, 128, 128, None, 12), (2, 3100, 32, 32, 128, 128, None, 12),
           (1, 4200, 8, 32, 64, 128, None, 8), (1, 2200, 16, 32, 128, 64, None, 4),
           (1, 2200, 8, 32, 64, 64, None, 4), (1, 6700, 16, 32, 128, 128, [3000, 0, 1, 2500, 64, 1135], 12),
           (1, 4300, 8, 32, 64, 128, [65, 4000, 0, 235], 8)]


@pytest.mark.parametrize("case", FORWARD, ids=lambda c: "-".join(map(str, c[:6])) + ("-packed" if c[6] else ""))
@pytest.mark.parametrize("g", ["token", "head"])
def test_forward(rocm_device, case, g):
    import avelang_amd as ave
    B, T, Hqk, Hv, K, V, lens, edge = case
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    assert chunks_of(B, T, lens) * Hv >= edge * cus
    t = make(rocm_device, *case[:6], g=g, N=len(lens) if lens else B)
    cu = cu_of(lens)
    o, ht = linear_ref.linear_attn_chunked(t["q"], t["k"], t["v"], t["g"], h0=t["h0"], cu=cu)
    args = (t["q"], t["k"], t["v"], t["g"])
    kw = dict(initial_state=t["h0"], cu_seqlens=None if cu is None else torch.tensor(cu, device=rocm_device))
    got, s = ave.chunk_linear_attn(*args, output_final_state=True, **kw)
    assert far(got, o) <= 2 ** -8 and far(s, ht) <= 2 ** -20
    got2, _ = ave.chunk_linear_attn(*args, **kw)            # o alone
    assert far(got2, o) <= 2 ** -8
    got3, s3, _ = ave.chunk_linear_attn_fwd_save(*args, output_final_state=True, **kw)
    assert far(got3, o) <= 2 ** -8 and far(s3, ht) <= 2 ** -20
    state = t["h0"].clone()
    kw["initial_state"] = state
    got4, s4 = ave.chunk_linear_attn(*args, output_final_state=True, final_state=state, **kw)
    assert s4 is state and torch.equal(got4, got) and torch.equal(s4, s)


# B, T, Hqk, Hv, K, V, lengths, chunks of all v-heads per CU from which a segment has several chunks
BACKWARD = [(1, 1400, 16, 32, 128, 128, None, 2), (1, 2000, 16, 16, 128, 128, None, 1),
            (1, 2300, 8, 24, 64, 64, None, 2), (1, 3000, 4, 16, 128, 64, None, 2),
            (2, 1300, 16, 32, 64, 128, None, 2), (1, 6200, 16, 32, 128, 128, None, 2),
            (1, 4100, 8, 16, 64, 64, None, 4),
            (1, 1700, 16, 32, 128, 128, [700, 0, 65, 1, 934], 2),
            (1, 2400, 16, 16, 64, 128, [2001, 399], 1), (1, 3400, 4, 16, 128, 64, [130, 3000, 270], 2)]


@pytest.mark.parametrize("case", BACKWARD, ids=lambda c: "-".join(map(str, c[:6])) + ("-packed" if c[6] else ""))
@pytest.mark.parametrize("g,g_dtype,h0", [("token", torch.float32, True), ("token", BF, False),
                                          ("head", torch.float32, True)])
def test_gradients(rocm_device, case, g, g_dtype, h0):
    import avelang_amd as ave
    B, T, Hqk, Hv, K, V, lens, edge = case
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    assert chunks_of(B, T, lens) * Hv > edge * cus
    t = make(rocm_device, *case[:6], g=g, g_dtype=g_dtype, N=len(lens) if lens else B, seed=3)
    cu = cu_of(lens)
    want = linear_ref.linear_attn_chunked(t["q"], t["k"], t["v"], t["g"], t["do"], t["dht"],
                                          h0=t["h0"] if h0 else None, cu=cu)
    names = ["q", "k", "v", "g"] + ["h0"] * h0
    mine = [t[n].clone().requires_grad_() for n in names]
    kw = dict(cu_seqlens=None if cu is None else torch.tensor(cu, device=rocm_device))
    o, ht = ave.chunk_linear_attn(*mine[:4], initial_state=mine[4] if h0 else None, output_final_state=True, **kw)
    got = torch.autograd.grad([o, ht], mine, [t["do"], t["dht"]])
    assert far(o.detach(), want[0]) <= 2 ** -8 and far(ht.detach(), want[1]) <= 2 ** -20
    for n, x, ref in zip(names, got, want[2:]):
        assert x.dtype == t[n].dtype
        assert far(x, ref) <= {"g": 2 ** -7, "h0": 2 ** -20}.get(n, 2 ** -8), n
    # the states formed again give the same bits
    again = ave.chunk_linear_attn_bwd(t["q"], t["k"], t["v"], t["g"], t["do"], t["dht"],
                                      initial_state=t["h0"] if h0 else None, **kw)
    assert all(torch.equal(x, y) for x, y in zip(again, got))


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_not_finite_stays_behind(rocm_device, bad):
    """As in the forms of short calls: every earlier token's output keeps its bits."""
    import avelang_amd as ave
    t = make(rocm_device, 1, 6200, 16, 32, 128, 128, seed=12)
    want = ave.chunk_linear_attn(t["q"], t["k"], t["v"], t["g"], initial_state=t["h0"])[0]
    for n in ("q", "k", "v", "g"):
        for at in (0, 33, 1000, 3007, 6199):
            x = t[n].clone()
            x[0, at, 0] = bad
            got = ave.chunk_linear_attn(*(x if m == n else t[m] for m in ("q", "k", "v", "g")),
                                        initial_state=t["h0"])[0]
            assert torch.equal(got[0, :at], want[0, :at]), (n, at)
            assert not got[0, at, 0].isfinite().all()
            assert torch.equal(got[0, :, 2:], want[0, :, 2:])   # (v-heads 0 and 1 share a qk-head)
            if n == "q":
                assert torch.equal(got[0, at + 1:], want[0, at + 1:])
