"""Linear attention with a decay per head against the 64-bit token recurrence.

Tolerances.  A rounding to bf16 is off by at most 2^-8 of its value.  o, dq, dk
and dv are rounded once at the end and hold up to two operands that were
rounded once (P and the state), each spread over at least some sixteen terms of
either sign: their differences are at most 2^-8 of the result in the norm, and
element by element 2^-8 of the result and of the sum of the terms' sizes.  The
states and dh0 are fp32 sums of terms in two bf16 parts: 2^-16 in the norm.  dg
adds up to 128 products of operands rounded once: 2^-6 in the norm.
"""
import pytest
import torch

from oracle import linear_ref

BF = torch.bfloat16


def make(B, T, Hqk, Hv, K, V, seed=0, g="token", g_dtype=torch.float32, h0=True, lens=None):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    q, k, v = r(B, T, Hqk, K).to(BF), r(B, T, Hqk, K).to(BF), r(B, T, Hv, V).to(BF)
    if g == "head":
        gt = -torch.exp2(-8.0 * torch.arange(1, Hv + 1) / Hv)
    else:
        gt = -torch.exp(2 * r(B, T, Hv) - 3)
    N = B if lens is None else len(lens)
    return dict(q=q, k=k, v=v, g=gt.to(g_dtype), h0=3 * r(N, Hv, K, V) if h0 else None,
                do=r(B, T, Hv, V).to(BF), dht=r(N, Hv, K, V))


def cu_of(lens):
    cu = [0]
    for x in lens:
        cu.append(cu[-1] + x)
    return cu


def far(x, ref):
    x, ref = x.detach().double().cpu(), ref.detach().double()
    assert x.shape == ref.shape and torch.isfinite(x).all()
    return ((x - ref).norm() / ref.norm().clamp_min(1e-30)).item()


def to(d, dev):
    return {n: x.to(dev) if isinstance(x, torch.Tensor) else x for n, x in d.items()}


SHAPES = [  # B, T, Hqk, Hv, K, V
    (1, 1, 1, 1, 64, 64), (2, 2, 1, 2, 128, 64), (1, 63, 2, 4, 64, 128), (1, 64, 1, 1, 128, 128),
    (3, 65, 1, 3, 64, 64), (1, 200, 2, 4, 128, 128), (1, 449, 1, 2, 128, 64),
    (2, 577, 2, 2, 64, 128), (1, 1100, 1, 4, 128, 128),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("g,h0", [("token", True), ("head", False)])
def test_chunk_forward(rocm_device, shape, g, h0):
    import avelang_amd as ave
    d = make(*shape, g=g, h0=h0)
    o, ht = linear_ref.linear_attn(d["q"], d["k"], d["v"], d["g"], h0=d["h0"])
    t = to(d, rocm_device)
    got, s = ave.chunk_linear_attn(t["q"], t["k"], t["v"], t["g"], initial_state=t["h0"],
                                   output_final_state=True)
    assert got.dtype == BF and s.dtype == torch.float32
    assert far(got, o) <= 2 ** -8
    assert far(s, ht) <= 2 ** -16
    o_abs, _ = linear_ref.linear_attn(*(d[n].abs() for n in "qkv"), d["g"],
                                      h0=None if d["h0"] is None else d["h0"].abs())
    assert ((got.double().cpu() - o).abs() <= 2 ** -8 * (o.abs() + 1.01 * o_abs) + 1e-30).all()


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[1], [0, 3, 0], [64, 1, 65, 300, 0, 17], [700, 0, 5, 600]])
@pytest.mark.parametrize("heads", [(1, 1), (2, 4)])
def test_packed(rocm_device, lens, heads):
    import avelang_amd as ave
    cu = cu_of(lens)
    d = make(1, cu[-1], *heads, 64, 128, seed=len(lens), lens=lens)
    t = to(d, rocm_device)
    o, ht = linear_ref.linear_attn(d["q"], d["k"], d["v"], d["g"], h0=d["h0"], cu=cu)
    for where in (rocm_device, "cpu"):
        for op in (ave.chunk_linear_attn, ave.fused_recurrent_linear_attn):
            kw = {} if op is ave.chunk_linear_attn else dict(inplace_final_state=False)
            got, s = op(t["q"], t["k"], t["v"], t["g"], initial_state=t["h0"],
                        output_final_state=True,
                        cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=where), **kw)
            assert far(got, o) <= 2 ** -8
            assert far(s, ht) <= 2 ** -16


@pytest.mark.gpu
def test_cu_violation_empties(rocm_device):
    import avelang_amd as ave
    t = to(make(1, 130, 1, 2, 64, 64, lens=[0, 0]), rocm_device)
    for cu in ([0, 140, 130], [1, 64, 130], [0, 64, 129]):
        cu = torch.tensor(cu, dtype=torch.int32, device=rocm_device)
        o, ht = ave.chunk_linear_attn(t["q"], t["k"], t["v"], t["g"], initial_state=t["h0"],
                                      output_final_state=True, cu_seqlens=cu)
        assert (o == 0).all() and torch.equal(ht, t["h0"])
        for x in ave.chunk_linear_attn_bwd(t["q"], t["k"], t["v"], t["g"], t["do"], t["dht"],
                                           initial_state=t["h0"], cu_seqlens=cu)[:4]:
            assert (x == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 64, 64), (1, 70, 1, 2, 128, 64), (2, 65, 2, 2, 64, 128),
                                   (1, 330, 1, 4, 128, 128), (1, 600, 2, 6, 64, 64),
                                   (1, 577, 1, 1, 128, 128)])
@pytest.mark.parametrize("g,h0,g_dtype", [("token", True, torch.float32), ("token", False, BF),
                                          ("head", True, torch.float32)])
def test_gradients(rocm_device, shape, g, h0, g_dtype):
    import avelang_amd as ave
    d = make(*shape, g=g, h0=h0, g_dtype=g_dtype, seed=3)
    names = ["q", "k", "v", "g"] + (["h0"] if h0 else [])
    leaves = [d[n].double().requires_grad_() for n in names]
    o, ht = linear_ref.linear_attn(*leaves[:4], h0=leaves[4] if h0 else None)
    want = torch.autograd.grad([o, ht], leaves, [d["do"].double(), d["dht"].double()])
    t = to(d, rocm_device)
    mine = [t[n].clone().requires_grad_() for n in names]
    o2, h2 = ave.chunk_linear_attn(*mine[:4], initial_state=mine[4] if h0 else None,
                                   output_final_state=True)
    got = torch.autograd.grad([o2, h2], mine, [t["do"], t["dht"]])
    assert far(o2, o) <= 2 ** -8 and far(h2, ht) <= 2 ** -16
    for n, x, ref in zip(names, got, want):
        assert x.dtype == d[n].dtype and x.shape == d[n].shape
        assert far(x, ref) <= {"g": 2 ** -6, "h0": 2 ** -16}.get(n, 2 ** -8), n
    # the states formed again, and twice the same bits
    kw = dict(initial_state=t["h0"])
    a = ave.chunk_linear_attn_bwd(t["q"], t["k"], t["v"], t["g"], t["do"], t["dht"], **kw)
    for x, y in zip(a, got):
        assert torch.equal(x.to(y.dtype), y)


@pytest.mark.gpu
def test_gradients_packed(rocm_device):
    import avelang_amd as ave
    lens = [70, 0, 1, 330, 64]
    cu = cu_of(lens)
    d = make(1, cu[-1], 2, 4, 128, 64, seed=5, lens=lens)
    leaves = [d[n].double().requires_grad_() for n in ("q", "k", "v", "g", "h0")]
    o, ht = linear_ref.linear_attn(*leaves[:4], h0=leaves[4], cu=cu)
    want = torch.autograd.grad([o, ht], leaves, [d["do"].double(), d["dht"].double()])
    t = to(d, rocm_device)
    mine = [t[n].clone().requires_grad_() for n in ("q", "k", "v", "g", "h0")]
    o2, h2 = ave.chunk_linear_attn(*mine[:4], initial_state=mine[4], output_final_state=True,
                                   cu_seqlens=torch.tensor(cu, device=rocm_device))
    got = torch.autograd.grad([o2, h2], mine, [t["do"], t["dht"]])
    for x, ref, tol in zip(got, want, (2 ** -8,) * 3 + (2 ** -6, 2 ** -16)):
        assert far(x, ref) <= tol


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 1, 16, 32, 128, 128), (3, 1, 1, 2, 64, 64), (2, 5, 1, 3, 128, 64),
                                   (40, 1, 2, 16, 64, 128), (17, 2, 16, 32, 128, 128)])
@pytest.mark.parametrize("g", ["token", "head"])
def test_recurrent(rocm_device, shape, g):
    import avelang_amd as ave
    d = make(*shape, g=g, g_dtype=BF if g == "token" else torch.float32)
    o, ht = linear_ref.linear_attn(d["q"], d["k"], d["v"], d["g"], h0=d["h0"])
    t = to(d, rocm_device)
    before = t["h0"].clone()
    got, s = ave.fused_recurrent_linear_attn(t["q"], t["k"], t["v"], t["g"], initial_state=t["h0"],
                                             output_final_state=True, inplace_final_state=False)
    assert far(got, o) <= 2 ** -8 and far(s, ht) <= 2 ** -20 and torch.equal(before, t["h0"])
    got2, s2 = ave.fused_recurrent_linear_attn(t["q"], t["k"], t["v"], t["g"], initial_state=t["h0"],
                                               output_final_state=True)
    assert s2 is t["h0"] and torch.equal(s2, s) and torch.equal(got, got2)


@pytest.mark.gpu
def test_slots(rocm_device):
    import avelang_amd as ave
    t = to(make(4, 1, 2, 4, 64, 128, seed=2), rocm_device)
    gen = torch.Generator().manual_seed(9)
    pool = torch.randn((6, 4, 64, 128), generator=gen).to(rocm_device)
    want_pool = pool.clone()
    idx = torch.tensor([5, 0, 7, 2], dtype=torch.int32, device=rocm_device)
    use = [0, 1, 3]
    o, s = ave.fused_recurrent_linear_attn(*(t[n][use] for n in ("q", "k", "v", "g")),
                                           initial_state=pool[idx[use].long()],
                                           output_final_state=True)
    want_pool[idx[use].long()] = s
    out = torch.full_like(t["v"], 7.0)
    got, p = ave.fused_recurrent_linear_attn(t["q"], t["k"], t["v"], t["g"], initial_state=pool,
                                             output_final_state=True, ssm_state_indices=idx, out=out)
    assert p is pool and torch.equal(pool, want_pool)
    assert torch.equal(got[use], o) and (got[2] == 7).all()
    # a slot named twice: left alone, its sequences' rows NaN, the others' as ever
    idx = torch.tensor([5, 0, 5, 2], dtype=torch.int32, device=rocm_device)
    keep = pool[5].clone()
    got, _ = ave.fused_recurrent_linear_attn(t["q"], t["k"], t["v"], t["g"], initial_state=pool,
                                             output_final_state=True, ssm_state_indices=idx)
    assert torch.equal(pool[5], keep) and got[[0, 2]].isnan().all() and got[[1, 3]].isfinite().all()


@pytest.mark.gpu
def test_decode_continues_a_prompt(rocm_device):
    """A prompt in one call, and split into two prompts and single tokens."""
    import avelang_amd as ave
    d = make(1, 300, 2, 4, 128, 128, seed=4)
    o, ht = linear_ref.linear_attn(d["q"], d["k"], d["v"], d["g"], h0=d["h0"])
    t = to(d, rocm_device)
    s, outs = t["h0"], []
    for a, b in ((0, 130), (130, 296), (296, 297), (297, 300)):
        op = ave.chunk_linear_attn if b - a > 10 else ave.fused_recurrent_linear_attn
        x, s = op(*(t[n][:, a:b] for n in ("q", "k", "v", "g")), initial_state=s.clone(),
                  output_final_state=True)
        outs.append(x)
    assert far(torch.cat(outs, 1), o) <= 2 ** -8 and far(s, ht) <= 2 ** -15


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 200])
def test_slices_in_place(rocm_device, T):
    """Column slices of one tensor give the bits of their copies."""
    import avelang_amd as ave
    y = torch.randn(2, T, 2 * 2 * 64 + 4 * 128 + 16, device=rocm_device).to(BF)
    q, k, v = (x.reshape(2, T, h, d) for x, h, d in zip(
        y[..., 8:-8].split([128, 128, 512], -1), (2, 2, 4), (64, 64, 128)))
    assert not q.is_contiguous() or T == 1
    g = -torch.rand(2, T, 4, device=rocm_device)
    for op in (ave.chunk_linear_attn, ave.fused_recurrent_linear_attn):
        a = op(q, k, v, g, output_final_state=True)
        b = op(q.contiguous(), k.contiguous(), v.contiguous(), g, output_final_state=True)
        assert all(torch.equal(x, z) for x, z in zip(a, b))
    # an odd base address, and heads that are not together
    flat = torch.randn(2 * T * 2 * 64 + 1, device=rocm_device).to(BF)
    q2 = flat[1:].view(2, T, 2, 64)
    a = ave.chunk_linear_attn(q2, k, v, g)[0]
    assert torch.equal(a, ave.chunk_linear_attn(q2.clone(), k.contiguous(), v.contiguous(), g)[0])


@pytest.mark.gpu
def test_resets_and_extremes(rocm_device):
    """-inf resets the state exactly; a sequence's NaN stays in it; large decays underflow to 0."""
    import avelang_amd as ave
    d = make(1, 150, 1, 2, 64, 64, seed=8, lens=[80, 70])
    d["g"][0, 40, 0] = -float("inf")
    d["g"][0, 90:130, 1] = -1e6
    cu = [0, 80, 150]
    o, ht = linear_ref.linear_attn(d["q"], d["k"], d["v"], d["g"], h0=d["h0"], cu=cu)
    t = to(d, rocm_device)
    args = dict(output_final_state=True, cu_seqlens=torch.tensor(cu, device=rocm_device))
    got, s = ave.chunk_linear_attn(t["q"], t["k"], t["v"], t["g"], initial_state=t["h0"], **args)
    assert far(got, o) <= 2 ** -8 and far(s, ht) <= 2 ** -16
    t["v"][0, 10] = float("nan")
    got2, s2 = ave.chunk_linear_attn(t["q"], t["k"], t["v"], t["g"], initial_state=t["h0"], **args)
    assert torch.equal(got2[0, 80:], got[0, 80:]) and torch.equal(s2[1], s[1])
    assert got2[0, 10].isnan().all()


@pytest.mark.gpu
def test_graph_replays(rocm_device):
    """Prompt, backward and decode captured into one graph, replayed with new inputs."""
    import avelang_amd as ave
    t = to(make(1, 400, 1, 2, 128, 64, seed=6), rocm_device)

    def work():
        o, s = ave.chunk_linear_attn(t["q"], t["k"], t["v"], t["g"], initial_state=t["h0"],
                                     output_final_state=True)
        r = ave.chunk_linear_attn_bwd(t["q"], t["k"], t["v"], t["g"], t["do"], t["dht"],
                                      initial_state=t["h0"])
        d = ave.fused_recurrent_linear_attn(t["q"][:, :1], t["k"][:, :1], t["v"][:, :1],
                                            t["g"][:, :1], initial_state=s,
                                            output_final_state=True, inplace_final_state=False)
        return (o, s) + r + d
    work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
    for seed in (1, 2, 3):
        new = make(1, 400, 1, 2, 128, 64, seed=seed)
        for n in ("q", "k", "v", "g", "h0", "do", "dht"):
            t[n].copy_(new[n])
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(held, work()):
            assert torch.equal(x, y)


@pytest.mark.gpu
def test_on_another_stream(rocm_device):
    import avelang_amd as ave
    t = to(make(1, 300, 1, 2, 64, 64, seed=7), rocm_device)
    want = ave.chunk_linear_attn(t["q"], t["k"], t["v"], t["g"])[0]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = ave.chunk_linear_attn(t["q"], t["k"], t["v"], t["g"])[0]
    st.synchronize()
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [False, True])
def test_final_state_over_the_initial_one(rocm_device, packed):
    """Sequences of several segments with final_state = initial_state: nothing reads it after it
    is written."""
    import avelang_amd as ave
    lens = [700, 0, 30, 570]
    shape = (1, 1300, 1, 2, 64, 64) if packed else (2, 700, 2, 4, 128, 128)
    t = to(make(*shape, seed=11, lens=lens if packed else None), rocm_device)
    cu = torch.tensor(cu_of(lens), device=rocm_device) if packed else None
    args = (t["q"], t["k"], t["v"], t["g"])
    o, s = ave.chunk_linear_attn(*args, initial_state=t["h0"], output_final_state=True, cu_seqlens=cu)
    for _ in range(5):
        state = t["h0"].clone()
        o2, s2 = ave.chunk_linear_attn(*args, initial_state=state, output_final_state=True,
                                       cu_seqlens=cu, final_state=state)
        assert s2 is state and torch.equal(s2, s) and torch.equal(o2, o)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 100, 1, 2, 64, 128), (2, 300, 1, 1, 128, 64), (1, 70, 2, 2, 128, 128)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_not_finite_stays_behind(rocm_device, shape, bad):
    """What is not finite in a token's q, k, v or g leaves every earlier token's output alone, and
    a token's own q all others'."""
    import avelang_amd as ave
    t = to(make(*shape, seed=12), rocm_device)
    want = ave.chunk_linear_attn(t["q"], t["k"], t["v"], t["g"], initial_state=t["h0"])[0]
    T = shape[1]
    for n in ("q", "k", "v", "g"):
        if n == "g" and bad < 0:
            continue   # a reset
        for at in (0, 13, 31, 33, T - 1):
            x = t[n].clone()
            x[0, at] = bad
            got = ave.chunk_linear_attn(*(x if m == n else t[m] for m in ("q", "k", "v", "g")),
                                        initial_state=t["h0"])[0]
            assert torch.equal(got[0, :at], want[0, :at]), (n, at)
            assert torch.equal(got[1:], want[1:])
            assert not got[0, at].isfinite().all()
            if n == "q":
                assert torch.equal(got[0, at + 1:], want[0, at + 1:])


@pytest.mark.gpu
def test_odd_addresses(rocm_device):
    """States, slices and gradients at addresses off 16 bytes are copied, in-place ones refused."""
    import avelang_amd as ave
    t = to(make(1, 70, 1, 2, 64, 64, seed=13), rocm_device)
    args = (t["q"], t["k"], t["v"], t["g"])

    def odd(x):
        y = torch.empty(x.numel() + 1, dtype=x.dtype, device=rocm_device)[1:].view(x.shape)
        return y.copy_(x)
    kw = dict(output_final_state=True)
    for op, more in ((ave.chunk_linear_attn, {}), (ave.fused_recurrent_linear_attn, dict(inplace_final_state=False))):
        want = op(*args, initial_state=t["h0"], **kw, **more)
        got = op(*map(odd, args), initial_state=odd(t["h0"]), **kw, **more)
        assert all(torch.equal(x, y) for x, y in zip(want, got))
    want = ave.chunk_linear_attn_bwd(*args, t["do"], t["dht"], initial_state=t["h0"])
    got = ave.chunk_linear_attn_bwd(*map(odd, args), odd(t["do"]), odd(t["dht"]), initial_state=odd(t["h0"]))
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    with pytest.raises(ValueError, match="aligned"):
        ave.fused_recurrent_linear_attn(*args, initial_state=odd(t["h0"]), output_final_state=True)
    with pytest.raises(ValueError, match="aligned"):
        ave.chunk_linear_attn(*args, initial_state=t["h0"], final_state=odd(t["h0"]), output_final_state=True)
    with pytest.raises(ValueError, match="aligned"):
        ave.chunk_linear_attn(*args, out=odd(t["v"]))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 130, 2, 4, 128, 128), (2, 256, 1, 1, 64, 64), (3, 500, 16, 32, 128, 64),
                                   (1, 640, 16, 32, 64, 128), (1, 650, 16, 32, 128, 128),
                                   (1, 384, 2, 4, 128, 128), (1, 385, 2, 4, 128, 128)])
def test_short_prompts(rocm_device, shape):
    """Prompts of a few chunks, each chunk's workgroup by itself, and just beyond them: o, the
    final state, also over the initial one, and the gradients' states."""
    import avelang_amd as ave
    d = make(*shape, seed=21)
    o, ht = linear_ref.linear_attn(d["q"], d["k"], d["v"], d["g"], h0=d["h0"])
    t = to(d, rocm_device)
    args = (t["q"], t["k"], t["v"], t["g"])
    got, s = ave.chunk_linear_attn(*args, initial_state=t["h0"], output_final_state=True)
    assert far(got, o) <= 2 ** -8 and far(s, ht) <= 2 ** -20
    state = t["h0"].clone()
    got2, _ = ave.chunk_linear_attn(*args, initial_state=state, output_final_state=True, final_state=state)
    assert torch.equal(got, got2) and torch.equal(state, s)
    _, _, states = ave.chunk_linear_attn_fwd_save(*args, initial_state=t["h0"])
    kw = dict(initial_state=t["h0"])
    a = ave.chunk_linear_attn_bwd(*args, t["do"], t["dht"], states=states, **kw)
    b = ave.chunk_linear_attn_bwd(*args, t["do"], t["dht"], **kw)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[100, 0, 200], [384], [385, 1], [64, 128, 1, 65, 130]])
def test_short_packed_prompts(rocm_device, lens):
    """Packed prompts of few tokens in all: each as by itself, the state also over the initial
    one, and the gradients' states formed again."""
    import avelang_amd as ave
    cu = cu_of(lens)
    d = make(1, cu[-1], 2, 4, 128, 128, seed=31, lens=lens)
    t = to(d, rocm_device)
    o, ht = linear_ref.linear_attn(d["q"], d["k"], d["v"], d["g"], h0=d["h0"], cu=cu)
    args, c = (t["q"], t["k"], t["v"], t["g"]), torch.tensor(cu, device=rocm_device)
    got, s = ave.chunk_linear_attn(*args, initial_state=t["h0"], output_final_state=True, cu_seqlens=c)
    assert far(got, o) <= 2 ** -8 and far(s, ht) <= 2 ** -20
    state = t["h0"].clone()
    got2, _ = ave.chunk_linear_attn(*args, initial_state=state, output_final_state=True, cu_seqlens=c,
                                    final_state=state)
    assert torch.equal(got, got2) and torch.equal(state, s)
    kw = dict(initial_state=t["h0"], cu_seqlens=c)
    _, _, states = ave.chunk_linear_attn_fwd_save(*args, **kw)
    a = ave.chunk_linear_attn_bwd(*args, t["do"], t["dht"], states=states, **kw)
    b = ave.chunk_linear_attn_bwd(*args, t["do"], t["dht"], **kw)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
