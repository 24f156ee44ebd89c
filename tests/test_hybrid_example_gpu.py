"""The example's hybrid block: norms, rotation, cache and attention together, as a program runs them, and the
gradients of the half that trains against the same layer written out in float64.

Tolerances: every bf16 tensor on the way is rounded once (2^-9 of it in the mean); the two ways to the same
tokens, and the layer in float64, differ by some ten such roundings, each carried on through products of unit
gain: 2^-9 sqrt(10) < 2^-7 in the norm, doubled for the operands' own.  An e4m3 cache rounds k and v by up to
2^-4 (2^-5.8 in the mean), an int8 one by 2^-8 of the row's largest (2^-7 in the mean).
"""
import importlib.util
import os

import pytest
import torch
import torch.nn.functional as F

import avelang_amd as ave
from oracle import attn_ref, linear_ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.gpu


def _example():
    spec = importlib.util.spec_from_file_location("hybrid_block", os.path.join(ROOT, "examples", "hybrid_block.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def _serve(m, block, x, dtype, steps):
    pages, state, parts = m.Pages(x.shape[0], 160, 16, block.heads[1], block.size, dtype), None, []
    at = 0
    for t in steps:
        codes, scale, h, state = block.serve(x[:, at:at + t], state, pages, decode=t == 1)
        parts.append(((codes.float() * scale[..., None]), h.float()))
        at += t
    return [torch.cat(p, 1) for p in zip(*parts)] + [state]


def _far(a, b):
    return ((a - b).norm() / b.norm()).item()


@pytest.mark.parametrize("size,rotated", [(64, 64), (128, 32)])
def test_pieces_and_tokens(rocm_device, size, rotated):
    torch.manual_seed(1)
    m = _example()
    block = m.HybridBlock(256, (2, 4), (4, 2), size, rotated)
    x = torch.randn(3, 100, 256, device=rocm_device).bfloat16()
    whole = _serve(m, block, x, torch.bfloat16, [50, 50])
    tokens = _serve(m, block, x, torch.bfloat16, [40, 3, 49] + [1] * 8)
    assert _far(tokens[1], whole[1]) <= 2 ** -6 and _far(tokens[2], whole[2]) <= 2 ** -6
    # the 8-bit output: half a step (2^-4 of a value at most, 2^-5.2 in the mean) of each
    assert _far(tokens[0], whole[0]) <= 2 ** -4
    for dtype, most in ((torch.float8_e4m3fn, 2 ** -4), (torch.int8, 2 ** -6)):
        assert _far(_serve(m, block, x, dtype, [50, 50])[1], whole[1]) <= most


def test_attention_layer_against_float64(rocm_device):
    torch.manual_seed(2)
    m = _example()
    block = m.HybridBlock(128, (1, 2), (4, 2), 64)
    y = torch.randn(2, 37, 128, device=rocm_device).bfloat16()
    pages = m.Pages(2, 64, 16, 2, 64, torch.bfloat16)
    with torch.no_grad():
        positions, slots = pages.grow(37)
        got = block.attention_layer(y, positions, slots, pages).double().cpu()
    q, k, v = (y.double().cpu() @ block.att_in.double().cpu().T).split(block.att_widths, -1)
    q, k, v = (t.unflatten(-1, (-1, 64)) for t in (q, k, v))
    q, k = (attn_ref.rotary(t, positions.cpu(), block.freq.cpu(), block.magnitude) for t in (q, k))
    o = torch.stack([attn_ref.attention(q[n], k[n].transpose(0, 1), v[n].transpose(0, 1), 64 ** -0.5)[0]
                     for n in range(2)])
    want = o.flatten(2) @ block.att_out.double().cpu().T
    assert _far(got, want) <= 2 ** -6


def test_training_half_gradients(rocm_device):
    torch.manual_seed(3)
    m = _example()
    block = m.HybridBlock(128, (1, 2), (4, 2), 64)
    x = torch.randn(2, 70, 128, device=rocm_device).bfloat16().requires_grad_()
    positions = torch.arange(70, device=rocm_device)
    names = ["lin_in", "decay", "lin_out"]
    leaves = [x, block.norms[0], block.norms[1]] + [getattr(block, n) for n in names]
    y, h = block.train_half(x, positions)
    dy, dh = torch.randn_like(y), torch.randn_like(h)
    got = torch.autograd.grad([y, h], leaves, [dy, dh])
    ref = [t.detach().double().cpu().requires_grad_() for t in leaves]
    xr, w0, w1, win, wdec, wout = ref
    z, _ = attn_ref.rms_norm(xr, w0, offset=1.0)
    q, k, v = ((z @ win.T).split(block.lin_widths, -1))
    q, k, v = (t.unflatten(-1, (-1, 64)) for t in (q, k, v))
    q, k = (attn_ref.rotary(t, positions.cpu()[None], block.freq.cpu(), block.magnitude) for t in (q, k))
    o, _ = linear_ref.linear_attn(q, k, v, F.logsigmoid(z @ wdec.T + 3.0))
    yr, hr = attn_ref.rms_norm(o.flatten(2) @ wout.T, w1, res=xr, offset=1.0, rounded=False)
    assert _far(y.detach().double().cpu(), yr.detach()) <= 2 ** -6 and _far(h.detach().double().cpu(), hr.detach()) <= 2 ** -6
    want = torch.autograd.grad([yr, hr], ref, [dy.double().cpu(), dh.double().cpu()])
    for name, a, b in zip(["x", "norm 0", "norm 1"] + names, got, want):
        assert _far(a.double().cpu(), b) <= 2 ** -5, name


def test_runs(rocm_device, capsys):
    _example().main()
    assert "step 2" in capsys.readouterr().out


def test_wrappers_refuse(rocm_device):
    """Refusals of the calls themselves, by tensors on the GPU."""
    dev = dict(device=rocm_device)
    x, r = torch.zeros(3, 64, **dev).bfloat16(), torch.zeros(3, 64, **dev)
    pos, f = torch.zeros(3, dtype=torch.int64, **dev), torch.ones(32, **dev)
    q = torch.zeros(3, 2, 64, **dev).bfloat16()
    c = ave.PagedKVCache.zeros(2, 16, 2, 64, torch.bfloat16)
    c8 = ave.PagedKVCache.zeros(2, 24, 2, 64, torch.int8)
    sl = torch.arange(3, **dev)
    q4, t, n = q[:, None], torch.zeros(3, 1, dtype=torch.int32, **dev), torch.ones(3, dtype=torch.int32, **dev)
    for call in (
            lambda: ave.rms_norm(x.int()), lambda: ave.rms_norm(x, r[0].bfloat16()[:32]), lambda: ave.rms_norm(x, r),
            lambda: ave.rms_norm(x, residual=r[:2]), lambda: ave.rms_norm(r, residual=x), lambda: ave.rms_norm(x.half(), residual=x),
            lambda: ave.rms_norm(x, r[0].cpu()), lambda: ave.rms_norm(x, out=r), lambda: ave.rms_norm(x, residual_out=x),
            lambda: ave.rms_norm(x, residual=x, out=x, residual_out=x),
            lambda: ave.rms_norm_quant(x, dtype=torch.uint8), lambda: ave.rms_norm_bwd(r, None, x, x),
            lambda: ave.rms_norm_bwd(x, None, x, r), lambda: ave.rms_norm_bwd(x, None, r),
            lambda: ave.rotary_embedding(q, None, pos[:2], f), lambda: ave.rotary_embedding(q, None, pos.float(), f),
            lambda: ave.rotary_embedding(q, None, pos, f.long()), lambda: ave.rotary_embedding(q, None, pos, torch.ones(33, **dev)),
            lambda: ave.rotary_embedding(q, q[:2], pos, f), lambda: ave.rotary_embedding(q, q.half(), pos, f),
            lambda: ave.rotary_embedding(q[..., :63], None, pos, f[:2]), lambda: ave.rotary_embedding(q[0], None, pos, f),
            lambda: ave.rotary_embedding(q[:1].expand(3, 2, 64), None, pos, f, inplace=True),
            lambda: ave.rotary_embedding(q.transpose(1, 2), None, pos, f[:1], inplace=True),
            lambda: ave.paged_cache_write(c, q, q, sl[:2]), lambda: ave.paged_cache_write(c, q, q.half(), sl),
            lambda: ave.paged_cache_write(c, q.half(), q.half(), sl), lambda: ave.paged_cache_write(c, q, q, sl.float()),
            lambda: ave.paged_cache_write(c, q, q, torch.tensor([1, 2, 1])), lambda: ave.paged_cache_write((c.k, c.v), q, q, sl),
            lambda: ave.paged_cache_read(c, sl, torch.float16), lambda: ave.paged_cache_read(c8, sl, torch.float32),
            lambda: ave.paged_attention(q, c, t, n), lambda: ave.paged_attention(q4.float(), c, t, n),
            lambda: ave.paged_attention(q4.half(), c, t, n), lambda: ave.paged_attention(q4, c8, t, n),
            lambda: ave.paged_attention(q4[:, :, :1], c, t, n), lambda: ave.paged_attention(q4, c, t.long(), n),
            lambda: ave.paged_attention(q4, c, t, n.long()), lambda: ave.paged_attention(q4, c, t[:2], n),
            lambda: ave.paged_attention(q4, c, t, n[:2]), lambda: ave.paged_attention(q4, c, t, n, window=-1),
            lambda: ave.paged_attention(q4, c, t, n, max_length=17), lambda: ave.paged_attention(q4, c, t, n, out=q4),
            lambda: ave.paged_attention(q4, c, t, n, out=torch.zeros(3, 1, 2, 64, **dev)),
            lambda: ave.paged_attention(q4, c, t, n, workspace=torch.empty(16, dtype=torch.uint8, **dev)),
            lambda: ave.paged_attention(q4, c, t, n, workspace=torch.empty(1 << 20, dtype=torch.uint8))):
        with pytest.raises(ValueError):
            call()


def test_wrappers_refuse_sizes(rocm_device):
    """Sizes past 32 bits, by expanded tensors without memory, are refused and not cut."""
    big, dev = 2 ** 32 + 3, dict(device=rocm_device)
    x, f = torch.zeros(1, **dev), torch.ones(1, **dev)
    pos, n = torch.zeros(1, dtype=torch.int64, **dev), torch.ones(1, dtype=torch.int32, **dev)
    c = ave.PagedKVCache.zeros(1, 16, 1, 64, torch.bfloat16)
    row = torch.zeros(1, 1, 64, **dev).bfloat16()
    for call in (
            lambda: ave.rms_norm(x.expand(big)), lambda: ave.rms_norm_quant(x.expand(1, big)),
            lambda: ave.rotary_embedding(x.expand(big, 1, 2), None, pos.expand(big), f),
            lambda: ave.rotary_embedding(x.expand(1, big, 2), None, pos, f),
            lambda: ave.paged_cache_write(c, row.expand(big, 1, 64), row.expand(big, 1, 64), pos.expand(big)),
            lambda: ave.paged_cache_read(c, pos.expand(big)),
            lambda: ave.paged_attention(row[None].expand(1, big, 1, 64), c, n[None], n),
            lambda: ave.paged_attention(row[None].expand(big, 1, 1, 64), c, n[None].expand(big, 1), n.expand(big)),
            lambda: ave.paged_attention(row[None], c, n[None].expand(1, big), n)):
        with pytest.raises(ValueError):
            call()
    n.fill_(16)
    q, t = torch.randn(1, 2, 1, 64, **dev).bfloat16(), torch.zeros(1, 1, dtype=torch.int32, **dev)
    c.v.normal_()
    assert torch.equal(ave.paged_attention(q, c, t, n, window=2 ** 32 + 1), ave.paged_attention(q, c, t, n))


def test_cache_tensors(rocm_device):
    """The cache's tensors are found where they are at a call, and cannot be exchanged for others."""
    c = ave.PagedKVCache.zeros(3, 16, 1, 64, torch.int8)
    with pytest.raises(AttributeError):
        c.k = c.v
    kv = torch.randn(2, 20, 1, 64, device=rocm_device).bfloat16()
    slots = torch.arange(20, device=rocm_device)
    ave.paged_cache_write(c, kv[0], kv[1], slots)
    before = ave.paged_cache_read(c, slots)
    old = c.k.data
    c.k.data = old.clone()
    old.zero_()
    assert all(torch.equal(a, b) for a, b in zip(ave.paged_cache_read(c, slots), before))


@pytest.mark.parametrize("code", [torch.bfloat16, torch.float8_e4m3fn, torch.int8])
def test_captured_decode_step(rocm_device, code):
    """Norm, rotation in place, cache write, attention and the 8-bit norm in one graph, replayed token by
    token beside the same calls run eagerly on a copy of the cache."""
    N, Hq, H, D, page, dev = 5, 8, 2, 128, 16, dict(device=rocm_device)
    gen = torch.Generator(rocm_device).manual_seed(3)
    rand = lambda *s: torch.randn(*s, generator=gen, **dev).bfloat16()  # noqa: E731
    x, res, w = rand(N, (Hq + 2 * H) * D), rand(N, (Hq + 2 * H) * D), rand((Hq + 2 * H) * D)
    f, size = ave.rotary_frequencies(D // 2, factor=4.0, original=2048, device=rocm_device)
    caches = [ave.PagedKVCache.zeros(64, page, H, D, code) for _ in "ab"]
    table = torch.randperm(64, generator=gen, **dev).int()[:N * 8].view(N, 8)
    lens = torch.tensor([0, 15, 16, 31, 100], dtype=torch.int32, **dev)
    first = int(lens.max())
    for c in caches:
        for t in (c.k, c.v):
            t.view(torch.uint8).fill_(0x30)
        for t in (c.k_scale, c.v_scale):
            if t is not None:
                t.fill_(0.01)

    def step(c, n):
        y, h = ave.rms_norm(x, w, residual=res, offset=1.0)
        q, k, v = (t.view(N, 1, -1, D) for t in y.split([Hq * D, H * D, H * D], -1))
        pos = n.long()[:, None]
        ave.rotary_embedding(q, k, pos, f, magnitude=size, inplace=True)
        slots = table.gather(1, pos // page).long() * page + pos % page
        ave.paged_cache_write(c, k, v, slots)
        o, lse = ave.paged_attention(q, c, table, n + 1, return_lse=True)
        return (h, o, lse) + ave.rms_norm_quant(o.flatten(2), dtype=torch.int8)

    spare = ave.PagedKVCache.zeros(64, page, H, D, code)
    step(spare, lens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(caches[0], lens)
    for i in range(4):
        x.normal_(generator=gen)
        res.normal_(generator=gen)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step(caches[1], lens)):
            assert torch.equal(a, b)
        assert torch.equal(caches[0].k.view(torch.uint8), caches[1].k.view(torch.uint8))
        assert torch.equal(caches[0].v.view(torch.uint8), caches[1].v.view(torch.uint8))
        lens += 1
    assert int(lens.max()) == first + 4


@pytest.mark.parametrize("rows,D,t", [(3, 256, torch.bfloat16), (700, 1000, torch.float32), (40, 9000, torch.bfloat16)])
def test_captured_gradients(rocm_device, rows, D, t):
    """The norm's and the rotation's gradients in one graph, replayed with new inputs."""
    dev = dict(device=rocm_device)
    x, r, dy, dh = (torch.randn(rows, D, **dev).to(t) for _ in range(4))
    w = torch.randn(D, **dev)
    q, dq = (torch.randn(rows, 2, 64, **dev).to(t) for _ in "qd")
    pos, f = torch.arange(rows, **dev), torch.ones(32, dtype=torch.float64, **dev)

    def work():
        y, h = ave.rms_norm(x, w, residual=r)
        return (y, h) + ave.rms_norm_bwd(h, w, dy, dh) + (ave.rotary_embedding(q, None, pos, f),)

    work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
    for _ in range(3):
        for a in (x, r, dy, dh, w, q):
            a.normal_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, work()):
            assert torch.equal(a, b)


def test_on_another_stream(rocm_device):
    """Inputs of the current stream, calls and gradients on another."""
    dev = dict(device=rocm_device)
    x, dy = (torch.randn(300, 512, **dev).bfloat16() for _ in "xy")
    w = torch.randn(512, **dev)
    q, dq = (torch.randn(300, 4, 64, **dev).bfloat16() for _ in "qd")
    pos, f = torch.arange(300, **dev), torch.ones(32, dtype=torch.float64, **dev)

    def work():
        a, b, c = (t.clone().requires_grad_() for t in (x, w, q))
        y = ave.rms_norm(a, b)
        z = ave.rotary_embedding(c, None, pos, f)
        c8 = ave.PagedKVCache.zeros(20, 16, 4, 64, torch.int8)
        ave.paged_cache_write(c8, z.detach(), dq, pos)
        return [y, z, *torch.autograd.grad([y, z], [a, b, c], [dy, dq]), *ave.paged_cache_read(c8, pos)]

    want = work()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = work()
    st.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_no_gradients_of_gradients(rocm_device):
    """Gradients with a graph of their own are right, and refuse to be differentiated again."""
    dev = dict(device=rocm_device)
    x, w, q = torch.randn(5, 64, **dev), torch.randn(64, **dev), torch.randn(5, 2, 32, **dev)
    pos, f = torch.arange(5, **dev), torch.ones(16, dtype=torch.float64, **dev)
    for call, leaves in ((lambda a, b: ave.rms_norm(a, b), (x, w)), (lambda a: ave.rotary_embedding(a, None, pos, f), (q,))):
        leaves = [t.clone().requires_grad_() for t in leaves]
        want = torch.autograd.grad(call(*leaves).square().sum(), leaves)
        got = torch.autograd.grad(call(*leaves).square().sum(), leaves, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        with pytest.raises(RuntimeError, match="once_differentiable"):
            got[0].sum().backward()
