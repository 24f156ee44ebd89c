"""What linear attention's and layer norm's autograd forms keep for the backward: saved tensors
come back from hooks (offloading to the host, say) in another layout than they went in with.

Tolerances: none, the same bits with a hook as without.
"""
import ctypes

import pytest
import torch

from avelang_amd import linear_attention as L
from avelang_amd import norm as N

BF = torch.bfloat16


def _slices(B, T, Hqk, Hv, K, V, device="cpu", seed=0):
    """q, k, v as column slices of one tensor, which are read in place, and g."""
    gen = torch.Generator().manual_seed(seed)
    widths = [Hqk * K, Hqk * K, Hv * V]
    y = torch.randn((B, T, sum(widths) + 16), generator=gen).to(BF).to(device)
    q, k, v = (x.reshape(B, T, h, d) for x, h, d in zip(y[..., :-16].split(widths, -1),
                                                       (Hqk, Hqk, Hv), (K, K, V)))
    return q, k, v, -torch.rand((B, T, Hv), generator=gen).to(device)


def _odd(x):
    """x at an address off 16 bytes (contiguous otherwise)."""
    if x.dtype is not BF:
        return x
    return torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)[1:].view(x.shape).copy_(x)


def _strided(x):
    """x's values with its last two axes stored the other way round."""
    return x if x.dim() < 2 else x.transpose(-1, -2).contiguous().transpose(-1, -2)


HOOKS = {"contiguous": lambda x: x.contiguous(), "odd": _odd, "strided": _strided}


@pytest.mark.parametrize("hook", sorted(HOOKS) + ["cpu"])
def test_strides_of_what_comes_back(monkeypatch, hook):
    """The backward is given the strides of the tensors it reads, not of those that were saved."""
    seen = {}

    def inputs(q, k, v, g, cu, name, out=None):   # the checks of devices left out
        q, k, v, rows = L._in_place(q, k, v, out)
        if rows is None:
            rows = tuple(x.shape[2] * x.shape[3] for x in (q, k, v))
            q, k, v = (x if x.data_ptr() % 16 == 0 else x.clone() for x in (q, k, v))
        dims = (*q.shape[:3], v.shape[2], q.shape[3], v.shape[3], q.shape[0])
        return q, k, v, g.contiguous(), cu, rows, dims

    def bwd(inputs, do, dht, scale, h0, states, *rest):
        seen["inputs"] = inputs
        q, k, v, g = inputs[:4]
        return torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(g), None
    monkeypatch.setattr(L, "_inputs", inputs)
    monkeypatch.setattr(L, "_chunk_fwd", lambda inputs, *a, **kw: (inputs[2].contiguous(), None, None))
    monkeypatch.setattr(L, "_chunk_bwd", bwd)
    args = [x.requires_grad_() for x in _slices(2, 5, 2, 4, 64, 128)]
    around = (torch.autograd.graph.save_on_cpu() if hook == "cpu" else
              torch.autograd.graph.saved_tensors_hooks(HOOKS[hook], lambda x: x))
    with around:
        o, _ = L.chunk_linear_attn(*args)
    o.sum().backward()
    q, k, v, g, _, rows, _ = seen["inputs"]
    for x, want, row in zip((q, k, v), args, rows):
        assert torch.equal(x, want)
        assert x.data_ptr() % 16 == 0
        assert x.stride() == (5 * row, row, x.shape[3], 1)
    assert g.is_contiguous()


@pytest.mark.gpu
@pytest.mark.parametrize("hook", sorted(HOOKS) + ["cpu"])
@pytest.mark.parametrize("save", [True, False])
@pytest.mark.parametrize("packed", [False, True])
def test_gradients_through_hooks(rocm_device, hook, save, packed):
    import avelang_amd as ave
    B, T = (1, 150) if packed else (2, 75)
    cu = torch.tensor([0, 70, 150], dtype=torch.int32, device=rocm_device) if packed else None
    gen = torch.Generator().manual_seed(3)
    h0 = torch.randn((2, 4, 64, 128), generator=gen).to(rocm_device).requires_grad_()
    do = torch.randn((B, T, 4, 128), generator=gen).to(BF).to(rocm_device)

    def grads(around):
        leaves = [x.requires_grad_() for x in _slices(B, T, 2, 4, 64, 128, rocm_device)] + [h0]
        with around:
            o, ht = ave.chunk_linear_attn(*leaves[:4], initial_state=h0, output_final_state=True,
                                          cu_seqlens=cu, save_for_backward=save)
        return torch.autograd.grad([o, ht], leaves, [do, torch.ones_like(ht)])
    want = grads(torch.autograd.graph.saved_tensors_hooks(lambda x: x, lambda x: x))
    got = grads(torch.autograd.graph.save_on_cpu() if hook == "cpu" else
                torch.autograd.graph.saved_tensors_hooks(HOOKS[hook], lambda x: x))
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("hook", ["contiguous", "strided"])
def test_layout_of_what_comes_back_to_the_norm(monkeypatch, hook):
    """The kernels are given rows that follow one another, whatever a hook returns."""
    def args(x, weight, bias, name):   # the checks of devices left out
        return x.contiguous(), weight.contiguous(), bias.contiguous(), 15, 3, 8, 1, 0

    class Lib:
        def gdn_layer_norm_fwd(self, *a):
            return 0

        def gdn_layer_norm_bwd_workspace_bytes(self, *a):
            return 8

        def gdn_layer_norm_bwd(self, x, w, dy, stats, *a):
            self.seen = [torch.frombuffer((ctypes.c_float * n).from_address(p), dtype=torch.float32).clone()
                         for p, n in ((x, 120), (w, 24), (dy, 120), (stats, 30))]
            return 0
    lib = Lib()
    monkeypatch.setattr(N, "_args", args)
    monkeypatch.setattr(N, "_stream", lambda dev: 0)
    monkeypatch.setattr(N._native, "lib", lambda: lib)
    gen = torch.Generator().manual_seed(1)
    x, w, b, dy = (torch.randn(s, generator=gen) for s in ((5, 3, 8), (3, 8), (3, 8), (5, 3, 8)))
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (kept.append(t), HOOKS[hook](t))[1], lambda t: t):
        y = N.layer_norm(x.requires_grad_(), w.requires_grad_(), b.requires_grad_())
    y.backward(_strided(dy))
    assert len(kept) == 4
    for got, want in zip(lib.seen, (x, w, dy, kept[3])):
        assert torch.equal(got.nan_to_num(), want.detach().reshape(-1).nan_to_num())


@pytest.mark.gpu
@pytest.mark.parametrize("hook", sorted(HOOKS) + ["cpu"])
@pytest.mark.parametrize("heads", [0, 3])
def test_norm_gradients_through_hooks(rocm_device, hook, heads):
    import avelang_amd as ave
    par = (heads, 40) if heads else (40,)
    gen = torch.Generator().manual_seed(2)
    x, w, b, dy = (torch.randn(s, generator=gen).to(rocm_device) for s in ((50,) + par, par, par, (50,) + par))

    def grads(around):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        with around:
            y = ave.layer_norm(*leaves)
        return torch.autograd.grad(y, leaves, dy)
    want = grads(torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t))
    got = grads(torch.autograd.graph.save_on_cpu() if hook == "cpu" else
                torch.autograd.graph.saved_tensors_hooks(HOOKS[hook], lambda t: t))
    assert all(torch.equal(g, r) for g, r in zip(got, want))


@pytest.mark.parametrize("save", [True, False])
@pytest.mark.parametrize("wanted", [True, False])
def test_what_the_backward_asks_for(monkeypatch, save, wanted):
    """A carried state without a gradient gets none, and is held only to form the states again."""
    seen = {}

    def fwd(inputs, scale, initial_state, output_final_state, name, save=False):
        return inputs[2].clone(), None, torch.zeros(8, dtype=torch.uint8) if save else None

    def bwd(inputs, do, dht, scale, initial_state, want_dh0, states, workspace, name):
        seen.update(h0=initial_state, want=want_dh0, states=states)
        return *(torch.zeros_like(x) for x in inputs[:4]), state * 0 if want_dh0 else None
    monkeypatch.setattr(L, "_inputs", lambda q, k, v, g, cu, name, out=None: (q, k, v, g, cu, None, None))
    monkeypatch.setattr(L, "_chunk_fwd", fwd)
    monkeypatch.setattr(L, "_chunk_bwd", bwd)
    args = [x.contiguous().requires_grad_() for x in _slices(1, 5, 2, 4, 64, 64)]
    state = torch.zeros(1, 4, 64, 64, requires_grad=wanted)
    o, _ = L.chunk_linear_attn(*args, initial_state=state, save_for_backward=save)
    if save:
        with torch.no_grad():
            state.fill_(1.0)   # the next step's state
    o.sum().backward()
    assert seen["want"] == wanted and (seen["h0"] is None) == save and (seen["states"] is None) != save
    assert (state.grad is not None) == wanted


@pytest.mark.gpu
def test_state_carried_in_place(rocm_device):
    import avelang_amd as ave
    gen = torch.Generator().manual_seed(6)
    h0 = torch.randn((1, 4, 64, 128), generator=gen).to(rocm_device)
    do = torch.randn((1, 300, 4, 128), generator=gen).to(BF).to(rocm_device)

    def grads(overwrite, wanted):
        leaves = [x.requires_grad_() for x in _slices(1, 300, 2, 4, 64, 128, rocm_device)]
        state = h0.clone().requires_grad_(wanted)
        o, ht = ave.chunk_linear_attn(*leaves, initial_state=state, output_final_state=True)
        if overwrite:
            with torch.no_grad():
                state.copy_(ht)
        return torch.autograd.grad(o, leaves + [state] * wanted, do)
    want = grads(False, False)
    assert all(torch.equal(x, y) for x, y in zip(grads(True, False), want))
    for x, y in zip(grads(True, True), grads(False, True)):
        assert torch.equal(x, y)
