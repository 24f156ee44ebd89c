"""Linear attention with a decay for each head, for MI355X (gfx950).

One state [K, V] per v-head, v-head h reading qk-head h // (Hv // Hqk):

    S_t = e^{g_t} S_{t-1} + k_t v_t^T          o_t = scale * S_t^T q_t

in the chunked form for prompts and training (``chunk_linear_attn``, with its
gradients) and token by token for decode (``fused_recurrent_linear_attn``).
Layouts, argument names and checks are those of the gated delta rule
(``gated_delta_rule.py``), whose recurrence without its delta term this is:

    q, k  [B, T, Hqk, K]  bf16        v, o  [B, T, Hv, V]  bf16
    g     [B, T, Hv] or [Hv], floating point: log-decays per token, or one
          per head (fixed slopes); -inf resets the state
    state [N, Hv, K, V]   fp32        K, V in {64, 128}

q, k and v may be column slices of a wider tensor (a layer's split): they are
read in place.  The kernels are the hand-written HIP code of
``csrc/gdn_linear*.hip`` behind ``include/gdn_linear.h``; there is no fallback
path.  The reference repository has no counterpart; the wrappers follow its
kernel-library convention (python/avelang_kernels/amdgpu_gemm.py:458-494).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _native
from .gated_delta_rule import (_HEAD_SIZES, _check_distinct_slots, _cu_on_device, _in_place, _out,
                               _ptr, _stream_ptr)
from .layer_ops import _DTYPES

__all__ = [
    "chunk_linear_attn",
    "chunk_linear_attn_fwd_save",
    "chunk_linear_attn_bwd",
    "fused_recurrent_linear_attn",
    "linear_attn_workspace_bytes",
]


def _inputs(q, k, v, g, cu_seqlens, name, out=None):
    """Checked q, k, v (as the kernels take them), g, cu_seqlens on the device,
    the token strides and the sizes (B, T, Hqk, Hv, K, V, N)."""
    bf16 = torch.bfloat16
    _native.no_tangents(name, q, k, v, g)
    for nm, t in (("q", q), ("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor):
            raise ValueError(f"{name}: {nm} must be a torch.Tensor")
        if t.dtype is not bf16:
            raise ValueError(f"{name}: {nm} must have dtype torch.bfloat16, got {t.dtype}.")
        if t.dim() != 4:
            raise ValueError(f"{name}: {nm} must be 4-D [B, T, H, D], got {tuple(t.shape)}.")
    B, T, Hqk, K = q.shape
    if k.shape != q.shape:
        raise ValueError(f"{name}: k must have shape {tuple(q.shape)}, got {tuple(k.shape)}.")
    Bv, Tv, Hv, V = v.shape
    if Bv != B or Tv != T:
        raise ValueError(f"{name}: v must have shape [B, T, Hv, V] with B, T = {B}, {T}.")
    if Hqk == 0 or Hv == 0 or Hv % Hqk != 0:
        raise ValueError(f"{name}: v-heads ({Hv}) must be a multiple of qk-heads ({Hqk}).")
    if K not in _HEAD_SIZES or V not in _HEAD_SIZES:
        raise ValueError(f"{name}: head sizes K={K}, V={V} unsupported (each in {_HEAD_SIZES}).")
    if not isinstance(g, torch.Tensor) or not g.is_floating_point():
        raise ValueError(f"{name}: g must be a floating point torch.Tensor")
    gs = g.shape
    if gs != (B, T, Hv) and gs != (Hv,):
        raise ValueError(f"{name}: g must have shape {(B, T, Hv)} or {(Hv,)}, got {tuple(gs)}.")
    dev = q.device
    if dev.type != "cuda":
        raise ValueError(f"{name}: tensors must be on a ROCm (cuda) device, got {dev}.")
    if k.device != dev or v.device != dev or g.device != dev:
        raise ValueError(f"{name}: q, k, v and g must all be on {dev}.")
    N, cu = B, None
    if cu_seqlens is not None:
        cu, N = _cu(cu_seqlens, B, T, dev, name)
    if g.dtype not in _DTYPES:
        g = g.float()
    q, k, v, rows = _in_place(q, k, v, out)
    if rows is None:
        rows = (Hqk * K, Hqk * K, Hv * V)
        if (q.data_ptr() | k.data_ptr() | v.data_ptr()) % 16:
            q, k, v = (t if t.data_ptr() % 16 == 0 else t.clone() for t in (q, k, v))
    return q, k, v, g.contiguous(), cu, rows, (B, T, Hqk, Hv, K, V, N)


def _cu(cu_seqlens, B, T, dev, name):
    if B != 1:
        raise ValueError(f"{name}: cu_seqlens requires batch size 1, got {B}.")
    if not isinstance(cu_seqlens, torch.Tensor) or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2:
        raise ValueError(f"{name}: cu_seqlens must be 1-D with at least 2 entries.")
    if cu_seqlens.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name}: cu_seqlens must be int32 or int64, got {cu_seqlens.dtype}.")
    N = cu_seqlens.numel() - 1
    if cu_seqlens.device.type == "cpu":
        c32 = cu_seqlens.to(torch.int32).contiguous()
        lib = _native.lib()
        if lib.gdn_cu_seqlens_check(c32.data_ptr(), N, T) != 0:
            raise ValueError(f"{name}: {lib.gdn_last_error().decode()} (T={T}).")
        return _cu_on_device(c32, dev), N
    if cu_seqlens.device != dev:
        raise ValueError(f"{name}: cu_seqlens must be on {dev} or the CPU.")
    return cu_seqlens.to(dtype=torch.int32).contiguous(), N


def _state(t, shape, dev, what, name):
    _native.no_tangents(name, t)
    if (not isinstance(t, torch.Tensor) or t.shape != shape or t.dtype is not torch.float32
            or t.device != dev):
        raise ValueError(f"{name}: {what} must be torch.float32 of shape {shape} on {dev}.")
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def linear_attn_workspace_bytes(B: int, T: int, Hqk: int, Hv: int, K: int, V: int, N: int,
                                has_cu_seqlens: bool, backward: bool = False) -> int:
    """Device scratch bytes ``chunk_linear_attn`` (or its backward) needs for these sizes, or
    for others of the same heads with B, T and N no larger."""
    lib = _native.lib()
    f = (lib.gdn_linear_chunk_bwd_workspace_bytes if backward
         else lib.gdn_linear_chunk_workspace_bytes)
    return int(f(B, T, Hqk, Hv, K, V, N, int(has_cu_seqlens)))


def _chunk_fwd(inputs, scale, initial_state, output_final_state, name, workspace=None, out=None,
               final_state=None, save=False, want_o=True):
    """gdn_linear_chunk_fwd on ``_inputs``' result: (o, final state, saved states)."""
    q, k, v, g, cu, rows, dims = inputs
    B, T, Hqk, Hv, K, V, N = dims
    dev = q.device
    lib = _native.lib()
    o = _out(v, out, name) if want_o else None
    h0 = None
    if initial_state is not None:
        h0 = _state(initial_state, (N, Hv, K, V), dev, "initial_state", name)
    ht = None
    if output_final_state:
        if final_state is None:
            ht = torch.empty((N, Hv, K, V), dtype=torch.float32, device=dev)
        else:
            ht = final_state
            if _state(ht, (N, Hv, K, V), dev, "final_state", name) is not ht:
                raise ValueError(f"{name}: final_state must be contiguous and 16-byte aligned.")
    states = None
    if save:
        states = torch.empty(max(1, lib.gdn_linear_states_bytes(B, T, Hv, K, V, N, cu is not None)),
                             dtype=torch.uint8, device=dev)
    if workspace is None:
        nbytes = lib.gdn_linear_chunk_workspace_bytes(*dims, cu is not None)
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    elif workspace.device != dev:   # (its size is checked by the entry point)
        raise ValueError(f"{name}: workspace must be on {dev}.")
    _native.check(lib.gdn_linear_chunk_fwd(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), *rows, g.data_ptr(), _DTYPES[g.dtype],
        g.dim() == 1, _ptr(h0), _ptr(ht), _ptr(o), _ptr(cu), *dims,
        K ** -0.5 if scale is None else float(scale), _ptr(states), _ptr(workspace),
        0 if workspace is None else workspace.numel() * workspace.element_size(),
        _stream_ptr(dev)), name)
    return o, ht, states


def chunk_linear_attn_fwd_save(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    g: torch.Tensor,
    scale: Optional[float] = None,
    initial_state: Optional[torch.Tensor] = None,
    output_final_state: bool = False,
    cu_seqlens: Optional[torch.Tensor] = None,
):
    """Training forward: ``(o, final_state, states)``, ``states`` (the state at
    every chunk's start in 16 bits, 2 K V bytes per 64 tokens and v-head) being
    what ``chunk_linear_attn_bwd`` takes for these same inputs."""
    name = "chunk_linear_attn_fwd_save"
    return _chunk_fwd(_inputs(q, k, v, g, cu_seqlens, name), scale, initial_state,
                      output_final_state, name, save=True)


def chunk_linear_attn_bwd(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    g: torch.Tensor,
    do: torch.Tensor,
    dht: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    initial_state: Optional[torch.Tensor] = None,
    cu_seqlens: Optional[torch.Tensor] = None,
    *,
    states: Optional[torch.Tensor] = None,
    workspace: Optional[torch.Tensor] = None,
):
    """Gradients of ``chunk_linear_attn``: ``(dq, dk, dv, dg, dh0)``, dq, dk, dv
    in bf16, dg with g's shape and type (an fp32 dg too holds the saved states'
    rounding, up to 2^-9 of each of its terms), dh0 fp32 (None without
    ``initial_state``).  ``do`` is dL/do (bf16, v's shape), ``dht`` (nullable)
    dL/d(final state).  Without ``states`` (``chunk_linear_attn_fwd_save``) the
    forward's states are formed again.  Deterministic.
    """
    name = "chunk_linear_attn_bwd"
    return _chunk_bwd(_inputs(q, k, v, g, cu_seqlens, name), do, dht, scale, initial_state,
                      initial_state is not None, states, workspace, name)


def _chunk_bwd(inputs, do, dht, scale, initial_state, want_dh0, states, workspace, name):
    q, k, v, g, cu, rows, dims = inputs
    B, T, Hqk, Hv, K, V, N = dims
    dev = q.device
    _native.no_tangents(name, do)
    if (not isinstance(do, torch.Tensor) or do.shape != v.shape or do.dtype != torch.bfloat16
            or do.device != dev):
        raise ValueError(f"{name}: do must be a bf16 tensor of shape {tuple(v.shape)} on {dev}.")
    do = do.contiguous()
    do = do if do.data_ptr() % 16 == 0 else do.clone()
    if dht is not None:
        dht = _state(dht, (N, Hv, K, V), dev, "dht", name)
    if initial_state is not None:
        _state(initial_state, (N, Hv, K, V), dev, "initial_state", name)
    lib = _native.lib()
    if states is None:
        _, _, states = _chunk_fwd(inputs, scale, initial_state, False, name, save=True,
                                  want_o=False)
    else:
        need = lib.gdn_linear_states_bytes(B, T, Hv, K, V, N, cu is not None)
        if states.device != dev or states.numel() * states.element_size() < need:
            raise ValueError(f"{name}: states must hold {need} bytes on {dev}.")
        states = states.contiguous()
    bf = dict(dtype=torch.bfloat16, device=dev)
    dq, dk = torch.empty((B, T, Hqk, K), **bf), torch.empty((B, T, Hqk, K), **bf)
    dv = torch.empty((B, T, Hv, V), **bf)
    dg = torch.empty_like(g)
    dh0 = None
    if want_dh0:
        dh0 = torch.empty((N, Hv, K, V), dtype=torch.float32, device=dev)
    if workspace is None:
        nbytes = lib.gdn_linear_chunk_bwd_workspace_bytes(*dims, cu is not None)
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    elif workspace.device != dev:
        raise ValueError(f"{name}: workspace must be on {dev}.")
    _native.check(lib.gdn_linear_chunk_bwd(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), *rows, g.data_ptr(), _DTYPES[g.dtype],
        g.dim() == 1, do.data_ptr(), _ptr(dht), states.data_ptr(), dq.data_ptr(), dk.data_ptr(),
        dv.data_ptr(), dg.data_ptr(), _ptr(dh0), _ptr(cu), *dims,
        K ** -0.5 if scale is None else float(scale), _ptr(workspace),
        0 if workspace is None else workspace.numel() * workspace.element_size(),
        _stream_ptr(dev)), name)
    return dq, dk, dv, dg, dh0


class _ChunkLinearAttn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, scale, initial_state, output_final_state, cu_seqlens, save):
        name = "chunk_linear_attn"
        inputs = _inputs(q, k, v, g, cu_seqlens, name)
        o, ht, states = _chunk_fwd(inputs, scale, initial_state, output_final_state, name, save=save)
        # (of a state that the backward has no need to form again only the shape counts)
        ctx.save_for_backward(*inputs[:5], None if save else initial_state, states)
        ctx.rest = scale, g.dtype
        ctx.set_materialize_grads(False)
        return (o, ht) if output_final_state else o

    @staticmethod
    @once_differentiable
    def backward(ctx, do, dht=None):
        q, k, v, g, cu, h0, states = ctx.saved_tensors
        scale, g_type = ctx.rest
        if do is None:
            do = torch.zeros(v.shape, dtype=v.dtype, device=v.device)
        # (token strides and alignment as they are now: a hook on saved tensors, one
        # that offloads them say, returns others of another layout)
        name = "chunk_linear_attn"
        dq, dk, dv, dg, dh0 = _chunk_bwd(_inputs(q, k, v, g, cu, name), do, dht, scale, h0,
                                         ctx.needs_input_grad[5], states, None, name)
        return dq, dk, dv, dg if dg.dtype is g_type else dg.to(g_type), None, dh0, None, None, None


def chunk_linear_attn(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    g: torch.Tensor,
    scale: Optional[float] = None,
    initial_state: Optional[torch.Tensor] = None,
    output_final_state: bool = False,
    cu_seqlens: Optional[torch.Tensor] = None,
    *,
    workspace: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    final_state: Optional[torch.Tensor] = None,
    save_for_backward: bool = True,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Chunked linear attention with a decay per head: ``(o, final_state)``,
    ``final_state`` None unless ``output_final_state``.

    ``scale`` defaults to ``K ** -0.5``.  ``cu_seqlens`` (int32 / int64 [N + 1],
    B = 1) packs N sequences; on the CPU a violation of its contract raises,
    on the device it empties every sequence.  ``workspace`` (uint8, of
    ``linear_attn_workspace_bytes(...)`` for this problem or any larger one),
    ``out`` and ``final_state`` (which may be ``initial_state`` itself) avoid
    allocation.  Infinities and NaN in a token's inputs reach its own and later
    outputs only (padding behind a batch's rows may hold anything); in the
    gradients they may reach others.

    Differentiable in q, k, v, g and initial_state (``chunk_linear_attn_bwd``).
    The forward then keeps the state at every chunk's start for the backward
    (134 MB at T = 8192 with 32 v-heads, K = V = 128); with
    ``save_for_backward=False`` it keeps the inputs alone and the backward
    forms the states again.
    """
    if torch.is_grad_enabled() and any(
            isinstance(t, torch.Tensor) and t.requires_grad for t in (q, k, v, g, initial_state)):
        if out is not None or workspace is not None or final_state is not None:
            raise ValueError("chunk_linear_attn: out / workspace / final_state buffers are not "
                             "supported when gradients are required.")
        res = _ChunkLinearAttn.apply(q, k, v, g, scale, initial_state, bool(output_final_state),
                                     cu_seqlens, bool(save_for_backward))
        return res if output_final_state else (res, None)
    name = "chunk_linear_attn"
    o, ht, _ = _chunk_fwd(_inputs(q, k, v, g, cu_seqlens, name, out), scale, initial_state,
                          output_final_state, name, workspace, out, final_state)
    return o, ht


def fused_recurrent_linear_attn(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    g: torch.Tensor,
    scale: Optional[float] = None,
    initial_state: Optional[torch.Tensor] = None,
    output_final_state: bool = False,
    cu_seqlens: Optional[torch.Tensor] = None,
    inplace_final_state: bool = True,
    ssm_state_indices: Optional[torch.Tensor] = None,
    *,
    out: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Token by token (decode): every state is read once, advanced through its
    sequence's tokens and written once.  Not differentiable.  ``cu_seqlens`` as in
    ``chunk_linear_attn``.

    With ``output_final_state`` and ``inplace_final_state`` (and an
    ``initial_state``) the final state overwrites ``initial_state`` and that
    tensor is returned; otherwise a new tensor is returned.  With
    ``ssm_state_indices`` (int32 [N]) ``initial_state`` is a pool [num_slots,
    Hv, K, V] and sequence n uses slot ``ssm_state_indices[n]``, updated in
    place with ``output_final_state``; a slot outside the pool marks a padding
    sequence (state untouched, output rows unwritten).  Sequences must use
    distinct slots: a repeated one raises where the indices are on the CPU;
    on the device its sequences leave it untouched and get NaN output rows.
    """
    name = "fused_recurrent_linear_attn"
    q, k, v, g, cu, rows, dims = _inputs(q, k, v, g, cu_seqlens, name, out)
    N, state = dims[6], (dims[3], dims[4], dims[5])
    dev = q.device
    o = _out(v, out, name)
    h0, ht, idx, slots = initial_state, None, None, N
    _native.no_tangents(name, h0)
    if ssm_state_indices is not None:
        idx = ssm_state_indices
        if not isinstance(h0, torch.Tensor) or h0.dim() != 4:
            raise ValueError(f"{name}: ssm_state_indices requires initial_state as a state pool "
                             "[num_slots, Hv, K, V].")
        if output_final_state and not inplace_final_state:
            raise ValueError(f"{name}: with ssm_state_indices the final state is written in place.")
        if (not isinstance(idx, torch.Tensor) or tuple(idx.shape) != (N,)
                or idx.dtype != torch.int32 or idx.device not in (dev, torch.device("cpu"))):
            raise ValueError(f"{name}: ssm_state_indices must be int32 of shape ({N},) on {dev} "
                             "or the CPU.")
        slots = h0.shape[0]
        _check_distinct_slots(idx, slots, name)
        idx = idx.to(dev).contiguous()
    if h0 is not None:
        h0 = _state(h0, (slots,) + state, dev, "initial_state", name)
        if output_final_state and inplace_final_state and h0 is not initial_state:
            raise ValueError(f"{name}: an in-place initial_state must be contiguous and "
                             "16-byte aligned.")
        if idx is not None and h0 is not initial_state:
            raise ValueError(f"{name}: the state pool must be contiguous and 16-byte aligned.")
    if output_final_state:
        ht = h0
        if h0 is None or not inplace_final_state:
            ht = torch.empty((N,) + state, dtype=torch.float32, device=dev)
    _native.check(_native.lib().gdn_linear_recurrent_fwd(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), *rows, g.data_ptr(), _DTYPES[g.dtype],
        g.dim() == 1, _ptr(h0), _ptr(ht), o.data_ptr(), _ptr(cu), _ptr(idx), *dims, slots,
        dims[4] ** -0.5 if scale is None else float(scale), _stream_ptr(dev)), name)
    return o, ht
