"""Layer norm for MI355X (gfx950), forward and backward.

    y = (x - mean) / sqrt(var + eps) * weight + bias

over the last axis with the biased variance, in fp32 whatever x's type.  The
weight and bias have the last axis' shape, or the last two's: every head's
row by itself with parameters of its own (the norm of an attention's output).
HIP kernels of ``csrc/gdn_norm.hip`` behind ``include/gdn_linear.h``; there is
no fallback path.  The reference repository has no counterpart; the wrappers
follow its kernel-library convention
(python/avelang_kernels/amdgpu_gemm.py:458-494).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _native
from .layer_ops import _dt, _ptr, _stream

__all__ = ["layer_norm", "layer_norm_fwd_save", "layer_norm_bwd"]


def _args(x, weight, bias, name):
    """Checked, contiguous x and parameters, with rows, heads, D and type codes."""
    if not isinstance(x, torch.Tensor) or x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{name}: x must be a tensor with a last axis of at least 1.")
    dt = _dt(x, name, "x")
    dev = x.device
    if dev.type != "cuda":
        raise ValueError(f"{name}: tensors must be on a ROCm (cuda) device, got {dev}.")
    D, heads, wdt = x.shape[-1], 1, dt
    p = bias if weight is None else weight
    if p is not None:
        for nm, t in (("weight", weight), ("bias", bias)):
            if t is None:
                continue
            if not isinstance(t, torch.Tensor):
                raise ValueError(f"{name}: {nm} must be a torch.Tensor or None.")
            if t.dim() == 1:
                ok = t.shape[0] == D
            else:
                ok = t.dim() == 2 <= x.dim() and t.shape == x.shape[-2:]
            if not ok:
                raise ValueError(f"{name}: {nm} must have the shape of x's last axis or last two "
                                 f"axes, got {tuple(t.shape)} for x {tuple(x.shape)}.")
            if t.device != dev:
                raise ValueError(f"{name}: {nm} must be on {dev}, got {t.device}.")
        if bias is not None and p is not bias and (bias.dtype != p.dtype or bias.dim() != p.dim()):
            raise ValueError(f"{name}: weight and bias must share a shape and a dtype.")
        wdt = _dt(p, name, "weight")
        if p.dim() == 2:
            heads = p.shape[0]
            if heads < 1:
                raise ValueError(f"{name}: x must have at least one head.")
        if weight is not None:
            weight = weight.contiguous()
        if bias is not None:
            bias = bias.contiguous()
    return x.contiguous(), weight, bias, x.numel() // D, heads, D, dt, wdt


def _grad(t) -> bool:
    return isinstance(t, torch.Tensor) and t.requires_grad


def _fwd(args, eps, name, out=None, save=False):
    x, weight, bias, rows, heads, D, dt, wdt = args
    if out is None:
        y = torch.empty_like(x)
    else:
        y = out
        if (not isinstance(y, torch.Tensor) or y.shape != x.shape or y.dtype != x.dtype
                or y.device != x.device or not y.is_contiguous()):
            raise ValueError(f"{name}: out must be a contiguous {x.dtype} tensor of shape "
                             f"{tuple(x.shape)}.")
    stats = torch.empty((rows, 2), dtype=torch.float32, device=x.device) if save else None
    _native.check(_native.lib().gdn_layer_norm_fwd(
        x.data_ptr(), _ptr(weight), _ptr(bias), y.data_ptr(), _ptr(stats), rows, heads, D,
        float(eps), dt, wdt, _stream(x.device)), name)
    return y, stats


def layer_norm_fwd_save(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
                        bias: Optional[torch.Tensor] = None,
                        eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor]:
    """Training forward: ``(y, stats)``, ``stats`` fp32 [rows, 2] holding each
    row's mean and 1 / sqrt(var + eps) for ``layer_norm_bwd``."""
    name = "layer_norm_fwd_save"
    return _fwd(_args(x, weight, bias, name), eps, name, save=True)


def layer_norm_bwd(x: torch.Tensor, weight: Optional[torch.Tensor], dy: torch.Tensor,
                   stats: torch.Tensor, has_bias: bool = True):
    """Gradients of ``layer_norm``: ``(dx, dweight, dbias)``.

    dweight is None without a weight, dbias unless ``has_bias``; both have the
    weight's shape and type (without one: x's last axis, fp32) and are summed
    over the rows in fp32 in a fixed order.
    """
    name = "layer_norm_bwd"
    x, weight, _, rows, heads, D, dt, wdt = _args(x, weight, None, name)
    dev = x.device
    if not isinstance(dy, torch.Tensor) or dy.shape != x.shape or dy.dtype != x.dtype or dy.device != dev:
        raise ValueError(f"{name}: dy must be a {x.dtype} tensor of shape {tuple(x.shape)} on {dev}.")
    stats = _stats(stats, rows, dev, name)
    return _bwd(x, weight, dy, stats, rows, heads, D, dt, wdt if weight is not None else 0,
                torch.empty_like(weight) if weight is not None else None,
                None if not has_bias else torch.empty_like(weight) if weight is not None
                else torch.empty(D, dtype=torch.float32, device=dev), name)


def _stats(stats, rows, dev, name):
    if (not isinstance(stats, torch.Tensor) or stats.shape != (rows, 2) or stats.device != dev
            or stats.dtype is not torch.float32):
        raise ValueError(f"{name}: stats must be torch.float32 of shape {(rows, 2)} on {dev}.")
    return stats.contiguous()


def _bwd(x, weight, dy, stats, rows, heads, D, dt, wdt, dw, db, name):
    dy = dy.contiguous()
    dx = torch.empty_like(x)
    lib = _native.lib()
    ws, nbytes = None, 0
    if dw is not None or db is not None:
        nbytes = lib.gdn_layer_norm_bwd_workspace_bytes(rows, heads, D, dt)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    _native.check(lib.gdn_layer_norm_bwd(
        x.data_ptr(), _ptr(weight), dy.data_ptr(), stats.data_ptr(), dx.data_ptr(), _ptr(dw),
        _ptr(db), rows, heads, D, dt, wdt, _ptr(ws), nbytes, _stream(x.device)), name)
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        args = _args(x, weight, bias, "layer_norm")
        y, stats = _fwd(args, eps, "layer_norm", save=True)
        ctx.save_for_backward(args[0], args[1], args[2], stats)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, stats = ctx.saved_tensors
        # (checked again: a hook on saved tensors may return others of another layout;
        # dy is as autograd checked it, like the output)
        name = "layer_norm"
        x, weight, bias, *sizes = _args(x, weight, bias, name)
        stats = _stats(stats, sizes[0], x.device, name)
        if x.shape != dy.shape or x.dtype is not dy.dtype:
            raise ValueError(f"{name}: x must be saved as it was.")
        _, want_w, want_b, _ = ctx.needs_input_grad
        dw = torch.empty_like(weight) if want_w and weight is not None else None
        db = torch.empty_like(bias) if want_b and bias is not None else None
        dx, dw, db = _bwd(x, weight, dy, stats, *sizes, dw, db, name)
        return dx, dw, db, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, eps: float = 1e-5, *,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Layer norm of ``x`` (fp32, bf16 or fp16) over its last axis.

    ``weight`` and ``bias`` (each optional, sharing a shape and a type of their
    own): the last axis' shape, or the last two's for parameters per head.
    ``out`` (contiguous, may be ``x`` itself) avoids allocation.
    Differentiable in x, weight and bias (``layer_norm_bwd``); the forward then
    keeps 8 bytes per row.
    """
    if torch.is_grad_enabled() and (_grad(x) or _grad(weight) or _grad(bias)):
        if out is not None:
            raise ValueError("layer_norm: out is not supported when gradients are required.")
        return _LayerNorm.apply(x, weight, bias, eps)
    return _fwd(_args(x, weight, bias, "layer_norm"), eps, "layer_norm", out)[0]
