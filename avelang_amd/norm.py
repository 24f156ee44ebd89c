"""Layer norm and root-mean-square norm for MI355X (gfx950), forward and backward.

    layer_norm   y = (x - mean) / sqrt(var + eps) * weight + bias
    rms_norm     y = h / sqrt(mean(h^2) + eps) * (weight + offset),  h = x [+ residual]

over the last axis with the biased variance, in fp32 whatever x's type.  The
layer norm's weight and bias have the last axis' shape, or the last two's: every
head's row by itself with parameters of its own (the norm of an attention's
output).  The RMS norm also adds the residual stream and can leave its output in
8 bits with a scale per row (``rms_norm_quant``).
HIP kernels of ``csrc/gdn_norm.hip`` behind ``include/gdn_linear.h`` and of
``csrc/gdn_rms.hip`` behind ``include/gdn_attn.h``; there is no fallback path.
The reference repository has no counterpart; the wrappers follow its
kernel-library convention (python/avelang_kernels/amdgpu_gemm.py:458-494).
"""
from __future__ import annotations

import functools
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _native
from .layer_ops import _DTYPES, _dt, _ptr, _stream

_CODES = {torch.float8_e4m3fn: _native.GDN_DTYPE_E4M3, torch.int8: _native.GDN_DTYPE_I8}

__all__ = ["layer_norm", "layer_norm_fwd_save", "layer_norm_bwd",
           "rms_norm", "rms_norm_quant", "rms_norm_bwd"]


def _args(x, weight, bias, name):
    """Checked, contiguous x and parameters, with rows, heads, D and type codes."""
    _native.no_tangents(name, x, weight, bias)
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
    _native.no_tangents(name, dy)
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


def _rms_args(x, weight, residual, name):
    """Checked, contiguous x, weight and residual, with rows, D and type codes."""
    _native.no_tangents(name, x, weight, residual)
    if not isinstance(x, torch.Tensor) or x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{name}: x must be a tensor with a last axis of at least 1.")
    dt = rdt = wdt = _dt(x, name, "x")
    dev, D = x.device, x.shape[-1]
    if D >= 2 ** 31:
        raise ValueError(f"{name}: rows must be shorter than 2^31, got {D}.")
    if dev.type != "cuda":
        raise ValueError(f"{name}: tensors must be on a ROCm (cuda) device, got {dev}.")
    if weight is not None:
        if not isinstance(weight, torch.Tensor) or weight.shape != (D,) or weight.device != dev:
            raise ValueError(f"{name}: weight must be a tensor of shape ({D},) on {dev}.")
        wdt = _dt(weight, name, "weight")
        weight = weight.contiguous()
    if residual is not None:
        if (not isinstance(residual, torch.Tensor) or residual.shape != x.shape
                or residual.device != dev or residual.dtype not in (x.dtype, torch.float32)):
            raise ValueError(f"{name}: residual must be a tensor of x's shape {tuple(x.shape)} and "
                             f"type or torch.float32 on {dev}.")
        rdt = _DTYPES[residual.dtype]
        residual = residual.contiguous()
    return x.contiguous(), weight, residual, x.numel() // D, D, dt, rdt, wdt


def _rms_out(t, like, name, what):
    if (not isinstance(t, torch.Tensor) or t.shape != like.shape or t.dtype != like.dtype
            or t.device != like.device or not t.is_contiguous()):
        raise ValueError(f"{name}: {what} must be a contiguous {like.dtype} tensor of shape "
                         f"{tuple(like.shape)} on {like.device}.")
    if not t.is_inference():
        increment_version(t)   # (it may be x or the residual, which autograd may have kept)
    return t


def _rms_fwd(args, eps, offset, name, out=None, residual_out=None, code=None):
    x, weight, residual, rows, D, dt, rdt, wdt = args
    dev, scale, ydt = x.device, None, dt
    if code is not None:
        y, ydt = torch.empty_like(x, dtype=code), _CODES[code]
        scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev)
    else:
        y = torch.empty_like(x) if out is None else _rms_out(out, x, name, "out")
    h = None
    if residual is not None:
        h = (torch.empty_like(residual) if residual_out is None
             else _rms_out(residual_out, residual, name, "residual_out"))
    elif residual_out is not None:
        raise ValueError(f"{name}: residual_out needs a residual.")
    _native.check(_native.on_device(
        dev, _native.lib().gdn_rms_norm_fwd, x.data_ptr(), _ptr(residual), _ptr(weight), y.data_ptr(),
        _ptr(h), _ptr(scale), rows, D, eps, offset, dt, rdt, wdt, ydt, _stream(dev)), name)
    return y, h, scale


def rms_norm_bwd(h: torch.Tensor, weight: Optional[torch.Tensor], dy: torch.Tensor,
                 dh: Optional[torch.Tensor] = None, eps: float = 1e-6, *, offset: float = 0.0):
    """Gradients of ``rms_norm``: ``(dx, dweight, dresidual)`` from h (x itself without a
    residual), dy = dL/dy (its type is x's) and dh = dL/dh (h's type; None where nothing
    else reads h).

    dresidual is dx itself where h has x's type; with an fp32 residual the same
    values in fp32.  dweight (None without a weight) has the weight's type and is
    summed over the rows in fp32 in a fixed order.
    """
    name = "rms_norm_bwd"
    if not isinstance(dy, torch.Tensor) or not isinstance(h, torch.Tensor):
        raise ValueError(f"{name}: h and dy must be tensors.")
    return _rms_bwd(_rms_args(dy, weight, h, name), dh, float(eps), float(offset),
                    weight is not None, True, name)


@functools.lru_cache(maxsize=256)
def _rms_bytes(device, rows, D, dt):
    return _native.on_device(torch.device("cuda", device), _native.lib().gdn_rms_norm_bwd_workspace_bytes,
                             rows, D, dt)


def _rms_bwd(args, dh, eps, offset, want_w, want_r, name):
    """On ``_rms_args`` of dy, weight and h."""
    _native.no_tangents(name, dh)
    dy, weight, h, rows, D, dt, hdt, wdt = args
    dev = dy.device
    if dh is not None:
        if (not isinstance(dh, torch.Tensor) or dh.shape != h.shape or dh.dtype is not h.dtype
                or dh.device != dev):
            raise ValueError(f"{name}: dh must be a {h.dtype} tensor of shape {tuple(h.shape)} on {dev}.")
        dh = dh.contiguous()
    dx, dw, dr, ws, nbytes = torch.empty_like(dy), None, None, None, 0
    if want_r and hdt != dt:
        dr = torch.empty_like(h)
    if want_w:
        dw = torch.empty_like(weight)
        nbytes = _rms_bytes(dev.index, rows, D, dt)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    _native.check(_native.on_device(
        dev, _native.lib().gdn_rms_norm_bwd, h.data_ptr(), _ptr(weight), dy.data_ptr(), _ptr(dh),
        dx.data_ptr(), _ptr(dr), _ptr(dw), rows, D, eps, offset, dt, hdt, wdt, _ptr(ws), nbytes,
        _stream(dev)), name)
    return dx, dw, (dr if dr is not None else dx) if want_r else None


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps, offset):
        args = _rms_args(x, weight, residual, "rms_norm")
        y, h, _ = _rms_fwd(args, eps, offset, "rms_norm")
        ctx.save_for_backward(args[0] if h is None else h, args[1])
        ctx.rest = eps, offset, x.dtype
        ctx.set_materialize_grads(False)
        return y if h is None else (y, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        h, weight = ctx.saved_tensors
        eps, offset, x_type = ctx.rest
        want_x, want_w, want_r, _, _ = ctx.needs_input_grad
        if dy is None:
            # (y unused: h's gradient alone)
            return (dh.to(x_type) if want_x and dh is not None else None,
                    torch.zeros_like(weight) if want_w else None, dh if want_r else None, None, None)
        # (checked again: a hook on saved tensors may return others of another layout)
        name = "rms_norm"
        dx, dw, dr = _rms_bwd(_rms_args(dy, weight, h, name), dh, eps, offset, want_w, want_r, name)
        return dx, dw, dr, None, None


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-6, *,
             residual: Optional[torch.Tensor] = None, offset: float = 0.0,
             out: Optional[torch.Tensor] = None, residual_out: Optional[torch.Tensor] = None):
    """RMS norm of ``x`` (fp32, bf16 or fp16) over its last axis:
    ``y = h * rsqrt(mean(h^2, -1) + eps) * (weight + offset)``.

    Without a ``residual`` h is x, and y is returned.  With one (x's shape; x's
    type or fp32) ``h = x + residual`` in the residual's type, and ``(y, h)`` is
    returned: h is what the next layer adds to, and y is the norm of h as
    returned.  ``weight`` (optional, any of the three types) has the last axis'
    shape; ``offset`` 1 is for weights stored about zero.  ``out`` (may be x)
    and ``residual_out`` (may be the residual, or x where the types are the same)
    avoid allocation; both contiguous.

    Differentiable in x, weight and residual (``rms_norm_bwd``, the gradient of h
    included); the forward then keeps h alone.
    """
    if torch.is_grad_enabled() and (_grad(x) or _grad(weight) or _grad(residual)):
        if out is not None or residual_out is not None:
            raise ValueError("rms_norm: out / residual_out are not supported when gradients are "
                             "required.")
        return _RmsNorm.apply(x, weight, residual, float(eps), float(offset))
    y, h, _ = _rms_fwd(_rms_args(x, weight, residual, "rms_norm"), eps, offset, "rms_norm", out,
                       residual_out)
    return y if h is None else (y, h)


def rms_norm_quant(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-6, *,
                   residual: Optional[torch.Tensor] = None, offset: float = 0.0,
                   dtype: torch.dtype = torch.float8_e4m3fn,
                   residual_out: Optional[torch.Tensor] = None):
    """``rms_norm`` with its output in 8 bits: ``(codes, scale)``, with a residual
    ``(codes, scale, h)``; y is ``codes * scale[..., None]``.

    ``dtype`` is torch.float8_e4m3fn (M = 448) or torch.int8 (M = 127); scale
    (fp32, one per row) is max |y| / M and codes are y / scale, rounded to nearest
    with ties to even: half a step off y (e4m3 2^-4 of it, int8 scale / 2).  A row of
    zeros has scale 0; one of less than 2^-100 is stored as if it reached that; one
    that is not finite has a scale of NaN.  Not differentiable.
    """
    name = "rms_norm_quant"
    if dtype not in _CODES:
        raise ValueError(f"{name}: dtype must be torch.float8_e4m3fn or torch.int8, got {dtype}.")
    y, h, scale = _rms_fwd(_rms_args(x, weight, residual, name), eps, offset, name, None,
                           residual_out, code=dtype)
    return (y, scale) if h is None else (y, scale, h)
