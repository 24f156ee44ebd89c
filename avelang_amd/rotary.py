"""Rotary positions for MI355X (gfx950).

The first ``2 * len(inv_freq)`` elements of every head turn in pairs, pair j at
position p by the angle ``p * inv_freq[j]``:

    (a, b) -> magnitude * (a cos - b sin, b cos + a sin)

pairs (j, j + r / 2) or, ``interleaved``, neighbours (2 j, 2 j + 1); the rest of
the head stays as it is.  There is no table: angles are formed and reduced in 64
bits where they are used, for any position.  The HIP kernel of
``csrc/gdn_rotary.hip`` behind ``include/gdn_attn.h``; there is no fallback path.
The reference repository has no counterpart; the wrappers follow its
kernel-library convention (python/avelang_kernels/amdgpu_gemm.py:458-494).
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _native
from .layer_ops import _dt, _stream

__all__ = ["rotary_embedding", "rotary_frequencies"]

_P2, _L6, _I2 = ctypes.c_void_p * 2, ctypes.c_longlong * 6, ctypes.c_int * 2


def rotary_frequencies(dim: int, base: float = 10000.0, *, factor: float = 1.0, original: int = 0,
                       slow: float = 1.0, fast: float = 32.0,
                       device: Optional[torch.device] = None) -> Tuple[torch.Tensor, float]:
    """Frequencies ``base ** (-2 j / dim)`` (fp64 [dim / 2]) and the magnitude for
    ``rotary_embedding``, stretched for contexts ``factor`` times as long as trained.

    With ``original`` = 0 every frequency is divided by ``factor`` and the
    magnitude is 1.  Else ``original`` is the trained context: pairs that turn
    less than ``slow`` times over it are divided by the factor, those that turn
    more than ``fast`` times keep theirs, a linear ramp lies between, and the
    magnitude is 0.1 ln(factor) + 1.
    """
    name = "rotary_frequencies"
    if dim < 2 or dim % 2 or not base > 0 or not factor > 0 or original < 0:
        raise ValueError(f"{name}: dim must be even and at least 2, base and factor positive and "
                         "original not negative.")
    f = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    size = 1.0
    if factor != 1 and original == 0:
        f = f / factor
    elif factor != 1:
        if not fast > slow:
            raise ValueError(f"{name}: fast must be more than slow.")
        keep = ((original * f / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
        size = 0.1 * math.log(factor) + 1 if factor > 1 else 1.0
    return f.to(device) if device is not None else f, size


def _apart(t) -> bool:
    """No two elements of t share memory (as far as strides in their order tell)."""
    reach = 0
    for stride, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if stride <= reach:
            return False
        reach += stride * (n - 1)
    return True


def _args(q, k, positions, inv_freq, name):
    """Checked q and k as 4-D views, positions with their batch stride, fp64 frequencies."""
    xs = []
    for nm, t in (("q", q), ("k", k)):
        if t is None and nm == "k":
            continue
        if not isinstance(t, torch.Tensor) or t.dim() not in (3, 4):
            raise ValueError(f"{name}: {nm} must be a tensor [B, T, H, D] or [T, H, D].")
        xs.append(t if t.dim() == 4 else t[None])
    q4 = xs[0]
    dt = _dt(q4, name, "q")
    dev, (B, T, _, D) = q4.device, q4.shape
    if dev.type != "cuda":
        raise ValueError(f"{name}: tensors must be on a ROCm (cuda) device, got {dev}.")
    if len(xs) == 2:
        k4 = xs[1]
        if (k.dim() != q.dim() or k4.shape[:2] != (B, T) or k4.shape[3] != D or k4.dtype != q4.dtype
                or k4.device != dev):
            raise ValueError(f"{name}: k must be {q4.dtype} like q on {dev}, with q's axes but heads.")
    if any(t.shape[2] < 1 for t in xs):
        raise ValueError(f"{name}: q and k must have at least one head.")
    if D < 2 or D > 512 or D % 2:
        raise ValueError(f"{name}: head size must be even and at most 512, got {D}.")
    if (not isinstance(inv_freq, torch.Tensor) or inv_freq.dim() != 1 or not inv_freq.is_floating_point()
            or inv_freq.device != dev or not 1 <= inv_freq.numel() <= D // 2):
        raise ValueError(f"{name}: inv_freq must be a 1-D floating point tensor on {dev} of 1 to "
                         f"{D // 2} frequencies.")
    if (not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64)
            or positions.device != dev or tuple(positions.shape) not in ((T,), (B, T))):
        raise ValueError(f"{name}: positions must be int32 or int64 of shape ({T},) or ({B}, {T}) on "
                         f"{dev}.")
    batch = T if positions.dim() == 2 else 0
    xs = [t if t.stride(3) == 1 else t.contiguous() for t in xs]
    return xs, positions.contiguous(), batch, inv_freq.double().contiguous(), dt


def _turn(xs, ys, positions, batch, freq, dt, magnitude, interleaved, inverse, name):
    """ys (4-D, of xs' shapes) from xs."""
    B, T, _, D = xs[0].shape
    x, y, heads = _P2(), _P2(), _I2()
    sx, sy = _L6(), _L6()
    for i, (a, b) in enumerate(zip(xs, ys)):
        x[i], y[i], heads[i] = a.data_ptr(), b.data_ptr(), a.shape[2]
        sx[3 * i:3 * i + 3] = a.stride()[:3]
        sy[3 * i:3 * i + 3] = b.stride()[:3]
    dev = xs[0].device
    _native.check(_native.on_device(
        dev, _native.lib().gdn_rotary, x, y, sx, sy, heads, positions.data_ptr(),
        positions.dtype is torch.int64, batch, freq.data_ptr(), B, T, D, 2 * freq.numel(),
        float(magnitude), bool(interleaved), bool(inverse), dt, _stream(dev)), name)


def _new(xs):
    return [torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in xs]


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, magnitude, interleaved):
        name = "rotary_embedding"
        xs, pos, batch, freq, dt = _args(q, k, positions, inv_freq, name)
        ys = _new(xs)
        _turn(xs, ys, pos, batch, freq, dt, magnitude, interleaved, False, name)
        ctx.save_for_backward(positions, inv_freq)
        ctx.rest = magnitude, interleaved, [t.shape for t in (q, k) if t is not None]
        ctx.set_materialize_grads(False)
        ys = [y.view(s) for y, s in zip(ys, ctx.rest[2])]
        return ys[0] if k is None else tuple(ys)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        positions, inv_freq = ctx.saved_tensors
        magnitude, interleaved, _ = ctx.rest
        name = "rotary_embedding"
        out = [None, None]
        at = [i for i, g in enumerate(grads) if g is not None and ctx.needs_input_grad[i]]
        if at:
            g = [grads[i] for i in at]
            xs, pos, batch, freq, dt = _args(g[0], g[1] if len(g) > 1 else None, positions, inv_freq, name)
            ys = _new(xs)
            _turn(xs, ys, pos, batch, freq, dt, magnitude, interleaved, True, name)
            for i, y in zip(at, ys):
                out[i] = y.view(grads[i].shape)
        return out[0], out[1], None, None, None, None


def rotary_embedding(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor,
                     inv_freq: torch.Tensor, *, magnitude: float = 1.0, interleaved: bool = False,
                     inplace: bool = False):
    """q and k (bf16, fp16 or fp32; [B, T, H, D] or [T, H, D], each with heads of its
    own) turned by their positions: ``(q', k')``, or q' alone where k is None.

    ``positions`` (int32 / int64, [T] or [B, T]) may be any integers; the first
    ``2 * len(inv_freq)`` elements of a head turn (``rotary_frequencies``; fp64 keeps
    far positions' angles), the rest is copied.  Strided inputs (column slices of a
    projection) are read in place; outputs are contiguous.  With ``inplace`` q and k
    themselves are turned and returned.  Differentiable in q and k (the gradient is
    turned back), not in place.
    """
    name = "rotary_embedding"
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (q, k)):
        if inplace:
            raise ValueError(f"{name}: inplace is not supported when gradients are required.")
        return _Rotary.apply(q, k, positions, inv_freq, float(magnitude), bool(interleaved))
    xs, pos, batch, freq, dt = _args(q, k, positions, inv_freq, name)
    if inplace:
        if any(t.stride(-1) != 1 or not _apart(t) for t in (q, k) if t is not None):
            raise ValueError(f"{name}: in place q and k must have contiguous heads and elements of "
                             "their own.")
        ys = xs
    else:
        ys = _new(xs)
    _turn(xs, ys, pos, batch, freq, dt, magnitude, interleaved, False, name)
    if inplace:
        return q if k is None else (q, k)
    ys = [y if t.dim() == 4 else y[0] for y, t in zip(ys, (q, k))]
    return ys[0] if k is None else (ys[0], ys[1])
