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
from torch.autograd.graph import increment_version

from . import _native
from .layer_ops import _dt, _ptr, _stream
from .norm import _grad

__all__ = ["rotary_embedding", "rotary_frequencies"]

_STRIDES = ctypes.c_longlong * 12


def _apart(t) -> bool:
    """No two elements of t share memory (as far as strides in their order tell)."""
    reach = 0
    for stride, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if stride <= reach:
            return False
        reach += stride * (n - 1)
    return True


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


def _args(q, k, positions, inv_freq, name):
    """Checked q and k as 4-D tensors with contiguous elements, positions, fp64 frequencies and
    the type's code."""
    if not isinstance(q, torch.Tensor) or not 3 <= q.dim() <= 4:
        raise ValueError(f"{name}: q must be a tensor [B, T, H, D] or [T, H, D].")
    dt, dev = _dt(q, name, "q"), q.device
    if k is not None and (not isinstance(k, torch.Tensor) or k.dim() != q.dim()
                          or k.dtype is not q.dtype or k.device != dev):
        raise ValueError(f"{name}: k must be a {q.dtype} tensor like q on {dev}.")
    if q.dim() == 3:
        q, k = q[None], None if k is None else k[None]
    if dev.type != "cuda":
        raise ValueError(f"{name}: tensors must be on a ROCm (cuda) device, got {dev}.")
    B, T, H, D = q.shape
    if B * T >= 2 ** 31 or max(H, 0 if k is None else k.shape[2]) > 1 << 20:
        raise ValueError(f"{name}: at most 2^31 - 1 tokens and 2^20 heads, got {tuple(q.shape)}.")
    if H < 1 or D < 2 or D > 512 or D % 2:
        raise ValueError(f"{name}: q must have at least one head, and heads of an even size of at "
                         f"most 512, got {H} of {D}.")
    if k is not None and (k.shape[0] != B or k.shape[1] != T or k.shape[3] != D or k.shape[2] < 1):
        raise ValueError(f"{name}: k must have q's axes but heads (at least one), got {tuple(k.shape)} "
                         f"beside {tuple(q.shape)}.")
    if (not isinstance(inv_freq, torch.Tensor) or inv_freq.dim() != 1 or not inv_freq.is_floating_point()
            or inv_freq.device != dev or not 1 <= inv_freq.shape[0] <= D // 2):
        raise ValueError(f"{name}: inv_freq must be a 1-D floating point tensor on {dev} of 1 to "
                         f"{D // 2} frequencies.")
    if (not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64)
            or positions.device != dev or positions.shape != (B, T) and positions.shape != (T,)):
        raise ValueError(f"{name}: positions must be int32 or int64 of shape ({T},) or ({B}, {T}) on "
                         f"{dev}.")
    if q.stride(3) != 1:
        q = q.contiguous()
    if k is not None and k.stride(3) != 1:
        k = k.contiguous()
    return q, k, positions.contiguous(), inv_freq.double().contiguous(), dt


def _turn(q, k, qo, ko, positions, freq, dt, magnitude, interleaved, inverse, name):
    """qo, ko (4-D, q's and k's shapes) from q and k."""
    B, T, Hq, D = q.shape
    a, b = q.stride(), qo.stride()
    if k is None:
        Hk, strides = 0, _STRIDES(a[0], a[1], a[2], 0, 0, 0, b[0], b[1], b[2])
    else:
        c, d = k.stride(), ko.stride()
        Hk = k.shape[2]
        strides = _STRIDES(a[0], a[1], a[2], c[0], c[1], c[2], b[0], b[1], b[2], d[0], d[1], d[2])
    dev = q.device
    _native.check(_native.on_device(
        dev, _native.lib().gdn_rotary, q.data_ptr(), _ptr(k), qo.data_ptr(), _ptr(ko), strides, B, T,
        Hq, Hk, D, positions.data_ptr(), positions.dtype is torch.int64,
        T if positions.dim() == 2 else 0, freq.data_ptr(), 2 * freq.shape[0], magnitude, interleaved,
        inverse, dt, _stream(dev)), name)


def _new(t):
    return None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device)


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, magnitude, interleaved):
        name = "rotary_embedding"
        q4, k4, pos, freq, dt = _args(q, k, positions, inv_freq, name)
        qo, ko = _new(q4), _new(k4)
        _turn(q4, k4, qo, ko, pos, freq, dt, magnitude, interleaved, False, name)
        ctx.save_for_backward(positions, inv_freq)
        ctx.rest = magnitude, interleaved
        ctx.set_materialize_grads(False)
        if q.dim() == 3:
            qo, ko = qo[0], None if ko is None else ko[0]
        return qo if k is None else (qo, ko)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk=None):
        positions, inv_freq = ctx.saved_tensors
        magnitude, interleaved = ctx.rest
        name = "rotary_embedding"
        want_q, want_k = ctx.needs_input_grad[:2]
        a = dq if want_q else None
        b = dk if want_k else None
        if a is None:
            a, b = b, None
        if a is None:
            return None, None, None, None, None, None
        x, y, pos, freq, dt = _args(a, b, positions, inv_freq, name)
        xo, yo = _new(x), _new(y)
        _turn(x, y, xo, yo, pos, freq, dt, magnitude, interleaved, True, name)
        if a.dim() == 3:
            xo, yo = xo[0], None if yo is None else yo[0]
        if not want_q or dq is None:
            xo, yo = None, xo
        return xo, yo, None, None, None, None


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
    if torch.is_grad_enabled() and (_grad(q) or _grad(k)):
        if inplace:
            raise ValueError(f"{name}: inplace is not supported when gradients are required.")
        return _Rotary.apply(q, k, positions, inv_freq, float(magnitude), bool(interleaved))
    q4, k4, pos, freq, dt = _args(q, k, positions, inv_freq, name)
    if inplace:
        for t in (q, k):
            if t is not None and (t.stride(-1) != 1 or not _apart(t)):
                raise ValueError(f"{name}: in place q and k must have contiguous heads and elements "
                                 "of their own.")
        qo, ko = q4, k4
    else:
        qo, ko = _new(q4), _new(k4)
    _turn(q4, k4, qo, ko, pos, freq, dt, float(magnitude), bool(interleaved), False, name)
    if inplace:
        qo, ko = q, k
        # (autograd, where it kept them, sees that they changed)
        increment_version([t for t in (q, k) if t is not None and not t.is_inference()])
    elif q.dim() == 3:
        qo, ko = qo[0], None if ko is None else ko[0]
    return qo if k is None else (qo, ko)
