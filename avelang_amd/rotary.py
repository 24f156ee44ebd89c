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
    more than ``fast`` times keep theirs, a ramp that is linear in the number of
    turns lies between, and the magnitude is 0.1 ln(factor) + 1 (the formulas of
    arXiv 2309.00071, "YaRN", 3.2 and 3.4).  Programs whose ramp is linear in the
    pair's index instead, between two borders rounded to whole pairs, get other
    frequencies there: give ``rotary_embedding`` theirs.
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


def _turn(q, k, positions, inv_freq, magnitude, interleaved, inverse, inplace, name):
    """q and k (or None) turned: new contiguous tensors, or with ``inplace`` themselves."""
    _native.no_tangents(name, q, k, inv_freq)
    if not isinstance(q, torch.Tensor) or not 3 <= (dims := q.dim()) <= 4:
        raise ValueError(f"{name}: q must be a tensor [B, T, H, D] or [T, H, D].")
    dt, dev, shape = _dt(q, name, "q"), q.device, q.shape
    if dev.type != "cuda":
        raise ValueError(f"{name}: tensors must be on a ROCm (cuda) device, got {dev}.")
    B, T, H, D = shape if dims == 4 else (1, *shape)
    if H < 1 or D < 2 or D > 512 or D % 2:
        raise ValueError(f"{name}: q must have at least one head, and heads of an even size of at "
                         f"most 512, got {H} of {D}.")
    Hk = 0
    if k is not None:
        if (not isinstance(k, torch.Tensor) or k.dim() != dims or k.dtype is not q.dtype
                or k.device != dev):
            raise ValueError(f"{name}: k must be a {q.dtype} tensor like q on {dev}.")
        Hk = k.shape[-2]
        if k.shape[:-2] != shape[:-2] or k.shape[-1] != D or Hk < 1:
            raise ValueError(f"{name}: k must have q's axes but heads (at least one), got "
                             f"{tuple(k.shape)} beside {tuple(shape)}.")
    if B * T >= 2 ** 31 or max(H, Hk) > 1 << 20:
        raise ValueError(f"{name}: at most 2^31 - 1 tokens and 2^20 heads, got {tuple(shape)}.")
    if (not isinstance(inv_freq, torch.Tensor) or inv_freq.dim() != 1 or not inv_freq.is_floating_point()
            or inv_freq.device != dev or not 1 <= (R := inv_freq.shape[0]) <= D // 2):
        raise ValueError(f"{name}: inv_freq must be a 1-D floating point tensor on {dev} of 1 to "
                         f"{D // 2} frequencies.")
    if (not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64)
            or positions.device != dev or positions.shape != (B, T) and positions.shape != (T,)):
        raise ValueError(f"{name}: positions must be int32 or int64 of shape ({T},) or ({B}, {T}) on "
                         f"{dev}.")
    if inplace:
        for t in (q, k):
            if t is not None and (t.stride(-1) != 1 or not _apart(t)):
                raise ValueError(f"{name}: in place q and k must have contiguous heads and elements "
                                 "of their own.")
        qo, ko = q, k
    else:
        qo, ko = _new(q), None if k is None else _new(k)
    a, c = q.stride(), (0,) * 4 if k is None else k.stride()
    if a[-1] != 1:
        q = q.contiguous()
        a = q.stride()
    if k is not None and c[-1] != 1:
        k = k.contiguous()
        c = k.stride()
    a, c = (a[:3], c[:3]) if dims == 4 else ((0, *a[:2]), (0, *c[:2]))
    b, d = (a, c) if inplace else ((T * H * D, H * D, D), (T * Hk * D, Hk * D, D))
    positions, inv_freq = positions.contiguous(), inv_freq.double().contiguous()
    _native.check(_native.on_device(
        dev, _native.lib().gdn_rotary, q.data_ptr(), _ptr(k), qo.data_ptr(), _ptr(ko),
        _STRIDES(*a, *c, *b, *d), B, T, H, Hk, D, positions.data_ptr(), positions.dtype is torch.int64,
        T if positions.dim() == 2 else 0, inv_freq.data_ptr(), 2 * R, magnitude, interleaved, inverse,
        dt, _stream(dev)), name)
    if inplace:
        # (autograd, where it kept them, sees that they changed)
        increment_version([t for t in (q, k) if t is not None and not t.is_inference()])
    return qo, ko


def _new(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, magnitude, interleaved):
        qo, ko = _turn(q, k, positions, inv_freq, magnitude, interleaved, False, False,
                       "rotary_embedding")
        ctx.save_for_backward(positions, inv_freq)
        ctx.rest = magnitude, interleaved
        ctx.set_materialize_grads(False)
        return qo if k is None else (qo, ko)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk=None):
        positions, inv_freq = ctx.saved_tensors
        want_q, want_k = ctx.needs_input_grad[:2]
        if not want_q:
            dq = None
        if not want_k:
            dk = None
        a, b = (dk, None) if dq is None else (dq, dk)
        if a is None:
            return None, None, None, None, None, None
        a, b = _turn(a, b, positions, inv_freq, *ctx.rest, True, False, "rotary_embedding")
        return (*((None, a) if dq is None else (a, b)), None, None, None, None)


def rotary_embedding(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor,
                     inv_freq: torch.Tensor, *, magnitude: float = 1.0, interleaved: bool = False,
                     inplace: bool = False):
    """q and k (bf16, fp16 or fp32; [B, T, H, D] or [T, H, D], each with heads of its
    own) turned by their positions: ``(q', k')``, or q' alone where k is None.

    ``positions`` (int32 / int64, [T] or [B, T]) may be any integers; the first
    ``2 * len(inv_freq)`` elements of a head turn (``rotary_frequencies``; fp64 keeps
    far positions' angles), the rest is copied.  Strided inputs (column slices of a
    projection) are read in place; outputs are contiguous.  With ``inplace`` q and k,
    which share no element, are turned themselves and returned.  Differentiable in q
    and k (the gradient is turned back), not in place.
    """
    name = "rotary_embedding"
    if torch.is_grad_enabled() and (_grad(q) or _grad(k)):
        if inplace:
            raise ValueError(f"{name}: inplace is not supported when gradients are required.")
        return _Rotary.apply(q, k, positions, inv_freq, float(magnitude), bool(interleaved))
    q, k = _turn(q, k, positions, inv_freq, float(magnitude), bool(interleaved), False, inplace, name)
    return q if k is None else (q, k)
