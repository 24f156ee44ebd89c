"""A paged key-value cache for MI355X (gfx950) and attention of the newest tokens over it.

Slot s of the cache is row ``s % page_size`` of page ``s // page_size``; a
sequence's tokens lie in the pages that its row of a block table names.  Rows are
kept as they come (bf16, fp16) or in 8 bits (float8_e4m3fn, int8) with an fp32
scale per token and kv-head, quantised as they are written:

    scale = max |row| / M (448, 127)      codes = row / scale, ties to even

The HIP kernels of ``csrc/gdn_paged*.hip`` behind ``include/gdn_attn.h``; there is
no fallback path.  The reference repository has no counterpart; the wrappers follow
its kernel-library convention (python/avelang_kernels/amdgpu_gemm.py:458-494).
"""
from __future__ import annotations

import functools
from typing import Optional, Tuple

import torch
from torch.autograd.graph import increment_version

from . import _native
from .layer_ops import _DTYPES, _ptr, _stream

__all__ = ["PagedKVCache", "paged_cache_write", "paged_cache_read", "paged_attention",
           "paged_attention_workspace_bytes"]

_SIZES = (64, 128, 256)
_HALF = (torch.bfloat16, torch.float16)
_CODES = {torch.float8_e4m3fn: _native.GDN_DTYPE_E4M3, torch.int8: _native.GDN_DTYPE_I8}
_TYPES = {torch.bfloat16: _native.GDN_DTYPE_BF16, torch.float16: _native.GDN_DTYPE_F16, **_CODES}


class PagedKVCache:
    """The tensors of a cache: ``k``, ``v`` [num_pages, kv_heads, page_size,
    head_size] (contiguous, 16-byte aligned; bf16, fp16, float8_e4m3fn or int8) and,
    in 8 bits, ``k_scale``, ``v_scale`` [num_pages, kv_heads, page_size] fp32.
    ``PagedKVCache.zeros`` allocates them; they are not replaced or resized later."""

    __slots__ = ("_held", "_versions", "sizes", "code")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                 v_scale: Optional[torch.Tensor] = None):
        name = "PagedKVCache"
        if not isinstance(k, torch.Tensor) or k.dim() != 4 or k.dtype not in _TYPES:
            raise ValueError(f"{name}: k must be a 4-D tensor [num_pages, kv_heads, page_size, "
                             "head_size] in bf16, fp16, float8_e4m3fn or int8.")
        dtype, dev, shape = k.dtype, k.device, k.shape
        pages, heads, page, size = shape
        if heads < 1 or page < 1 or size not in _SIZES:
            raise ValueError(f"{name}: kv_heads and page_size must be at least 1 and head_size one of "
                             f"{_SIZES}, got {tuple(shape)}.")
        if not isinstance(v, torch.Tensor) or v.shape != shape or v.dtype is not dtype or v.device != dev:
            raise ValueError(f"{name}: v must be like k, {dtype} of shape {tuple(shape)} on {dev}.")
        pk, pv = k.data_ptr(), v.data_ptr()
        if not k.is_contiguous() or not v.is_contiguous() or (pk | pv) % 16:
            raise ValueError(f"{name}: k and v must be contiguous and 16-byte aligned.")
        if dtype in _CODES:
            self._check_scale(k_scale, shape[:3], dev, "k_scale")
            self._check_scale(v_scale, shape[:3], dev, "v_scale")
        elif k_scale is not None or v_scale is not None:
            raise ValueError(f"{name}: a cache in {dtype} has no scales.")
        self._held = k, v, k_scale, v_scale
        self._versions = [t for t in self._held if t is not None and not t.is_inference()]
        self.sizes = heads, size, pages, page
        self.code = _TYPES[dtype]

    k = property(lambda self: self._held[0])
    v = property(lambda self: self._held[1])
    k_scale = property(lambda self: self._held[2])
    v_scale = property(lambda self: self._held[3])

    @property
    def ptrs(self):
        return [None if t is None else t.data_ptr() for t in self._held]

    @staticmethod
    def _check_scale(t, shape, dev, what):
        if (not isinstance(t, torch.Tensor) or t.shape != shape or t.device != dev
                or t.dtype is not torch.float32 or not t.is_contiguous() or t.data_ptr() % 16):
            raise ValueError(f"PagedKVCache: {what} must be a contiguous, 16-byte aligned "
                             f"torch.float32 tensor of shape {tuple(shape)} on {dev}.")

    @classmethod
    def zeros(cls, num_pages: int, page_size: int, kv_heads: int, head_size: int,
              dtype: torch.dtype = torch.bfloat16, device="cuda") -> "PagedKVCache":
        """An empty cache."""
        shape = (num_pages, kv_heads, page_size, head_size)
        rows = [torch.zeros(shape, dtype=dtype, device=device) for _ in "kv"]
        if dtype not in _CODES:
            return cls(*rows)
        return cls(*rows, *(torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in "kv"))


def _cache(cache, name):
    if not isinstance(cache, PagedKVCache):
        raise ValueError(f"{name}: cache must be a PagedKVCache.")
    if cache.k.device.type != "cuda":
        raise ValueError(f"{name}: tensors must be on a ROCm (cuda) device, got {cache.k.device}.")
    return cache


def _slots(slots, cache, name, distinct):
    """slots on the cache's device; one on the CPU is checked for two of a kind."""
    dev = cache.k.device
    if (not isinstance(slots, torch.Tensor) or slots.dtype not in (torch.int32, torch.int64)
            or slots.device not in (dev, torch.device("cpu"))):
        raise ValueError(f"{name}: slots must be int32 or int64 on {dev} or the CPU.")
    if slots.numel() >= 2 ** 31:
        raise ValueError(f"{name}: more than 2^31 - 1 slots in a call.")
    if slots.device.type == "cpu" and slots.numel():
        if distinct:
            used = slots[(slots >= 0) & (slots < cache.sizes[2] * cache.sizes[3])]
            if used.numel() != torch.unique(used).numel():
                raise ValueError(f"{name}: slots names one slot for two tokens.")
        slots = slots.to(dev)
    return slots.contiguous()


def paged_cache_write(cache: PagedKVCache, k: torch.Tensor, v: torch.Tensor,
                      slots: torch.Tensor) -> None:
    """Rows k, v [..., kv_heads, head_size] (bf16 or fp16; column slices of a projection
    are read in place) into the slots [...] (int32 / int64) of the cache, in its type:
    that of k and v, or 8 bits.

    A slot outside the cache marks a padding token, which is skipped.  Tokens must
    have distinct slots: two of a kind raise where the slots are on the CPU; on the
    device what that slot holds afterwards is not defined (no other slot is touched).
    In 8 bits a row of zeros has scale 0, one of less than 2^-100 is stored as if it
    reached that, and one that is not finite has a scale of NaN.
    """
    name = "paged_cache_write"
    _native.no_tangents(name, k, v)
    H, D, pages, page = _cache(cache, name).sizes
    dev = cache.k.device
    slots = _slots(slots, cache, name, True)
    shape = slots.shape + (H, D)
    if (not isinstance(k, torch.Tensor) or not isinstance(v, torch.Tensor) or k.shape != shape
            or v.shape != shape or k.device != dev or v.device != dev or v.dtype is not k.dtype
            or k.dtype not in _HALF):
        raise ValueError(f"{name}: k and v must be bf16 or fp16 tensors of one type and shape "
                         f"{tuple(shape)} on {dev}.")
    if cache.k.dtype is not k.dtype and cache.k.dtype not in _CODES:
        raise ValueError(f"{name}: a cache in {cache.k.dtype} takes rows of its type, got {k.dtype}.")
    if len(shape) != 3:
        k, v = k.reshape(-1, H, D), v.reshape(-1, H, D)
    if k.stride(2) != 1:
        k = k.contiguous()
    if v.stride(2) != 1:
        v = v.contiguous()
    sk, sv = k.stride(), v.stride()
    _native.check(_native.on_device(
        dev, _native.lib().gdn_paged_write, k.data_ptr(), v.data_ptr(), sk[0], sk[1], sv[0], sv[1],
        slots.data_ptr(), slots.dtype is torch.int64, *cache.ptrs, slots.numel(), H, D, pages, page,
        _DTYPES[k.dtype], cache.code, _stream(dev)), name)
    increment_version(cache._versions)   # (autograd, where it kept them, sees that they changed)


def paged_cache_read(cache: PagedKVCache, slots: torch.Tensor,
                     dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The rows ``(k, v)`` [..., kv_heads, head_size] that the slots [...] (int32 / int64)
    hold, codes times their scales rounded to ``dtype`` (bf16 or fp16; default the
    cache's own, bf16 in 8 bits).  A slot outside the cache gives zeros."""
    name = "paged_cache_read"
    _native.no_tangents(name, *getattr(cache, "_held", ()))
    H, D, pages, page = _cache(cache, name).sizes
    dev = cache.k.device
    slots = _slots(slots, cache, name, False)
    if dtype is None:
        dtype = torch.bfloat16 if cache.k.dtype in _CODES else cache.k.dtype
    if dtype not in _HALF or (cache.k.dtype not in _CODES and dtype != cache.k.dtype):
        raise ValueError(f"{name}: dtype must be bf16 or fp16, and the cache's unless it has 8 bits, "
                         f"got {dtype}.")
    k = torch.empty(slots.shape + (H, D), dtype=dtype, device=dev)
    v = torch.empty_like(k)
    _native.check(_native.on_device(
        dev, _native.lib().gdn_paged_read, *cache.ptrs, slots.data_ptr(),
        slots.dtype is torch.int64, k.data_ptr(), v.data_ptr(), slots.numel(), H, D, pages, page,
        _DTYPES[dtype], cache.code, _stream(dev)), name)
    return k, v


def paged_attention_workspace_bytes(N: int, L: int, Hq: int, Hkv: int, D: int, max_length: int) -> int:
    """Device scratch bytes ``paged_attention`` needs for N sequences of L new tokens each and
    lengths up to ``max_length``, or for any fewer or shorter with the same L and heads."""
    return int(_native.lib().gdn_paged_attn_workspace_bytes(N, L, Hq, Hkv, D, max_length))


@functools.lru_cache(maxsize=256)
def _workspace_bytes(device, *sizes):
    return _native.on_device(torch.device("cuda", device), _native.lib().gdn_paged_attn_workspace_bytes, *sizes)


def paged_attention(
    q: torch.Tensor,
    cache: PagedKVCache,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    scale: Optional[float] = None,
    *,
    window: int = 0,
    max_length: Optional[int] = None,
    return_lse: bool = False,
    out: Optional[torch.Tensor] = None,
    workspace: Optional[torch.Tensor] = None,
):
    """Attention of every sequence's newest L tokens over what it has cached, causal.

    ``q`` [N, L, Hq, D] bf16 or fp16 (the cache's type, or any of the two over an
    8-bit cache; q-head h reads kv-head h // (Hq // kv_heads)); ``lengths`` [N]
    int32: the tokens that are cached, the newest L (written before this call)
    among them; ``block_table`` [N, pages] int32: sequence n's token t is row
    ``t % page_size`` of page ``block_table[n, t // page_size]`` (page_size a
    multiple of 16).  ``scale`` defaults to ``D ** -0.5``.  With ``window`` > 0 a
    token sees itself and the ``window - 1`` before it.

    Returns o like q (contiguous), with ``return_lse`` ``(o, lse)``, lse fp32
    [N, L, Hq] the log of the softmax's sum.  A row that sees no token (lengths
    under L, or 0) is 0 with an lse of -inf.  ``max_length`` (default: what the
    table holds) bounds the lengths; a larger one counts as this.  How work is laid
    out follows from it: a tight one is faster where all are short.  Pages outside
    the cache give NaN; entries behind a sequence's last page are not read.
    ``out`` and ``workspace`` (uint8, ``paged_attention_workspace_bytes``; two
    captured graphs that may run at once need one each) avoid allocation.
    Deterministic.  Not differentiable.
    """
    name = "paged_attention"
    _native.no_tangents(name, q, *getattr(cache, "_held", ()))
    H, D, pages, page = _cache(cache, name).sizes
    dev = cache.k.device
    if (not isinstance(q, torch.Tensor) or q.dim() != 4 or q.shape[3] != D or q.device != dev
            or q.dtype not in _HALF):
        raise ValueError(f"{name}: q must be a bf16 or fp16 tensor [N, L, Hq, {D}] on {dev}.")
    N, L, Hq, _ = q.shape
    if L < 1 or Hq < 1 or Hq % H:
        raise ValueError(f"{name}: q must have at least one token, and heads ({Hq}) a multiple of the "
                         f"cache's ({H}).")
    if max(N, L, Hq) >= 2 ** 31:
        raise ValueError(f"{name}: q's axes must be under 2^31, got {tuple(q.shape)}.")
    if cache.k.dtype != q.dtype and cache.k.dtype not in _CODES:
        raise ValueError(f"{name}: a cache in {cache.k.dtype} takes queries of its type, got {q.dtype}.")
    if pages < 1 or page % 16:
        raise ValueError(f"{name}: the cache must have a page, and page_size be a multiple of 16, got "
                         f"{pages} of {page}.")
    if (not isinstance(lengths, torch.Tensor) or lengths.shape != (N,) or lengths.dtype != torch.int32
            or lengths.device != dev):
        raise ValueError(f"{name}: lengths must be int32 of shape ({N},) on {dev}.")
    if (not isinstance(block_table, torch.Tensor) or block_table.dim() != 2
            or block_table.shape[0] != N or block_table.dtype != torch.int32
            or block_table.device != dev):
        raise ValueError(f"{name}: block_table must be int32 of shape ({N}, pages) on {dev}.")
    if window < 0:
        raise ValueError(f"{name}: window must not be negative.")
    if block_table.stride(1) != 1 or block_table.stride(0) < block_table.shape[1]:
        block_table = block_table.contiguous()
    lengths = lengths.contiguous()   # (a copy lives until the launch)
    held = block_table.shape[1] * page
    if max_length is None:
        max_length = held
    elif not 0 <= max_length <= held:
        raise ValueError(f"{name}: max_length must be within the block table's {held} tokens.")
    if max_length > 1 << 30:
        raise ValueError(f"{name}: lengths of more than 2^30 tokens are not supported.")
    # (strides of an axis of one mean nothing)
    sn, sl, sh, se = q.stride()
    sn, sl, sh = sn if N > 1 else 0, sl if L > 1 else 0, sh if Hq > 1 else 0
    if se != 1 or (sn | sl | sh) % 8 or q.data_ptr() % 16:
        q = q.contiguous()
        q = q if q.data_ptr() % 16 == 0 else q.clone()
        sn, sl, sh = L * Hq * D, Hq * D, D
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    elif (not isinstance(out, torch.Tensor) or out.shape != q.shape or out.dtype != q.dtype
          or out.device != dev or not out.is_contiguous() or out.data_ptr() % 16):
        raise ValueError(f"{name}: out must be a contiguous, 16-byte aligned {q.dtype} tensor of shape "
                         f"{tuple(q.shape)} on {dev}.")
    elif not out.is_inference():
        increment_version(out)   # (autograd may have kept it)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=dev) if return_lse else None
    lib = _native.lib()
    if workspace is None:
        nbytes = _workspace_bytes(dev.index, N, L, Hq, H, D, max_length)
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    elif workspace.device != dev or not workspace.is_contiguous():   # (its size is checked by the entry point)
        raise ValueError(f"{name}: workspace must be contiguous on {dev}.")
    _native.check(_native.on_device(
        dev, lib.gdn_paged_attn_fwd, q.data_ptr(), sn, sl, sh, *cache.ptrs, block_table.data_ptr(),
        max(block_table.stride(0), block_table.shape[1]), lengths.data_ptr(), out.data_ptr(),
        _ptr(lse), N, L, Hq, H, D, pages, page, max_length, min(int(window), 1 << 30),
        D ** -0.5 if scale is None else float(scale), _DTYPES[q.dtype], cache.code, workspace.data_ptr(),
        workspace.numel() * workspace.element_size(), _stream(dev)), name)
    return (out, lse) if return_lse else out
