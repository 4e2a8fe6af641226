"""A paged key/value cache: the tensors, and the description the kernels take.

``k`` and ``v`` are ``[pages, page_size, kv_heads, head_dim]`` views with
contiguous vectors and equal strides, so pages may be stored token-major or
head-major. An e4m3 cache has one scale byte per vector, ``[pages, page_size,
kv_heads]`` uint8: byte b stands for ``2 ** (b - 127)`` and a code for ``code * 2
** (b - 127)``; b lies in 103 .. 134, or is 255 (NaN) or 0 (an unwritten slot).

Slot s of the cache is page ``s // page_size``, offset ``s % page_size``.
:func:`ops.kv_cache_write` fills slots, :func:`ops.kv_cache_read` reads them
back, :func:`ops.paged_attention` attends over them.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib

_CODES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16,
          torch.float8_e4m3fn: _lib.DTYPE_E4M3}


class PagedKVCache:
    """One layer's cache. The tensors stay the caller's: writing through them
    and through the ops is the same memory."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "num_pages", "page_size", "kv_heads", "head_dim",
                 "_struct", "desc")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.stride() != v.stride():
            raise ValueError("k and v must be [pages, page_size, kv_heads, head_dim], alike in type "
                             f"and strides, got {tuple(k.shape)} {k.dtype}, {tuple(v.shape)} {v.dtype}")
        if k.dtype not in _CODES:
            raise TypeError(f"the cache must be bf16, f16 or float8_e4m3fn, got {k.dtype}")
        if k.stride(3) != 1:
            raise ValueError("the vectors of k and v must be contiguous")
        quantized = k.dtype == torch.float8_e4m3fn
        if quantized != (k_scale is not None) or quantized != (v_scale is not None):
            raise ValueError("scales belong to an e4m3 cache, and an e4m3 cache needs both")
        if quantized:
            if k_scale.shape != k.shape[:3] or v_scale.shape != k.shape[:3] \
                    or k_scale.stride() != v_scale.stride():
                raise ValueError(f"scales must be {tuple(k.shape[:3])}, alike in strides, got "
                                 f"{tuple(k_scale.shape)}, {tuple(v_scale.shape)}")
            if k_scale.dtype != torch.uint8 or v_scale.dtype != torch.uint8:
                raise TypeError("scales must be uint8")
        if any(t is not None and t.device != k.device for t in (v, k_scale, v_scale)):
            raise ValueError("the cache's tensors are on different devices")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.num_pages, self.page_size, self.kv_heads, self.head_dim = (int(d) for d in k.shape)
        ss = k_scale.stride() if quantized else (0, 0, 0)
        self._struct = _lib.KVCacheDesc(
            k=k.data_ptr(), v=v.data_ptr(),
            k_scale=k_scale.data_ptr() if quantized else None,
            v_scale=v_scale.data_ptr() if quantized else None,
            num_pages=self.num_pages, page_size=self.page_size, kv_heads=self.kv_heads,
            head_dim=self.head_dim, dtype=_CODES[k.dtype], page_stride=k.stride(0),
            token_stride=k.stride(1), head_stride=k.stride(2), scale_page_stride=ss[0],
            scale_token_stride=ss[1], scale_head_stride=ss[2],
        )
        self.desc = ctypes.addressof(self._struct)

    @classmethod
    def empty(cls, num_pages: int, page_size: int, kv_heads: int, head_dim: int, device,
              dtype: torch.dtype = torch.float8_e4m3fn) -> "PagedKVCache":
        """A cache in the layout the kernels read best: head-major pages, so that
        one head's tokens of a page are one contiguous run."""
        raw = torch.uint8 if dtype == torch.float8_e4m3fn else dtype
        kv = [torch.empty(num_pages, kv_heads, page_size, head_dim, dtype=raw, device=device)
              .view(dtype).transpose(1, 2) for _ in range(2)]
        scales = [torch.zeros(num_pages, kv_heads, page_size, dtype=torch.uint8, device=device)
                  .transpose(1, 2) if dtype == torch.float8_e4m3fn else None for _ in range(2)]
        return cls(*kv, *scales)
