"""``PagedKVCache``: keys and values of cached tokens in pages.

The pages of one layer's key-value cache in HBM, for ``ops.append_kv`` and
``ops.paged_attention``.  Which pages a sequence owns is the caller's page
table (int32 [rows, pages], -1 where there is none): token j of row b lies in
page ``table[b, j // page_size]``, place ``j % page_size``.  No counterpart in
the reference (its attention blocks are mlx_lm's).
"""

from __future__ import annotations

import ctypes

import torch

from . import _abi

KV_DTYPES = {torch.bfloat16: 16, torch.float8_e4m3fn: 8}


class PagedKVCache:
    """Views of a layer's key and value pages, [pages, kv_heads, page_size,
    head_dim] each, bf16 or e4m3 (``float8_e4m3fn``).

    An 8-bit cache holds value / scale: ``k_scale`` and ``v_scale`` are fp32
    [kv_heads].  The tensors may be strided (pages of another order, keys and
    values in one buffer) as long as the last axis is contiguous, every stride
    is a multiple of 16 bytes, and keys and values have the same strides.
    """

    __slots__ = ("k", "v", "k_scale", "v_scale", "num_pages", "kv_heads", "page_size", "head_dim", "index", "address",
                 "_desc")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None):
        shape, strides, dtype, index = k.shape, k.stride(), k.dtype, k.get_device()
        same = v.stride() == strides
        if 1 in shape:  # the stride of an axis of one says nothing
            strides = tuple(0 if n == 1 else s for s, n in zip(strides, shape))
            same = v.shape == shape and strides == tuple(0 if n == 1 else s for s, n in zip(v.stride(), shape))
        if len(shape) != 4 or v.shape != shape or v.dtype != dtype or not same or v.get_device() != index:
            raise ValueError("k and v must be [pages, kv_heads, page_size, head_dim] tensors of one type and stride")
        bits = KV_DTYPES.get(dtype)
        if bits is None:
            raise TypeError(f"a cache holds bfloat16 or float8_e4m3fn values, not {dtype}")
        if index < 0:
            raise TypeError("a cache lies on a CUDA device")
        if strides[3] != 1:
            raise ValueError("the head axis of a cache must be contiguous")
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = shape
        ks = vs = None
        if bits == 8:
            for name, s in (("k_scale", k_scale), ("v_scale", v_scale)):
                if (s is None or s.dtype != torch.float32 or s.shape != (self.kv_heads,) or s.get_device() != index
                        or not s.is_contiguous()):
                    raise ValueError(f"an 8-bit cache needs {name}: contiguous fp32 [kv_heads]")
            ks, vs = k_scale.data_ptr(), v_scale.data_ptr()
        elif k_scale is not None or v_scale is not None:
            raise ValueError("scales belong to an 8-bit cache")
        self.k, self.v, self.k_scale, self.v_scale, self.index = k, v, k_scale, v_scale, index
        self._desc = _abi.sg_kv_cache(self.num_pages, self.kv_heads, self.page_size, self.head_dim, bits, 0, strides[0],
                                      strides[1], strides[2], k.data_ptr(), v.data_ptr(), ks, vs)
        self.address = ctypes.addressof(self._desc)  # the C-ABI descriptor

    @classmethod
    def empty(cls, num_pages: int, kv_heads: int, page_size: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
              k_scale: torch.Tensor | float = 1.0, v_scale: torch.Tensor | float = 1.0,
              device: str | torch.device = "cuda") -> "PagedKVCache":
        """A cache of its own, zeroed.  The scales of an 8-bit cache are one
        number for all heads or fp32 [kv_heads] (largest magnitude / 448 loses
        no range)."""
        if page_size < 1 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two")
        k, v = (torch.zeros((num_pages, kv_heads, page_size, head_dim), dtype=dtype, device=device) for _ in range(2))
        if KV_DTYPES.get(dtype) != 8:
            return cls(k, v)
        scales = [s if isinstance(s, torch.Tensor) else torch.full((kv_heads,), float(s), device=device)
                  for s in (k_scale, v_scale)]
        return cls(k, v, *scales)

    def nbytes(self) -> int:
        return 2 * self.k.numel() * self.k.element_size()
