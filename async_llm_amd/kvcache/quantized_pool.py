"""Paged K/V pool in 8 bits.

The counterpart of ``MHAKVCache`` for caches that hold twice the tokens: a row (one
token of one kv head) is ``head_dim`` codes of one byte and a scale byte, and stands
for ``code * 2 ** (scale - 127)``.  ``code_dtype`` is ``torch.float8_e4m3fn`` (an
element is off by at most 2^-4 of itself) or ``torch.int8`` (by at most half a step;
the row's largest magnitude is 64 to 127 steps).  Scales are powers of two, so that
reading back is exact in bfloat16 and float32, and storing what was read back stores
the same values.

Layout: codes ``[2, layers, num_pages, kv_heads, page_size, head_dim]`` and scales
without the last axis, K then V.  Within a page the rows of a kv head lie together,
which is how attention reads them; slot ``s`` is row ``s % page_size`` of page
``s // page_size``.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import native


class QuantizedKVCache:
    def __init__(self, num_kv_heads: int, num_layers: int, head_dim: int, num_pages: int, page_size: int,
                 dtype: torch.dtype, device: torch.device, code_dtype: torch.dtype = torch.float8_e4m3fn) -> None:
        """``dtype``: the type of the rows that are stored and read back."""
        native.code_id(code_dtype)
        shape = (2, num_layers, num_pages, num_kv_heads, page_size)
        self._adopt(torch.zeros((*shape, head_dim), device=device, dtype=torch.uint8).view(code_dtype),
                    torch.full(shape, 127, device=device, dtype=torch.uint8), dtype)

    @classmethod
    def from_buffers(cls, codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype) -> "QuantizedKVCache":
        """A pool over existing arrays of the layout above (``scales``: ``torch.uint8`` or ``torch.float8_e8m0fnu``)."""
        self = cls.__new__(cls)
        self._adopt(codes, scales, dtype)
        return self

    def _adopt(self, codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype) -> None:
        code_id = native.code_id(codes.dtype)
        if codes.dim() != 6 or codes.shape[0] != 2 or scales.shape != codes.shape[:-1]:
            raise ValueError("a quantised pool is codes [2, layers, pages, kv_heads, page_size, head_dim] and scales "
                             f"[2, layers, pages, kv_heads, page_size], got {tuple(codes.shape)} and {tuple(scales.shape)}")
        if scales.dtype not in (torch.uint8, torch.float8_e8m0fnu):
            raise ValueError(f"scales are torch.uint8 or torch.float8_e8m0fnu, got {scales.dtype}")
        if not codes.is_contiguous() or not scales.is_contiguous() or scales.device != codes.device:
            raise ValueError("codes and scales must be contiguous arrays on one device")
        if codes.shape[-1] not in (16, 32, 64, 128, 256):
            raise ValueError(f"head_dim {codes.shape[-1]} unsupported (16, 32, 64, 128 or 256)")
        _, self._num_layers, self._num_pages, self._num_kv_heads, self._page_size, self._head_dim = codes.shape
        if self._num_pages * self._page_size > 2**31 - 1:
            raise ValueError(f"{self._num_pages} pages of {self._page_size} tokens are more slots than 32 bits address")
        if codes.numel() and codes.data_ptr() % 16:
            raise ValueError("codes must start on a 16-byte boundary")
        self._codes, self._scales, self._dtype = codes, scales.view(torch.uint8), dtype
        self._shape = native.make_shape(self._num_kv_heads, self._num_kv_heads, self._head_dim, self._page_size, dtype)
        self._device = codes.device  # (asking the tensor costs a launch's arguments their time)
        # the descriptions of the layers' arrays, made once: addresses do not change
        c, s = codes.data_ptr(), scales.data_ptr()
        self.code_layer_bytes = self._num_pages * self._num_kv_heads * self._page_size * self._head_dim
        self.scale_layer_bytes = self.code_layer_bytes // self._head_dim
        L = self._num_layers
        self._layers = [native.VaQuantPool(c + l * self.code_layer_bytes, c + (L + l) * self.code_layer_bytes,
                                           s + l * self.scale_layer_bytes, s + (L + l) * self.scale_layer_bytes, code_id,
                                           self._num_pages) for l in range(L)]

    def k_codes(self, index: int) -> torch.Tensor:
        """``[num_pages, kv_heads, page_size, head_dim]`` of ``code_dtype``."""
        return self._codes[0, index]

    def v_codes(self, index: int) -> torch.Tensor:
        return self._codes[1, index]

    def k_scales(self, index: int) -> torch.Tensor:
        """``[num_pages, kv_heads, page_size]`` powers of two, as ``torch.float8_e8m0fnu``."""
        return self._scales[0, index].view(torch.float8_e8m0fnu)

    def v_scales(self, index: int) -> torch.Tensor:
        return self._scales[1, index].view(torch.float8_e8m0fnu)

    def layer(self, index: int) -> native.VaQuantPool:
        """A layer's arrays as the library takes them."""
        if not 0 <= index < self._num_layers:
            raise IndexError(f"layer {index} of a pool of {self._num_layers}")
        return self._layers[index]

    def store_kv(self, k: torch.Tensor, v: torch.Tensor, out_loc: torch.Tensor, layer_id: int) -> None:
        """Quantise rows of ``k`` / ``v`` as they are (keys already rotated) and write them to slots ``out_loc``;
        rows whose slot is negative are skipped."""
        store_quantized(self, k, v, out_loc, layer_id, None, None)

    def load_kv(self, slots: torch.Tensor, layer_id: int,
                out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """The K and V rows of ``slots`` (int64 on the device) as ``[n, kv_heads, head_dim]`` tensors of ``dtype``:
        new ones, or ``out``, whose rows may lie apart.  Negative slots give rows of zeros."""
        native.require_device(slots, "slots")
        device = self._device
        if slots.dim() != 1 or slots.dtype is not torch.int64 or slots.device != device:
            raise ValueError(f"slots must be one row of int64 on {device}, got {slots.dtype} "
                             f"{tuple(slots.shape)} on {slots.device}")
        slots = slots.contiguous()
        shape = (slots.numel(), self._num_kv_heads, self._head_dim)
        width = self._num_kv_heads * self._head_dim
        if out is None:
            k = torch.empty_strided(shape, (width, self._head_dim, 1), dtype=self._dtype, device=device)
            v = torch.empty_like(k)
            stride = width
        else:
            k, v = out
            for t in (k, v):
                rows_ok = t.stride()[1:] == (self._head_dim, 1) and t.stride() == k.stride() if t.dim() == 3 else False
                if tuple(t.shape) != shape or t.dtype != self._dtype or t.device != slots.device or not rows_ok:
                    raise ValueError(f"out must be two {self._dtype} tensors {shape} on {slots.device} with contiguous rows, "
                                     "equally far apart")
            stride = k.stride(0) if shape[0] > 1 else width
            if stride < width:
                raise ValueError("the rows of out overlap")
        native.call_on(device, native.lib.va_load_kv_q8, self.layer(layer_id), slots.data_ptr(), shape[0], k.data_ptr(),
                       v.data_ptr(), stride, self._shape, native.current_stream_ptr(device))
        return k, v

    @property
    def device(self) -> torch.device:
        return self._device

    @property
    def dtype(self) -> torch.dtype:
        return self._dtype

    @property
    def code_dtype(self) -> torch.dtype:
        return self._codes.dtype

    @property
    def num_layers(self) -> int:
        return self._num_layers

    @property
    def num_pages(self) -> int:
        return self._num_pages

    @property
    def page_size(self) -> int:
        return self._page_size

    @property
    def num_kv_heads(self) -> int:
        return self._num_kv_heads

    @property
    def head_dim(self) -> int:
        return self._head_dim


_NO_ROPE = native.VaRope(native.VA_ROPE_TABLE, 0, None, 0, 0, 0, None)


def _rows(pool: QuantizedKVCache, x: torch.Tensor, n: int, width: int, name: str):
    """``x`` as ``n`` rows of ``width`` adjacent elements, and how far apart they are."""
    shape = x.shape
    if x.dtype is not pool._dtype or x.device != pool._device or shape[0] != n or x.numel() != n * width:
        native.require_device(x, name)
        raise ValueError(f"{name} must be {n} rows of {width} {pool._dtype} elements on {pool._device}, got {x.dtype} "
                         f"{tuple(shape)} on {x.device}")
    if len(shape) != 2:
        x = x.reshape(n, width)
    stride, element = x.stride()
    return (x, stride) if element == 1 else (x.contiguous(), width)


def store_quantized(pool: QuantizedKVCache, k: torch.Tensor, v: torch.Tensor, out_loc: torch.Tensor, layer_id: int,
                    positions: Optional[torch.Tensor], rope: Optional[native.VaRope]) -> None:
    """Rotate the keys to ``positions`` (``[n]`` or ``[3, n]`` int64; ``None``: as they are), quantise and scatter."""
    width, device = pool._num_kv_heads * pool._head_dim, pool._device
    n = k.shape[0]
    k, k_stride = _rows(pool, k, n, width, "k")
    v, v_stride = _rows(pool, v, n, width, "v")
    wide = out_loc.dtype is torch.int64
    if not (wide or out_loc.dtype is torch.int32) or out_loc.numel() != n or out_loc.device != device:
        raise ValueError(f"out_loc must be {n} int32 or int64 slots on {device}, got {out_loc.numel()} {out_loc.dtype} "
                         f"on {out_loc.device}")
    native.require_device(k, "k")
    if n == 0:
        return
    out_loc = out_loc.contiguous()
    where, axis_stride = None, 0
    if positions is not None:
        if positions.dtype is not torch.int64 or positions.device != device:
            positions = positions.to(device=device, dtype=torch.int64)
        positions = positions.contiguous()
        if positions.numel() != n or positions.dim() != 1:
            if tuple(positions.shape) != (3, n):
                raise ValueError(f"positions must be [{n}] or [3, {n}], got {tuple(positions.shape)}")
            axis_stride = n
        where = positions.data_ptr()
    native.call_on(device, native.lib.va_store_kv_rope_q8, k.data_ptr(), v.data_ptr(), k_stride, v_stride,
                   pool.layer(layer_id), out_loc.data_ptr(), wide, where, axis_stride, n, pool._shape,
                   _NO_ROPE if rope is None else rope, native.current_stream_ptr(device))
