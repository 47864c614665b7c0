"""8-bit KV caches: the two cache records and the row format they share.

A cache row - one token of one KV head, ``D`` values of K or V - is held as ``D`` codes of 8 bits
(``torch.float8_e4m3fn`` or ``torch.int8``) and one power-of-two scale ``2 ** (e - 127)`` held as the
byte ``e`` (255: NaN): half the bytes of a 16-bit cache plus one per row.  ``e`` is the smallest
exponent (at least 27) with ``max|x| <= top * 2 ** (e - 127)``, ``top`` being 448 for e4m3 and 127 for
int8; a code is ``x / 2 ** (e - 127)`` rounded to the code's type, halves to even.  Dividing by a
power of two is exact, so the codes do not depend on the arithmetic that computed them, reading back
into bf16/fp16/fp32 is exact (short of the target's range), and quantising what was read back keeps the
values.  It keeps int8 codes and scale bytes too; an e4m3 row whose largest element was rounded down to the code 224
gets twice the codes and the next smaller scale.  A row that holds an infinity or a NaN is stored with ``e = 255`` and codes 0:
it reads back as NaN and makes the outputs of its KV head NaN.

Scales lie head-major whatever the codes' layout is, the K and the V byte of a token side by side:
``[B, Hkv, N, 2]`` or ``[num_pages, Hkv, page_size, 2]``, dtype ``torch.uint8`` (or
``torch.float8_e8m0fnu``, the same bytes as numbers).

The reference has no quantised cache.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Union

import torch

from . import native

_CODE_DTYPES = "float8_e4m3fn or int8"
_SCALE_DTYPES = (torch.uint8, torch.float8_e8m0fnu)


def _need(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def _empty_rows(shape, scale_shape, dtype, device):
    _need(dtype in native.SA_KV_CODE, f"8-bit cache codes must be {_CODE_DTYPES}")
    key = torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype)
    value = torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype)
    return key, value, torch.zeros(scale_shape, dtype=torch.uint8, device=device)


def _check_codes(key: torch.Tensor, value: torch.Tensor, scales: torch.Tensor) -> None:
    _need(key.dim() == 4 and value.dim() == 4, "8-bit key/value caches must be rank 4")
    _need(key.dtype in native.SA_KV_CODE and value.dtype == key.dtype, f"8-bit cache codes must be {_CODE_DTYPES}")
    _need(key.shape == value.shape and key.stride() == value.stride(),
          "8-bit key and value caches must have identical shape and strides")
    _need(min(key.shape) > 0, "8-bit cache dimensions must be positive")
    _need(int(key.shape[3]) <= 256, "head_dim must be no larger than 256")
    _need(key.stride(3) == 1 or int(key.shape[3]) == 1, "cache head_dim must be contiguous")
    _need(scales.dtype in _SCALE_DTYPES, "scales must be uint8 or float8_e8m0fnu")


@dataclass(frozen=True)
class QuantKVCache:
    """Contiguous 8-bit cache.

    ``key``/``value`` are codes ``[B, Hkv, N, D]`` (``layout="BHND"``) or ``[B, N, Hkv, D]`` (``"BNHD"``),
    ``scales`` is ``[B, Hkv, N, 2]``; ``sequence_lengths`` (``[B]`` int32/int64 on the device, read by
    every run) says how many tokens the rows hold, ``None`` that they hold ``N``.  The tensor-core
    decode kernel wants ``N`` to be a multiple of 8 (:meth:`empty` rounds up); other capacities are
    served by the generic kernel.
    """

    key: torch.Tensor
    value: torch.Tensor
    scales: torch.Tensor
    sequence_lengths: Optional[torch.Tensor] = None
    layout: str = "BHND"

    @classmethod
    def empty(cls, batch: int, kv_heads: int, capacity: int, head_dim: int, *, dtype: torch.dtype = torch.float8_e4m3fn,
              layout: str = "BHND", device: Union[str, torch.device] = "cuda") -> "QuantKVCache":
        """An empty cache (lengths 0) with room for at least ``capacity`` tokens a row."""

        _need(min(batch, kv_heads, capacity, head_dim) > 0, "8-bit cache dimensions must be positive")
        _need(str(layout).upper() in ("BHND", "BNHD"), "layout must be BHND or BNHD")
        capacity = -(-capacity // 8) * 8
        shape = (batch, kv_heads, capacity, head_dim) if str(layout).upper() == "BHND" else (batch, capacity, kv_heads, head_dim)
        key, value, scales = _empty_rows(shape, (batch, kv_heads, capacity, 2), dtype, device)
        return cls(key=key, value=value, scales=scales, layout=layout,
                   sequence_lengths=torch.zeros(batch, dtype=torch.int32, device=device))

    @property
    def normalized_layout(self) -> str:
        return str(self.layout).upper()

    @property
    def batch_size(self) -> int:
        return int(self.key.shape[0])

    @property
    def kv_heads(self) -> int:
        return int(self.key.shape[1 if self.normalized_layout == "BHND" else 2])

    @property
    def max_sequence_length(self) -> int:
        return int(self.key.shape[2 if self.normalized_layout == "BHND" else 1])

    @property
    def head_dim(self) -> int:
        return int(self.key.shape[3])

    def check(self) -> None:
        """Shapes, dtypes and strides (no device access)."""

        _check_codes(self.key, self.value, self.scales)
        _need(self.normalized_layout in ("BHND", "BNHD"), "layout must be BHND or BNHD")
        _need(tuple(self.scales.shape) == (self.batch_size, self.kv_heads, self.max_sequence_length, 2),
              "scales must be [batch, kv_heads, capacity, 2]")
        _need(self.scales.stride(3) == 1 and (self.scales.stride(2) == 2 or self.max_sequence_length == 1),
              "the (K, V) scale pairs of a head's tokens must be contiguous")
        _need(self.scales.stride(0) % 2 == 0 and self.scales.stride(1) % 2 == 0 and self.scales.storage_offset() % 2 == 0,
              "scale pairs must not straddle pairs")
        lens = self.sequence_lengths
        if lens is not None:
            _need(lens.dtype in native.SA_INDEX and tuple(lens.shape) == (self.batch_size,) and lens.is_contiguous(),
                  "sequence_lengths must be a contiguous [batch] int32/int64 tensor")

    def tensors(self) -> tuple:
        return self.key, self.value, self.scales, self.sequence_lengths

    def descriptor(self) -> "native.QuantCacheStruct":
        """The C ABI's view of the cache (call :meth:`check` first; the tensors must stay alive)."""

        at = (0, 2, 1) if self.normalized_layout == "BHND" else (0, 1, 2)
        sb, sn, sh = (int(self.key.stride(i)) for i in at)
        # Axes of one entry may carry any stride; none is ever taken along them.
        return native.QuantCacheStruct(
            key=self.key.data_ptr(), value=self.value.data_ptr(), scales=self.scales.data_ptr(),
            code=native.SA_KV_CODE[self.key.dtype], batch=self.batch_size, kv_heads=self.kv_heads,
            head_dim=self.head_dim, capacity=self.max_sequence_length,
            stride_b=sb if self.batch_size > 1 else 0, stride_n=sn if self.max_sequence_length > 1 else max(sn, 1),
            stride_h=sh if self.kv_heads > 1 else 0,
            scale_stride_b=int(self.scales.stride(0)) // 2 if self.batch_size > 1 else 0,
            scale_stride_h=int(self.scales.stride(1)) // 2 if self.kv_heads > 1 else 0, page_table=None)


@dataclass(frozen=True)
class QuantPagedKVCache:
    """Paged 8-bit cache: :class:`PagedKVCache` with codes for elements, plus ``scales``.

    NHD pages are ``[num_pages, page_size, Hkv, D]``, HND pages ``[num_pages, Hkv, page_size, D]``, the
    scales ``[num_pages, Hkv, page_size, 2]`` in both cases; ``page_table`` is
    ``[batch, max_pages_per_request]`` and ``sequence_lengths`` ``[batch]``, both int32/int64 and read on
    the device by every run.  All tensors are contiguous.
    """

    key: torch.Tensor
    value: torch.Tensor
    scales: torch.Tensor
    page_table: torch.Tensor
    sequence_lengths: torch.Tensor
    layout: str = "NHD"

    @classmethod
    def empty(cls, num_pages: int, page_size: int, kv_heads: int, head_dim: int, *, batch: int,
              max_pages_per_request: int, dtype: torch.dtype = torch.float8_e4m3fn, layout: str = "HND",
              device: Union[str, torch.device] = "cuda") -> "QuantPagedKVCache":
        """A pool of empty pages and ``batch`` empty requests (page table -1, lengths 0)."""

        _need(min(num_pages, page_size, kv_heads, head_dim, batch, max_pages_per_request) > 0,
              "8-bit cache dimensions must be positive")
        _need(str(layout).upper() in ("NHD", "HND"), "paged KV layout must be NHD or HND")
        shape = (num_pages, page_size, kv_heads, head_dim) if str(layout).upper() == "NHD" \
            else (num_pages, kv_heads, page_size, head_dim)
        key, value, scales = _empty_rows(shape, (num_pages, kv_heads, page_size, 2), dtype, device)
        return cls(key=key, value=value, scales=scales, layout=layout,
                   page_table=torch.full((batch, max_pages_per_request), -1, dtype=torch.int32, device=device),
                   sequence_lengths=torch.zeros(batch, dtype=torch.int32, device=device))

    @property
    def normalized_layout(self) -> str:
        return str(self.layout).upper()

    @property
    def num_pages(self) -> int:
        return int(self.key.shape[0])

    @property
    def page_size(self) -> int:
        return int(self.key.shape[1 if self.normalized_layout == "NHD" else 2])

    @property
    def kv_heads(self) -> int:
        return int(self.key.shape[2 if self.normalized_layout == "NHD" else 1])

    @property
    def head_dim(self) -> int:
        return int(self.key.shape[3])

    @property
    def batch_size(self) -> int:
        return int(self.page_table.shape[0])

    @property
    def max_pages_per_request(self) -> int:
        return int(self.page_table.shape[1])

    @property
    def max_sequence_length(self) -> int:
        return self.max_pages_per_request * self.page_size

    def check(self) -> None:
        """Shapes, dtypes and contiguity (no device access)."""

        _check_codes(self.key, self.value, self.scales)
        _need(self.normalized_layout in ("NHD", "HND"), "paged KV layout must be NHD or HND")
        _need(tuple(self.scales.shape) == (self.num_pages, self.kv_heads, self.page_size, 2),
              "scales must be [num_pages, kv_heads, page_size, 2]")
        _need(self.page_table.dim() == 2 and self.page_table.numel() > 0, "page_table must be [batch, max_pages_per_request]")
        _need(self.sequence_lengths.dim() == 1, "sequence_lengths must be [batch]")
        _need(self.sequence_lengths.numel() == self.batch_size, "sequence_lengths size must match batch")
        _need(self.page_table.dtype in native.SA_INDEX, "page_table must use int32 or int64")
        _need(self.sequence_lengths.dtype in native.SA_INDEX, "sequence_lengths must use int32 or int64")
        _need(all(t.is_contiguous() for t in self.tensors()), "paged cache tensors must be contiguous")

    def check_metadata(self) -> None:
        """Host-side check (synchronises) that lengths and active page ids are in range."""

        lengths = self.sequence_lengths.detach().to(device="cpu", dtype=torch.int64)
        _need(not bool((lengths < 0).any()), "sequence_lengths must not be negative")
        _need(not bool((lengths > self.max_sequence_length).any()), "sequence_lengths exceed page_table capacity")
        table = self.page_table.detach().to(device="cpu", dtype=torch.int64)
        active_pages = (lengths + self.page_size - 1) // self.page_size
        active = torch.arange(self.max_pages_per_request).unsqueeze(0) < active_pages.unsqueeze(1)
        _need(not bool((active & ((table < 0) | (table >= self.num_pages))).any()),
              "active page_table entries must reference physical pages")

    def tensors(self) -> tuple:
        return self.key, self.value, self.scales, self.page_table, self.sequence_lengths

    def descriptor(self) -> "native.QuantCacheStruct":
        """The C ABI's view of the cache (call :meth:`check` first; the tensors must stay alive)."""

        return native.QuantCacheStruct(
            key=self.key.data_ptr(), value=self.value.data_ptr(), scales=self.scales.data_ptr(),
            code=native.SA_KV_CODE[self.key.dtype], batch=self.batch_size, kv_heads=self.kv_heads,
            head_dim=self.head_dim, page_table=self.page_table.data_ptr(),
            table_dtype=native.SA_INDEX[self.page_table.dtype], page_size=self.page_size,
            max_pages=self.max_pages_per_request, num_pages=self.num_pages,
            layout=native.SA_LAYOUT[self.normalized_layout])


QuantCache = Union[QuantKVCache, QuantPagedKVCache]

__all__ = ["QuantKVCache", "QuantPagedKVCache", "QuantCache"]
