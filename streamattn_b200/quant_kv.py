"""Writing, reading back and attending to 8-bit KV caches (:mod:`streamattn_b200.quant_cache`).

* :func:`quantize_kv` / :class:`QuantizeKVPlan` - the cache update before each decode (one token a
  row) or of a prompt chunk (any number, different for each row): rotates K, quantises K and V into a
  contiguous or paged cache, advances the lengths, rotates the query beside it;
* :func:`dequantize_kv` / :class:`DequantizeKVPlan` - any range of the rows' tokens back as K and V;
* :func:`stream_attn_quant_decode` / :class:`QuantDecodePlan` - exact one-token attention over the
  values the cache holds.

Positions, lengths, counts and page tables are read on the device when a plan runs; nothing here
synchronises, so update and decode can be captured in one CUDA graph.  The reference has no
quantised cache; its 16-bit counterparts are cited in ``kv_update``, ``exact`` and ``paged``.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass, field
from typing import Any, Optional, Tuple

import torch

from . import native
from .kv_update import AppendKVPlan, _heads_axis, _positions
from .quant_cache import QuantCache, QuantKVCache, QuantPagedKVCache

QUANT_EXACT_SM100_BACKEND = "streamattn_quant_sm100_exact"
QUANT_EXACT_NATIVE_BACKEND = "streamattn_quant_exact_native"


def _cache(cache: QuantCache) -> QuantCache:
    if not isinstance(cache, (QuantKVCache, QuantPagedKVCache)):
        raise ValueError("cache must be a QuantKVCache or a QuantPagedKVCache")
    cache.check()
    return cache


def _token_rows(t: torch.Tensor, layout: str, name: str) -> Tuple[tuple, tuple]:
    """((batch, tokens, heads, dim), (stride_b, stride_t, stride_h)) of [B,T,H,D] or [B,H,T,D]."""

    heads = _heads_axis(layout)
    if t.dim() != 4 or min(t.shape) < 1 or (t.stride(3) != 1 and int(t.shape[3]) > 1):
        raise ValueError(f"{name} must be a non-empty 4-D tensor with a contiguous last dimension")
    axes = (0, 3 - heads, heads)
    # A stride along an axis of one entry is never taken: 0 keeps it out of the alignment rules.
    strides = tuple(int(t.stride(i)) if int(t.shape[i]) > 1 else 0 for i in axes)
    return (*(int(t.shape[i]) for i in axes), int(t.shape[3])), strides


def _optional_counts(t: Optional[torch.Tensor], batch: int, name: str) -> int:
    if t is None:
        return 0
    if t.dtype not in native.SA_INDEX or tuple(t.shape) != (batch,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous [batch] int32/int64 tensor")
    return native.SA_INDEX[t.dtype]


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two contiguous tensors share memory.  Of others (slices of one buffer may interleave) only their start is compared."""

    if not (a.is_contiguous() and b.is_contiguous()):
        return a.data_ptr() == b.data_ptr()
    return a.device == b.device and a.data_ptr() < b.data_ptr() + b.numel() * b.element_size() \
        and b.data_ptr() < a.data_ptr() + a.numel() * a.element_size()


def _folded(t: torch.Tensor) -> bool:
    """Whether entries along an axis are the same memory (an expanded tensor)."""

    return any(stride == 0 and size > 1 for stride, size in zip(t.stride(), t.shape))


def _angles(cos, sin, batch: int, tokens: int, dim: int, dtype: torch.dtype):
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin must be given together")
    if cos is None:
        return None, None, (0, 0)
    for t, name in ((cos, "cos"), (sin, "sin")):
        if t.dtype != dtype:
            raise ValueError(f"{name} must have the dtype of the new rows")
        if t.dim() != 3 and not (t.dim() == 2 and tokens == 1):
            raise ValueError(f"{name} must be [batch_or_1, tokens, dim]")
    cos, sin = (t.unsqueeze(1) if t.dim() == 2 else t for t in (cos, sin))
    for t, name in ((cos, "cos"), (sin, "sin")):
        if int(t.shape[0]) not in (1, batch) or tuple(t.shape[1:]) != (tokens, dim) or (t.stride(2) != 1 and dim > 1):
            raise ValueError(f"{name} must be [batch_or_1, tokens, dim] with a contiguous last dimension")
    if cos.shape != sin.shape or cos.stride() != sin.stride():
        raise ValueError("cos and sin must share shape and strides")
    return cos, sin, (0 if int(cos.shape[0]) == 1 else int(cos.stride(0)), int(cos.stride(1)) if tokens > 1 else 0)


class QuantizeKVPlan(AppendKVPlan):
    """A validated, bound update of an 8-bit cache: ``run()`` is one native call.

    Bound by address like :class:`AppendKVPlan`: refill the new rows, the query, ``cos``/``sin`` and
    ``counts`` in place between runs.
    """

    @classmethod
    def build(cls, cache: QuantCache, key_new: torch.Tensor, value_new: torch.Tensor, *,
              positions: Optional[torch.Tensor] = None, counts: Optional[torch.Tensor] = None,
              new_layout: str = "BNHD", cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None,
              query: Optional[torch.Tensor] = None, query_out: Optional[torch.Tensor] = None,
              query_layout: str = "BNHD", lengths_out: Optional[torch.Tensor] = None,
              advance_lengths: Optional[bool] = None, status: Optional[torch.Tensor] = None) -> "QuantizeKVPlan":
        """Arguments as :func:`quantize_kv`."""

        _cache(cache)
        lens = cache.sequence_lengths
        if positions is None:
            if lens is None:
                raise ValueError("positions are required for a cache without sequence_lengths")
            positions = lens
            advance_lengths = True if advance_lengths is None else advance_lengths
        if advance_lengths:
            if lens is None:
                raise ValueError("advance_lengths needs a cache with sequence_lengths")
            if lengths_out is not None and lengths_out is not lens:
                raise ValueError("lengths_out and advance_lengths exclude each other")
            lengths_out = lens
        dtype = key_new.dtype
        if dtype not in native.SA_DTYPE or value_new.dtype != dtype:
            raise ValueError("key_new and value_new must share a dtype of bf16, fp16 or fp32")
        (batch, tokens, heads, dim), strides = _token_rows(key_new, new_layout, "key_new")
        if value_new.shape != key_new.shape or _token_rows(value_new, new_layout, "value_new")[1] != strides:
            raise ValueError("key_new and value_new must have identical shape and strides")
        if (batch, heads, dim) != (cache.batch_size, cache.kv_heads, cache.head_dim):
            raise ValueError("key_new / value_new must have the cache's batch, KV heads and head_dim")
        if lengths_out is not None and lengths_out.dtype != positions.dtype:
            raise ValueError("positions must have the dtype of the lengths that are written")
        pos_dtype, num_positions = _positions(positions, batch, lengths_out)
        counts_dtype = _optional_counts(counts, batch, "counts")
        if any(_folded(t) for t in (cache.key, cache.value, cache.scales)) or _overlap(cache.key, cache.value):
            raise ValueError("the rows of a cache that is written must not share memory")
        if lengths_out is not None and counts is not None and _overlap(lengths_out, counts):
            raise ValueError("counts must not alias the lengths that are written")
        if lengths_out is not None and lengths_out.data_ptr() != positions.data_ptr() and _overlap(lengths_out, positions):
            raise ValueError("the lengths that are written may be the positions, but not a part of them")
        cos, sin, rope_strides = _angles(cos, sin, batch, tokens, dim, dtype)
        q_heads, qi, qo = 0, (0, 0, 0), (0, 0, 0)
        if query is None and query_out is not None:
            raise ValueError("query_out needs query")
        if query is not None:
            if query_out is None:
                query_out = torch.empty_like(query)
            shape, qi = _token_rows(query, query_layout, "query")
            out_shape, qo = _token_rows(query_out, query_layout, "query_out")
            if out_shape != shape or (shape[0], shape[1], shape[3]) != (batch, tokens, dim) \
                    or query.dtype != dtype or query_out.dtype != dtype:
                raise ValueError("query / query_out must match the new rows in batch, tokens, head_dim and dtype")
            if _overlap(query_out, query):
                raise ValueError("query_out must not alias query")
            if any(_overlap(query_out, t) for t in (key_new, value_new)):
                raise ValueError("query_out must not alias the new rows")
            if _folded(query_out):
                raise ValueError("the rows of query_out must not share memory")
            q_heads = shape[2]
        if status is not None and (status.dtype != torch.int32 or status.numel() < 1):
            raise ValueError("status must be an int32 tensor")
        device = native.require_cuda(*cache.tensors(), key_new, value_new, positions, counts, cos, sin, query, query_out,
                                     lengths_out, status)
        desc = cache.descriptor()
        ptr = native._ptr
        args = (ctypes.byref(desc), ptr(key_new), ptr(value_new), tokens, *strides, ptr(positions), pos_dtype, num_positions,
                ptr(counts), counts_dtype, ptr(lengths_out), ptr(cos), ptr(sin), *rope_strides,
                ptr(query), ptr(query_out), q_heads, *qi, *qo, native.SA_DTYPE[dtype], ptr(status))
        keep = (desc, cache, key_new, value_new, positions, counts, lengths_out, cos, sin, query, query_out, status)
        return cls("sa_quantize_kv", args, device, keep, query_out)

    @classmethod
    def build_paged(cls, cache: QuantPagedKVCache, key_new: torch.Tensor, value_new: torch.Tensor,
                    **kwargs) -> "QuantizeKVPlan":
        """Same as :meth:`build`, which takes both kinds of cache."""

        return cls.build(cache, key_new, value_new, **kwargs)


def quantize_kv(cache: QuantCache, key_new: torch.Tensor, value_new: torch.Tensor, **kwargs) -> Optional[torch.Tensor]:
    """Quantise new K/V rows into an 8-bit cache (one launch for a decode step, no host sync).

    ``key_new``/``value_new`` hold the same number of tokens for every row, ``[B, T, Hkv, D]``
    (``new_layout="BNHD"``, default) or ``[B, Hkv, T, D]``, in bf16, fp16 or fp32; with ``counts``
    (device ``[B]``, clipped to ``[0, T]``) only the first ``counts[b]`` of them are real and the rest is
    padding that is neither read nor written.  They go to token indices ``positions[b]`` and up;
    ``positions`` is a device int32/int64 tensor, one entry or one per row, by default
    ``cache.sequence_lengths``, which is then advanced in place (``advance_lengths=False`` leaves it;
    with explicit ``positions``, ``advance_lengths=True`` or ``lengths_out`` writes ``positions + counts``).

    With ``cos``/``sin`` (``[B or 1, T, D]`` in the rows' dtype; ``[B or 1, D]`` for one token) K is rotated,
    ``x * cos + rotate_half(x) * sin`` in fp32, and quantised without being rounded in between.  ``query``
    (``[B, T, Hq, D]``, or ``query_layout="BHND"``) is rotated likewise, rounded once, into ``query_out``,
    which is returned; without ``cos``/``sin`` it is copied.  All ``T`` tokens of it are, whatever ``counts``
    says, so that no row of ``query_out`` is left undefined.

    ``status`` (device int32) collects ``SA_DEV_BAD_POSITION`` for rows whose tokens do not fit the
    cache - such a row is left out as a whole - and ``SA_DEV_BAD_PAGE`` for tokens whose page is not
    assigned; in both cases the row's length does not advance.  Two rows must not share the pages
    they write.
    """

    return QuantizeKVPlan.build(cache, key_new, value_new, **kwargs).run()


class DequantizeKVPlan:
    """A validated, bound read-back of an 8-bit cache: ``run()`` is one native call."""

    def __init__(self, args: tuple, device: torch.device, keep: tuple, outputs: tuple) -> None:
        self._plan = AppendKVPlan("sa_dequantize_kv", args, device, keep, outputs)

    def run(self) -> Tuple[torch.Tensor, torch.Tensor]:
        return self._plan.run()

    @classmethod
    def build(cls, cache: QuantCache, key_out: torch.Tensor, value_out: torch.Tensor, *,
              starts: Optional[torch.Tensor] = None, counts: Optional[torch.Tensor] = None,
              out_layout: str = "BNHD", status: Optional[torch.Tensor] = None) -> "DequantizeKVPlan":
        """Tokens ``[starts[b], starts[b] + counts[b])`` of every row into ``key_out`` / ``value_out``.

        ``key_out``/``value_out`` are ``[B, T, Hkv, D]`` (``out_layout="BNHD"``) or ``[B, Hkv, T, D]`` in bf16,
        fp16 or fp32; rows behind ``counts[b]`` are left as they were.  ``starts`` (device ``[B]``) defaults
        to 0 and ``counts`` to ``T``; both are read when the plan runs.  A token outside the cache or
        with a bad page id is left out and reported through ``status`` (device int32).
        """

        _cache(cache)
        dtype = key_out.dtype
        if dtype not in native.SA_DTYPE or value_out.dtype != dtype:
            raise ValueError("key_out and value_out must share a dtype of bf16, fp16 or fp32")
        (batch, tokens, heads, dim), strides = _token_rows(key_out, out_layout, "key_out")
        if value_out.shape != key_out.shape or _token_rows(value_out, out_layout, "value_out")[1] != strides:
            raise ValueError("key_out and value_out must have identical shape and strides")
        if (batch, heads, dim) != (cache.batch_size, cache.kv_heads, cache.head_dim):
            raise ValueError("key_out / value_out must have the cache's batch, KV heads and head_dim")
        starts_dtype = _optional_counts(starts, batch, "starts")
        counts_dtype = _optional_counts(counts, batch, "counts")
        if status is not None and (status.dtype != torch.int32 or status.numel() < 1):
            raise ValueError("status must be an int32 tensor")
        if _folded(key_out) or _overlap(key_out, value_out):
            raise ValueError("the rows of key_out and value_out must not share memory")
        device = native.require_cuda(*cache.tensors(), key_out, value_out, starts, counts, status)
        desc = cache.descriptor()
        ptr = native._ptr
        args = (ctypes.byref(desc), ptr(key_out), ptr(value_out), tokens, *strides, ptr(starts), starts_dtype,
                ptr(counts), counts_dtype, native.SA_DTYPE[dtype], ptr(status))
        keep = (desc, cache, key_out, value_out, starts, counts, status)
        return cls(args, device, keep, (key_out, value_out))


def dequantize_kv(cache: QuantCache, *, tokens: Optional[int] = None, dtype: torch.dtype = torch.bfloat16,
                  starts: Optional[torch.Tensor] = None, counts: Optional[torch.Tensor] = None,
                  out_layout: str = "BNHD", status: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Read rows of an 8-bit cache back as ``(key, value)``, ``[B, T, Hkv, D]`` (or ``out_layout="BHND"``).

    By default every row's tokens from 0 up to its length, padded with zeros to ``tokens`` (default:
    the capacity of a row); ``starts``/``counts`` select another range (see
    :meth:`DequantizeKVPlan.build`).
    """

    _cache(cache)
    tokens = cache.max_sequence_length if tokens is None else int(tokens)
    if tokens <= 0:
        raise ValueError("tokens must be positive")
    if starts is None and counts is None:
        counts = cache.sequence_lengths
    shape = (cache.batch_size, tokens, cache.kv_heads, cache.head_dim) if _heads_axis(out_layout) == 2 \
        else (cache.batch_size, cache.kv_heads, tokens, cache.head_dim)
    native.require_cuda(*cache.tensors())
    key = torch.zeros(shape, dtype=dtype, device=cache.key.device)
    return DequantizeKVPlan.build(cache, key, torch.zeros_like(key), starts=starts, counts=counts,
                                  out_layout=out_layout, status=status).run()


@dataclass
class QuantDecodePlan:
    """Allocation-free exact decode bound to an 8-bit cache (contiguous or paged)."""

    query: torch.Tensor
    cache: QuantCache
    output: torch.Tensor
    workspace: torch.Tensor
    splits: int
    backend: str
    trace: Optional[torch.Tensor] = None
    _plan: Any = field(default=None, repr=False)

    @classmethod
    def build(cls, query: torch.Tensor, cache: QuantCache, *, output: Optional[torch.Tensor] = None,
              splits: Optional[int] = None, validate_metadata: bool = True, record_page_walk: bool = False,
              return_state: bool = False, kernel: str = "auto",
              row_indices: Optional[torch.Tensor] = None) -> "QuantDecodePlan":
        """Validate once and bind a plan.

        ``query`` is ``[B, 1, Hq, D]`` in bf16, fp16 or fp32, the output has its shape and dtype; both
        may be pinned host tensors.  ``return_state`` asks for the unnormalised state instead, fp32
        ``[B, Hq, D + 2]`` (what ``sa_merge_states`` joins).  ``splits``, ``kernel``, ``record_page_walk`` (paged caches) and ``row_indices`` as in :class:`PagedExactDecodePlan` and
        :class:`ExactDecodePlan`; ``validate_metadata`` checks a paged cache's lengths and page ids
        on the host, once.  Rows of no tokens give zeros.

        Scores, probabilities and sums are fp32 on both kernels and the query is used as it is; the
        tensor-core kernel rounds a probability times its token's V scale to fp16 before it meets the
        codes (2^-11 of the product, or 2^-31 of the head's largest).
        """

        _cache(cache)
        paged = isinstance(cache, QuantPagedKVCache)
        if query.dim() != 4 or query.shape[1] != 1:
            raise ValueError("decode query must be [batch, 1, heads, dim]")
        if query.dtype not in native.SA_DTYPE:
            raise ValueError("query must be bf16, fp16 or fp32")
        batch, _, q_heads, dim = (int(x) for x in query.shape)
        if (batch, dim) != (cache.batch_size, cache.head_dim):
            raise ValueError("query/KV batch and head_dim must match")
        if q_heads < 1 or q_heads % cache.kv_heads:
            raise ValueError("query heads must be a multiple of KV heads")
        if record_page_walk and not paged:
            raise ValueError("record_page_walk needs a paged cache")
        if splits is not None and int(splits) <= 0:
            raise ValueError("splits must be positive")
        device = native.require_cuda(*cache.tensors(), host_io=(query, output))
        if paged and validate_metadata:
            cache.check_metadata()
        if output is None:
            output = torch.empty((batch, q_heads, dim + 2), dtype=torch.float32, device=device) if return_state \
                else torch.empty(query.shape, dtype=query.dtype, device=device)
        native._check_output(output, query, return_state)
        q_sb, q_sh = native._q_strides(query)
        num_ctas = 0 if splits is None else int(splits) * batch * cache.kv_heads
        workspace = native.new_workspace(device, batch, q_heads, cache.kv_heads, dim, num_ctas)
        trace = torch.full_like(cache.page_table, -1, dtype=torch.int32) if record_page_walk else None
        lens = cache.sequence_lengths
        desc = cache.descriptor()
        with torch.cuda.device(device):
            handle = native.load().sa_quant_plan_create(
                native._ptr(query), ctypes.byref(desc), native._ptr(output), native._ptr(workspace), workspace.numel(),
                native._ptr(lens), native.SA_INDEX[lens.dtype] if lens is not None else 0, native._ptr(trace),
                q_heads, q_sb, q_sh, native.SA_DTYPE[query.dtype],
                native.SA_OUT_STATE if return_state else native.SA_OUT_FINAL, num_ctas,
                native._kernel_code(kernel, False))
        plan = native.NativePlan(handle, device, (query, cache, output, workspace, trace))
        if row_indices is not None:
            plan.set_rows(row_indices)
        stream = plan.kernel == native.SA_KERNEL_STREAM
        return cls(query=query, cache=cache, output=output, workspace=workspace,
                   splits=max(1, -(-plan.num_ctas // (batch * cache.kv_heads))),
                   backend=QUANT_EXACT_SM100_BACKEND if stream else QUANT_EXACT_NATIVE_BACKEND, trace=trace, _plan=plan)

    @property
    def workspace_bytes(self) -> int:
        return self.workspace.numel()

    @property
    def kernel_name(self) -> str:
        return self._plan.kernel_name

    @property
    def num_ctas(self) -> int:
        return self._plan.num_ctas

    @property
    def launches_per_run(self) -> int:
        return self._plan.launches

    def run(self) -> torch.Tensor:
        """Execute on the bound buffers; cache contents, page table and lengths are read on the device."""

        self._plan.run()
        return self.output

    def set_row_indices(self, row_indices: Optional[torch.Tensor]) -> None:
        """Compute only the listed batch rows from now on (``None``: every row again)."""

        self._plan.set_rows(row_indices)

    def device_status(self) -> int:
        """Synchronise and return the kernels' status bits (0 = clean)."""

        return native.workspace_status(self.workspace)


def stream_attn_quant_decode(query: torch.Tensor, cache: QuantCache, *, output: Optional[torch.Tensor] = None,
                             splits: Optional[int] = None) -> torch.Tensor:
    """Plan and execute one exact decode call over an 8-bit cache."""

    return QuantDecodePlan.build(query, cache, output=output, splits=splits).run()


__all__ = ["QuantizeKVPlan", "quantize_kv", "DequantizeKVPlan", "dequantize_kv", "QuantDecodePlan",
           "stream_attn_quant_decode", "QUANT_EXACT_SM100_BACKEND", "QUANT_EXACT_NATIVE_BACKEND"]
