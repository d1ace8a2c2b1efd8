"""Quantized key/value cache of a decoder, and the attention that reads it.

No counterpart in the reference, whose path ends at the GEMMs.  The cache is
a pool of pages that sequences share; a page holds ``page_size`` tokens of
every key head as int8 or packed int4 codes with one bf16 scale per row of
``head_dim`` codes:

    scale = bf16(max|x| / Q)          Q = 7 (int4) or 127 (int8)
    code  = clamp(round(x / scale), -Q, Q)        value = code * scale

in 32 bits, rounding half to even.  A row of zeros has scale 0 and reads back
as zeros; a row that holds an infinity or a NaN reads back as NaN.

``kv_cache_write`` quantizes new tokens into their slots, ``kv_cache_read``
dequantizes slots, and ``kv_cache_attention`` is softmax attention of each
sequence's newest tokens over its pages, after a prefix that the whole batch
may share.  All run on the current stream of the tensors' device, or on
``stream`` (which is then the current one for the call, its allocations
included), and read nothing back to the host.  There is no CPU path and no
gradient: what is written into a cache is cut from its graph, and asking the
attention's outputs for a gradient raises.
"""

from __future__ import annotations

import math
import struct
from dataclasses import dataclass
from typing import Any

from . import kernel_table as kt
from .native import (
    _check,
    _current_stream,
    _no_gradient,
    _on_stream,
    _require_device,
    _torch,
    _verified_library,
)

HEAD_DIMS = (64, 128, 256)


# The structs of include/strix_halo_gfx950.h, field by field; every field is 8
# bytes (pointers and int64 alike, one double), so packing them is a tenth of
# the time that filling ctypes.Structure takes.
_CACHE = struct.Struct("=9q")
_ROWS = struct.Struct("=10q")
_ATTENTION = struct.Struct("=14qd4q")


@dataclass(frozen=True, eq=False)
class KVCache:
    """The tensors of one layer's cache; ``new_kv_cache`` makes them.

    ``key_codes`` and ``value_codes`` are ``[pages, kv_heads, page_size,
    head_dim]`` int8, or ``[..., head_dim / 2]`` uint8 with int4 pairs along
    head_dim (the even element in the low nibble, as ``pack_int4_k_major``
    packs); ``key_scales`` and ``value_scales`` are ``[pages, kv_heads,
    page_size]`` bf16.  head_dim is 64, 128 or 256, page_size a power of two
    from 16 to 1024.
    """

    key_codes: Any
    value_codes: Any
    key_scales: Any
    value_scales: Any

    def __post_init__(self) -> None:
        torch = _torch()
        codes = self.key_codes
        if codes.dtype not in (torch.uint8, torch.int8):
            raise ValueError(f"key_codes must be int8 codes or packed int4 torch.uint8; got {codes.dtype}")
        if codes.ndim != 4:
            raise ValueError("key_codes must have shape (pages, kv_heads, page_size, head_dim or head_dim/2); "
                             f"got {tuple(codes.shape)}")
        bits = 4 if codes.dtype == torch.uint8 else 8
        pages, heads, page_size, row = (int(n) for n in codes.shape)
        head_dim = row * 8 // bits
        for name, want_shape, want_dtype in (("value_codes", codes.shape, codes.dtype),
                                             ("key_scales", codes.shape[:3], torch.bfloat16),
                                             ("value_scales", codes.shape[:3], torch.bfloat16)):
            t = getattr(self, name)
            if tuple(t.shape) != tuple(want_shape) or t.dtype != want_dtype:
                raise ValueError(f"{name} must have shape {tuple(want_shape)} and dtype {want_dtype}; "
                                 f"got {tuple(t.shape)} and {t.dtype}")
        for name in ("key_codes", "value_codes", "key_scales", "value_scales"):
            t = getattr(self, name)
            if not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
            if t.device != codes.device:
                raise ValueError(f"{name} is on {t.device}, expected {codes.device}")
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}; got {head_dim}")
        if not 16 <= page_size <= 1024 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from 16 to 1024; got {page_size}")
        if not 1 <= heads <= 65535 or pages < 1:
            raise ValueError(f"the cache needs at least one page and 1 to 65535 heads; got {pages} and {heads}")
        where = (codes.data_ptr, self.value_codes.data_ptr, self.key_scales.data_ptr, self.value_scales.data_ptr)
        at = tuple(address() for address in where)
        packed = _CACHE.pack(*at, pages, heads, page_size, head_dim, bits)
        for name, value in (("pages", pages), ("kv_heads", heads), ("page_size", page_size), ("head_dim", head_dim),
                            ("bits", bits), ("device", codes.device), ("_packed", (where, at, packed)),
                            ("_workspaces", {})):
            object.__setattr__(self, name, value)

    def __reduce__(self) -> Any:
        # copies and loaded caches are made of their own tensors
        return KVCache, (self.key_codes, self.value_codes, self.key_scales, self.value_scales)

    @property
    def _native(self) -> bytes:
        """shk_kv_cache, at the addresses that the tensors have now."""
        (kc, vc, ks, vs), at, packed = self._packed
        if (kc(), vc(), ks(), vs()) == at:
            return packed
        self.__post_init__()  # a tensor was given other memory: all checks again
        return self._packed[2]


def new_kv_cache(pages: int, page_size: int, kv_heads: int, head_dim: int, *, bits: int = 4,
                 device: Any = "cuda") -> KVCache:
    """A zero-filled cache of ``pages`` pages (every row reads back as zeros)."""
    torch = _torch()
    if bits not in (4, 8):
        raise ValueError("bits must be 4 or 8")
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS}; got {head_dim}")
    shape = (pages, kv_heads, page_size)
    dtype = torch.uint8 if bits == 4 else torch.int8
    codes = [torch.zeros((*shape, head_dim * bits // 8), dtype=dtype, device=device) for _ in range(2)]
    scales = [torch.zeros(shape, dtype=torch.bfloat16, device=device) for _ in range(2)]
    return KVCache(*codes, *scales)


def _row_type(torch: Any, name: str, dtype: Any) -> int:
    if dtype == torch.bfloat16:
        return kt.SRC_BF16
    if dtype == torch.float16:
        return kt.SRC_F16
    if dtype == torch.float32:
        return kt.SRC_F32
    raise ValueError(f"{name} must have dtype torch.bfloat16, torch.float16 or torch.float32; got {dtype}")


def _check_slots(torch: Any, slots: Any, tokens: int | None) -> None:
    if slots.dtype != torch.int64 and slots.dtype != torch.int32:
        raise ValueError(f"slots must have dtype torch.int64 or torch.int32; got {slots.dtype}")
    if slots.ndim != 1 or (tokens is not None and slots.shape[0] != tokens):
        want = "(tokens,)" if tokens is None else f"({tokens},)"
        raise ValueError(f"slots must have shape {want}; got {tuple(slots.shape)}")
    if not slots.is_contiguous():
        raise ValueError("slots must be contiguous")


def _rows(keys: Any, values: Any, slots: Any, kind: int, tokens: int) -> bytes:
    ks, vs = keys.stride(), values.stride()
    return _ROWS.pack(keys.data_ptr(), values.data_ptr(), ks[0], ks[1], vs[0], vs[1], kind, slots.data_ptr(),
                      slots.element_size(), tokens)


def _check_devices(cache: KVCache, **tensors: Any) -> None:
    index = cache.key_codes.get_device()
    for t in tensors.values():
        if t is not None and t.get_device() != index:
            break
    else:
        if index >= 0:
            return
    _require_device(_torch(), {"cache": cache.key_codes, **tensors})  # says what is wrong


def kv_cache_write(cache: KVCache, keys: Any, values: Any, slots: Any, *, stream: Any | None = None) -> None:
    """Quantizes ``keys`` and ``values`` [tokens, kv_heads, head_dim] (bf16,
    f16 or f32; head_dim contiguous, other strides free) into the cache.

    Token t goes to ``slots[t] = page * page_size + position`` (int64 or
    int32).  Slots outside the cache, such as -1 for padding, are skipped; the
    others are distinct.  One pass over memory, no copy of the inputs.
    """
    torch = _torch()
    native = cache._native  # first: the sizes that follow are the tensors' own
    _check_devices(cache, keys=keys, values=values, slots=slots)
    if stream is not None:
        with _on_stream(torch, keys, stream):
            return kv_cache_write(cache, keys, values, slots)
    kind = _row_type(torch, "keys", keys.dtype)
    if values.dtype != keys.dtype:
        raise ValueError(f"values must have the dtype of keys, {keys.dtype}; got {values.dtype}")
    tokens = int(keys.shape[0]) if keys.ndim else 0
    shape = (tokens, cache.kv_heads, cache.head_dim)
    for name, t in (("keys", keys), ("values", values)):
        if t.shape != shape:
            raise ValueError(f"{name} must have shape {shape} == (tokens, kv_heads, head_dim); got {tuple(t.shape)}")
        if t.stride(2) != 1:
            raise ValueError(f"{name} must be contiguous along head_dim")
    _check_slots(torch, slots, tokens)
    if tokens == 0:
        return
    lib = _verified_library()
    index = keys.get_device()
    _check(lib, lib.amd_strix_halo_kernels_kv_write(index, _current_stream(torch, index), native,
                                                    _rows(keys, values, slots, kind, tokens)))


def kv_cache_read(cache: KVCache, slots: Any, *, dtype: Any = None, stream: Any | None = None) -> tuple[Any, Any]:
    """The keys and values of ``slots`` [tokens], dequantized to ``dtype``
    (bf16, the default, f16 or f32): two [tokens, kv_heads, head_dim]
    tensors.  Slots outside the cache give NaN."""
    torch = _torch()
    native = cache._native  # first: the sizes that follow are the tensors' own
    _check_devices(cache, slots=slots)
    if stream is not None:
        with _on_stream(torch, slots, stream):
            return kv_cache_read(cache, slots, dtype=dtype)
    dtype = torch.bfloat16 if dtype is None else dtype
    kind = _row_type(torch, "the result", dtype)
    _check_slots(torch, slots, None)
    tokens = int(slots.shape[0])
    shape = (tokens, cache.kv_heads, cache.head_dim)
    keys = torch.empty(shape, dtype=dtype, device=cache.device)
    values = torch.empty_like(keys)
    if tokens:
        lib = _verified_library()
        index = keys.get_device()
        _check(lib, lib.amd_strix_halo_kernels_kv_read(index, _current_stream(torch, index), native,
                                                       _rows(keys, values, slots, kind, tokens)))
    return keys, values


def kv_cache_attention(
    q: Any,
    cache: KVCache,
    page_table: Any,
    lengths: Any,
    *,
    prefix_pages: Any | None = None,
    prefix_length: int = 0,
    softmax_scale: float | None = None,
    return_lse: bool = False,
    out: Any | None = None,
    stream: Any | None = None,
) -> Any:
    """Softmax attention of each sequence's newest tokens over its cached ones.

    ``q`` is [batch, heads, head_dim] (one new token a sequence) or [batch,
    queries, heads, head_dim], bf16 or f16, head_dim contiguous; heads is a
    multiple of the cache's kv_heads, and query head h reads key head
    ``h // (heads // kv_heads)``.  Sequence b holds ``lengths[b]`` tokens
    (int32), the ``queries`` newest among them, in the pages
    ``page_table[b]`` (int32 [batch, pages]); query t sees the first
    ``lengths[b] - queries + t + 1``.

    ``prefix_pages`` (int32 [pages]) and ``prefix_length`` name tokens that
    come before every sequence's own, stored once and read once for the whole
    batch; every query sees all of them.

    Returns ``softmax(softmax_scale * q k^T) v`` in q's shape and dtype
    (softmax_scale defaults to 1 / sqrt(head_dim)), and with ``return_lse``
    also the natural logarithm of each row's sum of exponentials (f32, q's
    shape without head_dim).  A query that sees nothing gives 0 and -inf, and
    what it does not see may hold anything.  A length past the table counts as
    the whole table, a negative one as 0; a page outside the cache makes its
    sequence's outputs NaN.  Scores, the softmax and the sums are f32; products
    take the codes as they are.
    """
    torch = _torch()
    native = cache._native  # first: the sizes that follow are the tensors' own
    _check_devices(cache, q=q, page_table=page_table, lengths=lengths, prefix_pages=prefix_pages, out=out)
    if stream is not None:
        with _on_stream(torch, q, stream):
            return kv_cache_attention(q, cache, page_table, lengths, prefix_pages=prefix_pages,
                                      prefix_length=prefix_length, softmax_scale=softmax_scale,
                                      return_lse=return_lse, out=out)
    if q.dtype != torch.bfloat16 and q.dtype != torch.float16:
        raise ValueError(f"q must have dtype torch.bfloat16 or torch.float16; got {q.dtype}")
    if q.ndim not in (3, 4) or q.shape[-1] != cache.head_dim:
        raise ValueError(f"q must have shape (batch, heads, {cache.head_dim}) or (batch, queries, heads, "
                         f"{cache.head_dim}); got {tuple(q.shape)}")
    given, shape = q, q.shape
    batch, heads = int(shape[0]), int(shape[-2])
    queries = int(shape[1]) if q.ndim == 4 else 1
    if heads == 0 or heads % cache.kv_heads:
        raise ValueError(f"q's heads must be a multiple of the cache's {cache.kv_heads}; got {heads}")
    if q.stride(-1) != 1:
        raise ValueError("q must be contiguous along head_dim")
    if page_table.dtype != torch.int32 or lengths.dtype != torch.int32:
        raise ValueError(f"page_table and lengths must have dtype torch.int32; got {page_table.dtype} and "
                         f"{lengths.dtype}")
    if page_table.ndim != 2 or page_table.shape[0] != batch:
        raise ValueError(f"page_table must have shape ({batch}, pages); got {tuple(page_table.shape)}")
    if page_table.stride(1) != 1 and page_table.shape[1] > 1:
        raise ValueError("rows of page_table must be contiguous")
    if lengths.shape != (batch,) or not lengths.is_contiguous():
        raise ValueError(f"lengths must be contiguous with shape ({batch},); got {tuple(lengths.shape)}")
    if isinstance(prefix_length, bool) or not isinstance(prefix_length, int) or prefix_length < 0:
        raise ValueError(f"prefix_length must be a non-negative int; got {prefix_length!r}")
    if prefix_length:
        if prefix_pages is None:
            raise ValueError("prefix_length needs prefix_pages")
        if prefix_pages.dtype != torch.int32 or prefix_pages.ndim != 1 or not prefix_pages.is_contiguous():
            raise ValueError("prefix_pages must be a contiguous one-dimensional torch.int32 tensor; got "
                             f"{prefix_pages.dtype} {tuple(prefix_pages.shape)}")
        if prefix_pages.shape[0] * cache.page_size < prefix_length:
            raise ValueError(f"prefix_pages holds {prefix_pages.shape[0] * cache.page_size} tokens; prefix_length is "
                             f"{prefix_length}")
    scale = 1.0 / math.sqrt(cache.head_dim) if softmax_scale is None else float(softmax_scale)
    if not abs(scale) < 2.0**128 - 2.0**103:  # what rounds to a finite f32
        raise ValueError(f"softmax_scale must be finite in 32 bits; got {softmax_scale}")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != shape or out.dtype != q.dtype or not out.is_contiguous():
        raise ValueError(f"out must be contiguous with shape {tuple(shape)} and dtype {q.dtype}; got "
                         f"{tuple(out.shape)} and {out.dtype}")
    lse = q.new_empty(shape[:-1], dtype=torch.float32) if return_lse else None
    if batch * queries:
        strides = q.stride()
        sb, sq, sh = (strides[0], strides[1], strides[2]) if q.ndim == 4 else (strides[0], 0, strides[1])
        if q.data_ptr() % 16 or sb % 8 or sq % 8 or sh % 8:
            # 16-byte reads: rows that do not start on 16 bytes are copied
            q = q.clone(memory_format=torch.contiguous_format)
            sb, sq, sh = queries * heads * cache.head_dim, heads * cache.head_dim, cache.head_dim
        kind = kt.SRC_BF16 if q.dtype == torch.bfloat16 else kt.SRC_F16
        table_pages = page_table.shape[1]

        def args(work: Any, nbytes: int) -> bytes:
            return _ATTENTION.pack(q.data_ptr(), sb, sq, sh, kind, batch, queries, heads, page_table.data_ptr(),
                                   page_table.stride(0), table_pages, lengths.data_ptr(),
                                   prefix_pages.data_ptr() if prefix_length else 0, prefix_length, scale,
                                   out.data_ptr(), lse.data_ptr() if return_lse else 0,
                                   work.data_ptr() if nbytes else 0, nbytes)

        lib = _verified_library()
        # the workspace's size is a function of the sizes alone
        key = (batch, queries, heads, table_pages, prefix_length)
        nbytes = cache._workspaces.get(key)
        if nbytes is None:
            nbytes = lib.amd_strix_halo_kernels_kv_attention_workspace(native, args(None, 0))
            if nbytes < 0:
                _check(lib, 1)
            if len(cache._workspaces) < 4096:
                cache._workspaces[key] = nbytes
        work = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        index = q.get_device()
        _check(lib, lib.amd_strix_halo_kernels_kv_attention(index, _current_stream(torch, index), native,
                                                            args(work, nbytes)))
    if given.requires_grad:
        out = _no_gradient(torch, "kv_cache_attention", out, given)
        lse = _no_gradient(torch, "kv_cache_attention", lse, given) if return_lse else None
    return (out, lse) if return_lse else out
