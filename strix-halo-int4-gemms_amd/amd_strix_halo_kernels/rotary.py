"""Norm and rotation of query and key heads, on their way into the cache.

No counterpart in the reference.  ``rotary_frequencies`` gives how fast each
pair of a head turns with the position, plain or for a context longer than the
trained one; ``new_rotary`` puts that on a device, and ``rotate_qk`` norms and
turns the heads of new tokens in one pass, the keys, with their values, straight
into a quantized cache if there is one.  Angles are formed and reduced in 64
bits: off by at most 2^-52 of the whole angle, which up to 10^8 radians is less
than 32 bits lose of what is left of it.  There is no CPU path, and asking a result
for a gradient raises.
"""

from __future__ import annotations

import math
import struct
from dataclasses import dataclass
from typing import Any, Sequence

from .kv_cache import KVCache, _check_slots, _row_type
from .native import (
    _check,
    _current_stream,
    _no_gradient,
    _on_stream,
    _require_device,
    _torch,
    _verified_library,
)

ROTARY_SCALINGS = ("none", "linear", "ntk", "yarn")

# shk_rotate of include/strix_halo_gfx950.h: every field is 8 bytes
_ROTATE = struct.Struct("=16qd3qd11q")


def rotary_frequencies(rotated: int, *, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                       trained: int = 0, fast: float = 32.0, slow: float = 1.0) -> tuple[list[float], float]:
    """``(frequencies, amplitude)`` of the ``rotated / 2`` pairs of a head:
    radians a position, and what cosines and sines are multiplied by.

    * ``none``: pair i turns by ``base ** (-2 i / rotated)``;
    * ``linear``: positions are divided by ``factor``;
    * ``ntk``: the base grows by ``factor ** (rotated / (rotated - 2))``, which
      slows the slowest pair by ``factor`` and the fastest not at all;
    * ``yarn``: pairs that turn more than ``fast`` times over the ``trained``
      positions stay, those that turn less than ``slow`` times are slowed by
      ``factor``, those between in proportion to their index (both ends in whole
      pairs, the second at most ``rotated - 1``); the amplitude is ``0.1
      ln(factor) + 1``, 1 for factors below 1.
    """
    if isinstance(rotated, bool) or not isinstance(rotated, int) or rotated < 2 or rotated % 2:
        raise ValueError(f"rotated must be a positive even int; got {rotated!r}")
    if scaling not in ROTARY_SCALINGS:
        raise ValueError(f"scaling must be one of {ROTARY_SCALINGS}; got {scaling!r}")
    if not base > 1.0 or not math.isfinite(base) or not factor > 0.0 or not math.isfinite(factor):
        raise ValueError(f"base must be above 1 and factor positive, both finite; got {base} and {factor}")
    half = rotated // 2
    if scaling == "ntk":
        base *= factor ** (half / max(1, half - 1))
    plain = [base ** (-i / half) for i in range(half)]
    if scaling == "linear":
        return [f / factor for f in plain], 1.0
    if scaling != "yarn":
        return plain, 1.0
    if trained < 1 or not fast > slow > 0.0:
        raise ValueError(f"yarn needs the trained positions and fast > slow > 0; got {trained}, {fast} and {slow}")

    def pair(turns: float) -> float:  # the pair that turns so often over the trained positions
        return half * math.log(trained / (turns * 2 * math.pi)) / math.log(base)

    low, high = max(0, math.floor(pair(fast))), min(rotated - 1, math.ceil(pair(slow)))
    share = [min(1.0, max(0.0, (i - low) / max(1e-3, high - low))) for i in range(half)]
    return [f * (1 - s) + f / factor * s for f, s in zip(plain, share)], 0.1 * math.log(max(1.0, factor)) + 1.0


@dataclass(frozen=True, eq=False)
class Rotary:
    """How heads turn; ``new_rotary`` makes it.  ``turns`` is a float64 tensor
    of turns a position, one for each pair; pairs are values ``2i`` and ``2i +
    1`` (``interleaved``) or ``i`` and ``i + len(turns)``."""

    turns: Any
    amplitude: float
    interleaved: bool

    def __post_init__(self) -> None:
        torch = _torch()
        if self.turns.dtype != torch.float64 or self.turns.ndim != 1 or not self.turns.is_contiguous():
            raise ValueError("turns must be a contiguous one-dimensional torch.float64 tensor; got "
                             f"{self.turns.dtype} {tuple(self.turns.shape)}")

    @property
    def rotated(self) -> int:
        return 2 * int(self.turns.shape[0])


def new_rotary(frequencies: Sequence[float], *, amplitude: float = 1.0, interleaved: bool = False,
               device: Any = "cuda") -> Rotary:
    """Puts ``frequencies`` (radians a position, one for each pair) on a device."""
    torch = _torch()
    turns = [float(f) / (2 * math.pi) for f in frequencies]
    if not all(math.isfinite(t) for t in (*turns, amplitude)):
        raise ValueError("frequencies and amplitude must be finite")
    return Rotary(torch.tensor(turns, dtype=torch.float64, device=device), float(amplitude), bool(interleaved))


def _heads(name: str, t: Any, shape: tuple, strides: tuple) -> None:
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {shape} == (tokens, heads, head_dim); got {tuple(t.shape)}")
    if strides[2] != 1:
        raise ValueError(f"{name} must be contiguous along head_dim")


def rotate_qk(
    q: Any,
    k: Any,
    positions: Any,
    rotary: Rotary,
    *,
    q_weight: Any | None = None,
    k_weight: Any | None = None,
    eps: float = 1e-6,
    cache: KVCache | None = None,
    values: Any | None = None,
    slots: Any | None = None,
    q_out: Any | None = None,
    k_out: Any | None = None,
    stream: Any | None = None,
) -> Any:
    """Norms and turns the heads of ``q`` [tokens, heads, head_dim] and ``k``
    [tokens, kv_heads, head_dim].

    q and k are bf16, f16 or f32, contiguous along head_dim (even, up to 256),
    other strides free: slices of a projection's result are taken as they are.
    With ``q_weight`` and ``k_weight`` [head_dim] (q's dtype or f32) each head is
    first normed, ``x / sqrt(mean(x^2) + eps) * weight``.  Then the first
    ``rotary.rotated`` of its values turn by ``positions`` [tokens] (int64 or
    int32, any value; above 2^53 rounded to 53 bits); the others stay.  Sums and
    products are f32, rounded once.

    Returns ``(q, k)`` of the inputs' dtype, in ``q_out`` and ``k_out`` if given
    (``q`` and ``k`` themselves for a result in place; rows that overlap raise).  With a ``cache``, the
    keys and ``values`` [tokens, kv_heads, head_dim] go into ``slots`` as
    ``kv_cache_write`` puts them there, without the keys' way through memory,
    and q alone is returned.
    """
    torch = _torch()
    index = q.get_device()
    for t in (k, positions, rotary.turns, q_weight, k_weight, values, slots, q_out, k_out,
              None if cache is None else cache.key_codes):
        if index < 0 or (t is not None and t.get_device() != index):
            _require_device(torch, {"q": q, "k": k, "positions": positions, "rotary": rotary.turns,
                                    "q_weight": q_weight, "k_weight": k_weight, "values": values, "slots": slots,
                                    "q_out": q_out, "k_out": k_out,
                                    "cache": None if cache is None else cache.key_codes})
    if stream is not None:
        with _on_stream(torch, q, stream):
            return rotate_qk(q, k, positions, rotary, q_weight=q_weight, k_weight=k_weight, eps=eps, cache=cache,
                             values=values, slots=slots, q_out=q_out, k_out=k_out)
    native = None if cache is None else cache._native
    dtype = q.dtype
    kind = _row_type(torch, "q", dtype)
    if k.dtype != dtype:
        raise ValueError(f"k must have the dtype of q, {dtype}; got {k.dtype}")
    if q.ndim != 3:
        raise ValueError(f"q must have shape (tokens, heads, head_dim); got {tuple(q.shape)}")
    if k.ndim != 3:
        raise ValueError(f"k must have shape (tokens, heads, head_dim); got {tuple(k.shape)}")
    tokens, heads, dim = q.shape
    kv_heads = k.shape[1] if cache is None else cache.kv_heads
    q_strides, k_strides, k_shape = q.stride(), k.stride(), (tokens, kv_heads, dim)
    _heads("q", q, (tokens, heads, dim), q_strides)
    _heads("k", k, k_shape, k_strides)
    if dim % 2 or not 2 <= dim <= 256:
        raise ValueError(f"head_dim must be even, from 2 to 256; got {dim}")
    if rotary.rotated > dim:
        raise ValueError(f"rotary turns {rotary.rotated} values; head_dim is {dim}")
    if positions.dtype != torch.int64 and positions.dtype != torch.int32:
        raise ValueError(f"positions must have dtype torch.int64 or torch.int32; got {positions.dtype}")
    if positions.shape != (tokens,) or not positions.is_contiguous():
        raise ValueError(f"positions must be contiguous with shape ({tokens},); got {tuple(positions.shape)}")
    if (q_weight is None) != (k_weight is None):
        raise ValueError("q_weight and k_weight are given both or neither")
    weight_kind = kind
    if q_weight is not None:
        for name, t in (("q_weight", q_weight), ("k_weight", k_weight)):
            if t.dtype not in (q.dtype, torch.float32) or t.dtype != q_weight.dtype:
                raise ValueError(f"q_weight and k_weight must have dtype {q.dtype} or torch.float32, both the same; "
                                 f"got {q_weight.dtype} and {k_weight.dtype}")
            if t.shape != (dim,) or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous with shape ({dim},); got {tuple(t.shape)}")
        weight_kind = _row_type(torch, "q_weight", q_weight.dtype)
    eps = float(eps)
    if not 0.0 <= eps < 3e38:
        raise ValueError(f"eps must be finite and not negative; got {eps}")
    if q_out is None:
        q_out = torch.empty((tokens, heads, dim), dtype=dtype, device=q.device)
        qo_strides = (heads * dim, dim)
    else:
        qo_strides = q_out.stride()
        _heads("q_out", q_out, (tokens, heads, dim), qo_strides)
        if q_out.dtype != dtype:
            raise ValueError(f"q_out must have dtype {dtype}; got {q_out.dtype}")
    k_at = v_at = (0, 0, 0)
    slots_at = (0, 4)
    if cache is None:
        if values is not None or slots is not None:
            raise ValueError("values and slots need a cache")
        if k_out is None:
            k_out = torch.empty(k_shape, dtype=dtype, device=q.device)
            k_at = (k_out.data_ptr(), kv_heads * dim, dim)
        else:
            strides = k_out.stride()
            _heads("k_out", k_out, k_shape, strides)
            if k_out.dtype != dtype:
                raise ValueError(f"k_out must have dtype {dtype}; got {k_out.dtype}")
            k_at = (k_out.data_ptr(), strides[0], strides[1])
    else:
        if k_out is not None:
            raise ValueError("with a cache the keys have no other result")
        if values is None or slots is None:
            raise ValueError("a cache needs values and slots")
        if dim != cache.head_dim:
            raise ValueError(f"head_dim must be the cache's, {cache.head_dim}; got {dim}")
        if values.ndim != 3:
            raise ValueError(f"values must have shape {k_shape}; got {tuple(values.shape)}")
        strides = values.stride()
        _heads("values", values, k_shape, strides)
        if values.dtype != dtype:
            raise ValueError(f"values must have the dtype of q, {dtype}; got {values.dtype}")
        _check_slots(torch, slots, tokens)
        v_at = (values.data_ptr(), strides[0], strides[1])
        slots_at = (slots.data_ptr(), slots.element_size())
    if tokens:
        if heads < 1 or kv_heads < 1:
            raise ValueError("q and k need at least one head")
        lib = _verified_library()
        _check(lib, lib.amd_strix_halo_kernels_rotate(
            index, _current_stream(torch, index), native,
            _ROTATE.pack(q.data_ptr(), q_strides[0], q_strides[1], k.data_ptr(), k_strides[0], k_strides[1], kind,
                         tokens, heads, kv_heads, dim, rotary.rotated, rotary.interleaved, positions.data_ptr(),
                         positions.element_size(), rotary.turns.data_ptr(), rotary.amplitude,
                         0 if q_weight is None else q_weight.data_ptr(),
                         0 if k_weight is None else k_weight.data_ptr(), weight_kind, eps, q_out.data_ptr(),
                         qo_strides[0], qo_strides[1], *k_at, *v_at, *slots_at)))
    if q.requires_grad or k.requires_grad or (q_weight is not None and (q_weight.requires_grad or k_weight.requires_grad)):
        given = (q, k) if q_weight is None else (q, k, q_weight, k_weight)
        q_out = _no_gradient(torch, "rotate_qk", q_out, *given)
        k_out = None if cache is not None else _no_gradient(torch, "rotate_qk", k_out, *given)
    return q_out if cache is not None else (q_out, k_out)
