"""Products in 8-bit floating point with a scale for each block of 128 values.

No counterpart in the reference, whose GEMMs are int4 and int8.  An operand is
e4m3 or e5m2 codes with one f32 scale for each block of 128 values along K, of
one row (activations, gradients) or of 128 rows (weights):

    scale = max|x| / L            L = 448 (e4m3) or 57344 (e5m2)
    code  = fp8(clamp(x / scale, -L, L))        value = code * scale

``quantize_fp8`` makes codes and scales of a tensor or of its transpose, and
``mm_fp8`` multiplies two of them.  The three products of a linear layer
``y = x w^T`` are one kernel, fed along its K:

    y  = mm_fp8(*q(x), *q(w, block_rows=128))
    dx = mm_fp8(*q(dy), *q(w, block_rows=128, transpose=True))
    dw = mm_fp8(*q(dy, transpose=True), *q(x, transpose=True))

(q for ``quantize_fp8``, its codes and scales passed as a and a_scale, b and
b_scale).  Both run on the current stream of the tensors' device, or on
``stream`` (which is then the current one for the call, its allocations
included), and read nothing back to the host.  There is no CPU path, and asking
a result for a gradient raises: the products above are the gradients.
"""

from __future__ import annotations

import struct
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

FP8_BLOCK = 128

# bytes of workspace by what they follow from: sizes, the result's type, and
# whether the operands' rows start on 16 bytes
_WORKSPACES: dict[tuple, int] = {}

# the structs of include/strix_halo_gfx950.h: every field is 8 bytes
_QUANTIZE = struct.Struct("=13q")
_MM = struct.Struct("=21q")


# of dtypes, filled at the first call
_KINDS: dict[Any, int] = {}
_SOURCES: dict[Any, int] = {}


def _fill(torch: Any) -> None:
    _SOURCES.update({torch.bfloat16: kt.SRC_BF16, torch.float16: kt.SRC_F16, torch.float32: kt.SRC_F32})
    _KINDS.update({torch.float8_e4m3fn: kt.FP8_E4M3, torch.float8_e5m2: kt.FP8_E5M2})


def _kind(name: str, dtype: Any) -> int:
    kind = _KINDS.get(dtype)
    if kind is None:
        raise ValueError(f"{name} must have dtype torch.float8_e4m3fn or torch.float8_e5m2; got {dtype}")
    return kind


def _value_type(name: str, dtype: Any) -> int:
    source = _SOURCES.get(dtype)
    if source is None:
        raise ValueError(f"{name} must have dtype torch.bfloat16, torch.float16 or torch.float32; got {dtype}")
    return source


def quantize_fp8(x: Any, *, block_rows: int = 1, transpose: bool = False, dtype: Any = None,
                 stream: Any | None = None) -> tuple[Any, Any]:
    """Codes and scales of ``x`` [rows, cols] (bf16, f16 or f32; contiguous
    along either axis), or of its transpose.

    Returns ``(codes, scales)`` of the operand, x or x^T, [R, C]: codes [R, C]
    in ``dtype`` (``torch.float8_e4m3fn``, the default, or
    ``torch.float8_e5m2``), each row on 16 bytes, on 128 where C is above 1024
    (what lies between two rows is not written), and f32 scales
    [ceil(R / block_rows), ceil(C / 128)] (stored with the blocks of one row
    ``ceil(R / block_rows)`` apart), ``block_rows`` 1 or 128.  A block of zeros
    has scale 0; one that holds an infinity or a NaN has that as its scale and
    zero codes, so that what it is multiplied with becomes NaN.
    """
    torch = _torch()
    index = x.get_device()
    if index < 0:
        _require_device(torch, {"x": x})
    if stream is not None:
        with _on_stream(torch, x, stream):
            return quantize_fp8(x, block_rows=block_rows, transpose=transpose, dtype=dtype)
    if not _KINDS:
        _fill(torch)
    dtype = torch.float8_e4m3fn if dtype is None else dtype
    kind, source = _kind("the result", dtype), _value_type("x", x.dtype)
    if block_rows not in (1, FP8_BLOCK):
        raise ValueError(f"block_rows must be 1 or {FP8_BLOCK}; got {block_rows}")
    if x.ndim != 2:
        raise ValueError(f"x must have shape (rows, cols); got {tuple(x.shape)}")
    (m, n), (m_stride, n_stride) = x.shape, x.stride()
    rows, cols = (n, m) if transpose else (m, n)  # of the operand
    turn = bool(transpose)
    if n_stride != 1 and n > 1:
        if m_stride != 1 and m > 1:
            raise ValueError("x must be contiguous along rows or columns")
        m, n, m_stride, turn = n, m, n_stride, not turn
    # rows on whole lines where that adds little: a product with K of 8111 takes 278 us
    # instead of 292, with 2064 180 instead of 190
    pitch = -(-cols // 128) * 128 if cols > 1024 else -(-cols // 16) * 16
    groups = rows if block_rows == 1 else -(-rows // FP8_BLOCK)
    codes = x.new_empty((rows, pitch), dtype=dtype)
    scales = x.new_empty_strided((groups, -(-cols // FP8_BLOCK)), (1, groups), dtype=torch.float32)
    if rows and cols:
        lib = _verified_library()
        _check(lib, lib.amd_strix_halo_kernels_fp8_quantize(
            index, _current_stream(torch, index),
            _QUANTIZE.pack(x.data_ptr(), source, m, n, m_stride if m > 1 else n, turn, block_rows, kind,
                           codes.data_ptr(), pitch, scales.data_ptr(), 1, groups)))
    if pitch != cols:
        codes = codes[:, :cols]
    if x.requires_grad:
        scales = _no_gradient(torch, "quantize_fp8", scales, x)
    return codes, scales


def mm_fp8(a: Any, b: Any, *, a_scale: Any, b_scale: Any, out_dtype: Any = None, out: Any | None = None,
           stream: Any | None = None) -> Any:
    """``out[m, n] = sum_k (a * a_scale)[m, k] (b * b_scale)[n, k]`` of fp8
    codes, K along the rows of both.

    ``a`` is [M, K] and ``b`` [N, K] (``torch.float8_e4m3fn`` or
    ``torch.float8_e5m2`` each; rows contiguous, any pitch), ``a_scale`` [M,
    ceil(K / 128)] and ``b_scale`` [ceil(N / 128), ceil(K / 128)] (a weight's
    blocks) or [N, ceil(K / 128)], f32 of any strides.  Returns [M, N] in
    ``out_dtype`` (bf16, the default, f16 or f32).  Sums are f32: inside a
    block of K by the matrix unit, over the blocks in an order that follows from
    the sizes (the same call has the same bits); rounded once at the end.

    f32 results, and results of a decode step's few rows, go through the 16-bit
    unit, whose sums are as f32 ones.  Other bf16 and f16 results go through the
    8-bit unit, which keeps the products of eight neighbours along K to 2^-13 of
    the power of two of the largest of them, cut towards zero.  That is 2e-5 of the
    results' rms where channels are alike, 8e-5 where some are hundreds of times
    the others, and up to 1.5e-4, nearly all of it towards zero, where the
    operands are of one sign besides (at worst 8.5e-4 of the largest products added
    up).  A bf16 result's own rounding is 1.7e-3; an f16 one's 2.1e-4 is no longer
    well above it.  ``out_dtype=torch.float32`` is the way around.

    Operands whose rows do not all start on 16 bytes are copied first; the codes
    of ``quantize_fp8`` do.
    """
    torch = _torch()
    index = a.get_device()
    for t in (b, a_scale, b_scale, a if out is None else out):
        if index < 0 or t.get_device() != index:
            _require_device(torch, {"a": a, "b": b, "a_scale": a_scale, "b_scale": b_scale, "out": out})
    if stream is not None:
        with _on_stream(torch, a, stream):
            return mm_fp8(a, b, a_scale=a_scale, b_scale=b_scale, out_dtype=out_dtype, out=out)
    if not _KINDS:
        _fill(torch)
    a_kind, b_kind = _kind("a", a.dtype), _kind("b", b.dtype)
    if a.ndim != 2 or b.ndim != 2 or a.shape[1] != b.shape[1]:
        raise ValueError(f"a and b must have shapes (M, K) and (N, K); got {tuple(a.shape)} and {tuple(b.shape)}")
    (m, k), n = a.shape, b.shape[0]
    (a_pitch, a_step), (b_pitch, b_step) = a.stride(), b.stride()
    if k > 1 and (a_step != 1 or b_step != 1):
        raise ValueError("rows of a and b must be contiguous")
    blocks = -(-k // FP8_BLOCK)
    if a_scale.dtype != torch.float32 or b_scale.dtype != torch.float32:
        name, t = ("a_scale", a_scale) if a_scale.dtype != torch.float32 else ("b_scale", b_scale)
        raise ValueError(f"{name} must have dtype torch.float32; got {t.dtype}")
    if a_scale.shape != (m, blocks):
        raise ValueError(f"a_scale must have shape {(m, blocks)} == (M, ceil(K/128)); got {tuple(a_scale.shape)}")
    if b_scale.shape == (-(-n // FP8_BLOCK), blocks):
        b_rows = FP8_BLOCK
    elif b_scale.shape == (n, blocks):
        b_rows = 1
    else:
        raise ValueError(f"b_scale must have shape {(-(-n // FP8_BLOCK), blocks)} == (ceil(N/128), ceil(K/128)) or "
                         f"{(n, blocks)} == (N, ceil(K/128)); got {tuple(b_scale.shape)}")
    if out is None:
        out_dtype = torch.bfloat16 if out_dtype is None else out_dtype
        out_type, out_stride = _value_type("the result", out_dtype), n
        out = a.new_empty((m, n), dtype=out_dtype)
    else:
        out_type, out_stride = _value_type("out", out.dtype), out.stride(0) if m > 1 else n
        if out_dtype is not None and out.dtype != out_dtype:
            raise ValueError(f"out must have dtype {out_dtype}; got {out.dtype}")
        if out.shape != (m, n) or (n > 1 and out.stride(1) != 1) or out_stride < n:
            raise ValueError(f"out must have shape {(m, n)} and contiguous rows; got {tuple(out.shape)}")
    if m and n:
        if m == 1:
            a_pitch = k
        if n == 1:
            b_pitch = k
        a_at, b_at = a.data_ptr(), b.data_ptr()
        lib = _verified_library()
        given = (a_at, a_pitch, a_kind, b_at, b_pitch, b_kind, a_scale.data_ptr(), *a_scale.stride(),
                 b_scale.data_ptr(), *b_scale.stride(), b_rows, m, n, k, out.data_ptr(), out_stride, out_type)
        key = (m, n, k, out_type, (a_at | (a_pitch if m > 1 else 0)) % 16 == 0,
               (b_at | (b_pitch if n > 1 else 0)) % 16 == 0)
        nbytes = _WORKSPACES.get(key)
        if nbytes is None:
            nbytes = lib.amd_strix_halo_kernels_fp8_mm_workspace(_MM.pack(*given, 0, 0))
            if nbytes < 0:
                _check(lib, 1)
            if len(_WORKSPACES) < 4096:
                _WORKSPACES[key] = nbytes
        work = a.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        _check(lib, lib.amd_strix_halo_kernels_fp8_mm(
            index, _current_stream(torch, index), _MM.pack(*given, 0 if work is None else work.data_ptr(), nbytes)))
    if a_scale.requires_grad or b_scale.requires_grad or a.requires_grad or b.requires_grad:
        return _no_gradient(torch, "mm_fp8", out, a, b, a_scale, b_scale)
    return out
