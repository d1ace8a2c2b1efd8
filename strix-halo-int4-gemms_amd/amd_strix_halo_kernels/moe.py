"""The gated mixture-of-experts layer for a few tokens.

No counterpart in the reference, whose ragged dots take int4 activations
sorted by expert.  ``moe_swiglu_int4`` takes a decode step's tokens as they
are (bf16 or f16, unsorted, with the router's choices) and the experts' int4
weights in the layouts of ``ragged_dot_int4``, and runs the whole layer:
gather, up and gate products, SwiGLU, down product, weighted sum.
"""

from __future__ import annotations

import struct
from typing import Any

from . import kernel_table as kt
from .metadata import SUPPORTED_SUBCHANNELS, GemmLayout, ScaleMode, ScaleSpec
from .native import (
    _check,
    _current_stream,
    _no_gradient,
    _on_stream,
    _require_device,
    _torch,
    _verified_library,
)

MOE_MAX_TOKENS = 64
MOE_MAX_PAIRS = 1024
MOE_MAX_EXPERTS = 1024


# shk_moe of include/strix_halo_gfx950.h: every field is 8 bytes
_MOE = struct.Struct("=20q")


def _require(name: str, tensor: Any, shape: tuple[int, ...], dtype: Any, what: str) -> None:
    if tensor.shape != shape:
        raise ValueError(f"{name} must have shape {shape} == {what}; got {tuple(tensor.shape)}")
    if tensor.dtype != dtype:
        raise ValueError(f"{name} must have dtype {dtype}; got {tensor.dtype}")
    if not tensor.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _outputs(torch: Any, out: Any, a: Any, b: Any, c: Any, d: Any) -> Any:
    if a.requires_grad or b.requires_grad or c.requires_grad or d.requires_grad:
        return _no_gradient(torch, "moe_swiglu_int4", out, a, b, c, d)
    return out


def moe_swiglu_int4(
    x: Any,
    up_gate: Any,
    down: Any,
    expert_ids: Any,
    expert_weights: Any,
    *,
    up_gate_scale: Any,
    down_scale: Any,
    scale: ScaleSpec = ScaleSpec(ScaleMode.PER_CHANNEL),
    layout: GemmLayout = GemmLayout.NN,
    out: Any | None = None,
    stream: Any | None = None,
) -> Any:
    """y[t] = sum_j expert_weights[t, j] * down_e(up_e(x[t]) * silu(gate_e(x[t]))),
    with e = expert_ids[t, j].

    ``x`` is [tokens, hidden] (bf16 or f16, rows contiguous), ``expert_ids``
    [tokens, top] (int64 or int32) and ``expert_weights`` [tokens, top] f32,
    as ``torch.topk`` over a router's probabilities leaves them; ids outside
    the experts, such as -1 for padding, add nothing.  Weights are packed int4
    (K in byte pairs) in the layouts of ``ragged_dot_int4``:

    * NN: ``up_gate[E, ceil(hidden/2), 2*inner]`` with the columns [up | gate]
      of ``fused_swiglu_up_gate``, ``down[E, ceil(inner/2), hidden]``;
    * NT: ``up_gate[E, 2*inner, ceil(hidden/2)]``, ``down[E, hidden,
      ceil(inner/2)]``.

    Scales are bf16: per-channel ``up_gate_scale[E, 2*inner]`` and
    ``down_scale[E, hidden]``, or with subchannel S ``[E, ceil(K/S), columns]``.
    Activations are not quantized; sums and the value between the products
    are f32.  Takes up to 64 tokens (``ragged_dot_int4`` takes more, quantized
    and sorted by expert), 1024 (token, expert) pairs and 1024 experts.  Returns [tokens, hidden] in
    x's dtype.  Runs on the current stream, or on ``stream`` (which is then the
    current one for the call, its allocations included); nothing is read back
    to the host, and there is no gradient (asking the result for one raises).
    """
    layout = GemmLayout(layout)
    if layout not in (GemmLayout.NN, GemmLayout.NT):
        raise ValueError(f"unsupported MoE layout {layout.value}; supported layouts are nn, nt")
    torch = _torch()
    index = x.get_device()
    for t in (up_gate, down, expert_ids, expert_weights, up_gate_scale, down_scale, x if out is None else out):
        if index < 0 or t.get_device() != index:
            _require_device(torch, {"x": x, "up_gate": up_gate, "down": down, "expert_ids": expert_ids,
                                    "expert_weights": expert_weights, "up_gate_scale": up_gate_scale,
                                    "down_scale": down_scale, "out": out})  # says what is wrong
    if stream is not None:
        with _on_stream(torch, x, stream):
            return moe_swiglu_int4(x, up_gate, down, expert_ids, expert_weights, up_gate_scale=up_gate_scale,
                                   down_scale=down_scale, scale=scale, layout=layout, out=out)
    if x.dtype != torch.bfloat16 and x.dtype != torch.float16:
        raise ValueError(f"x must have dtype torch.bfloat16 or torch.float16; got {x.dtype}")
    if x.ndim != 2 or x.shape[1] < 1:
        raise ValueError(f"x must have shape (tokens, hidden); got {tuple(x.shape)}")
    if x.stride(1) != 1 and x.shape[1] > 1:
        raise ValueError("rows of x must be contiguous")
    tokens, hidden = int(x.shape[0]), int(x.shape[1])
    if up_gate.ndim != 3 or up_gate.shape[0] < 1:
        raise ValueError(f"up_gate must have shape (experts, K/2, N) or (experts, N, K/2); got {tuple(up_gate.shape)}")
    experts = int(up_gate.shape[0])
    nt = layout is GemmLayout.NT
    columns = int(up_gate.shape[1 if nt else 2])
    if columns < 2 or columns % 2:
        raise ValueError(f"up_gate needs an even number of [up | gate] columns; got {columns}")
    inner = columns // 2
    k_up, k_down = (hidden + 1) // 2, (inner + 1) // 2
    _require("up_gate", up_gate, (experts, columns, k_up) if nt else (experts, k_up, columns), torch.uint8,
             "(experts, 2*inner, hidden/2)" if nt else "(experts, hidden/2, 2*inner)")
    _require("down", down, (experts, hidden, k_down) if nt else (experts, k_down, hidden), torch.uint8,
             "(experts, hidden, inner/2)" if nt else "(experts, inner/2, hidden)")
    group = 0
    if scale.mode is ScaleMode.SUBCHANNEL:
        group = scale.subchannel_size or 0
        if group not in SUPPORTED_SUBCHANNELS:
            raise ValueError(f"subchannel_size must be one of {SUPPORTED_SUBCHANNELS}; got {group}")
    for name, t, k, n in (("up_gate_scale", up_gate_scale, hidden, columns), ("down_scale", down_scale, inner, hidden)):
        if group:
            _require(name, t, (experts, -(-k // group), n), torch.bfloat16, "(experts, ceil(K/S), columns)")
        else:
            _require(name, t, (experts, n), torch.bfloat16, "(experts, columns)")
    if expert_ids.ndim != 2 or expert_ids.shape[0] != tokens:
        raise ValueError(f"expert_ids must have shape ({tokens}, top); got {tuple(expert_ids.shape)}")
    top = int(expert_ids.shape[1])
    if expert_ids.dtype != torch.int64 and expert_ids.dtype != torch.int32:
        raise ValueError(f"expert_ids must have dtype torch.int64 or torch.int32; got {expert_ids.dtype}")
    _require("expert_weights", expert_weights, (tokens, top), torch.float32, "(tokens, top)")
    if not expert_ids.is_contiguous():
        raise ValueError("expert_ids must be contiguous")
    if tokens > MOE_MAX_TOKENS or tokens * top > MOE_MAX_PAIRS:
        raise ValueError(f"moe_swiglu_int4 takes up to {MOE_MAX_TOKENS} tokens and {MOE_MAX_PAIRS} (token, expert) "
                         f"pairs; got {tokens} and {tokens * top}. ragged_dot_int4 takes more, quantized and sorted by "
                         "expert")
    if up_gate.numel() < 4 or down.numel() < 4:
        raise ValueError("up_gate and down must hold at least 4 bytes each")
    if experts > MOE_MAX_EXPERTS:
        raise ValueError(f"moe_swiglu_int4 takes up to {MOE_MAX_EXPERTS} experts; got {experts}")
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    else:
        _require("out", out, (tokens, hidden), x.dtype, "(tokens, hidden)")
    if tokens == 0:
        return _outputs(torch, out, x, expert_weights, up_gate_scale, down_scale)
    # h as two bf16 terms with rows of whole 128s, and f32 results, for each
    # pair; a counter for each 128 columns of the output
    nbytes = 4 * (tokens * top * (-(-inner // 128) * 128 + hidden) + -(-hidden // 128))
    work = x.new_empty(nbytes, dtype=torch.uint8)
    args = _MOE.pack(x.data_ptr(), x.stride(0), kt.SRC_BF16 if x.dtype == torch.bfloat16 else kt.SRC_F16, tokens,
                     hidden, inner, experts, top, up_gate.data_ptr(), up_gate_scale.data_ptr(), down.data_ptr(),
                     down_scale.data_ptr(), group, kt.LAYOUT_NT if nt else kt.LAYOUT_NN, expert_ids.data_ptr(),
                     expert_ids.element_size(), expert_weights.data_ptr(), out.data_ptr(),
                     work.data_ptr(), nbytes)
    lib = _verified_library()
    _check(lib, lib.amd_strix_halo_kernels_moe(index, _current_stream(torch, index), args))
    return _outputs(torch, out, x, expert_weights, up_gate_scale, down_scale)
