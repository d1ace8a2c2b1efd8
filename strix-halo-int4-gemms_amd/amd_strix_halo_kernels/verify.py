"""Verification of drafted tokens against the target's probabilities.

No counterpart in the reference.  A draft model (or a lookup) proposes tokens for
each sequence, the target model scores all of them in one step
(``kv_cache_attention`` takes several newest tokens of a sequence), and
``verify_draft`` keeps those that the target would have drawn as well and draws
the token that follows, so that what comes out is distributed as the target's own
tokens.  Random numbers are inputs.
"""

from __future__ import annotations

import struct
from typing import Any

from .kv_cache import _row_type
from .native import _check, _current_stream, _on_stream, _require_device, _torch, _verified_library

MOST_DRAFTS = 63

# shk_verify of include/strix_halo_gfx950.h: every field is 8 bytes
_VERIFY = struct.Struct("=19q")

_WORKSPACES: dict[tuple, int] = {}  # bytes, by batch and vocabulary


def verify_draft(
    target: Any,
    draft: Any | None,
    tokens: Any,
    uniforms: Any,
    *,
    counts: Any | None = None,
    lengths: Any | None = None,
    stream: Any | None = None,
) -> tuple[Any, Any]:
    """``(out, kept)``: the tokens that each sequence goes on with.

    ``tokens`` [batch, drafts] (int64 or int32, up to 63 drafts) were drawn from
    ``draft`` [batch, drafts, vocab], or taken for certain where that is None;
    ``target`` [batch, drafts + 1, vocab] are the target's probabilities at each
    of them and after the last (bf16, f16 or f32, the draft's of the same dtype,
    contiguous along the vocabulary; they need not add up to 1), ``uniforms``
    [batch, drafts + 1] f32 numbers from [0, 1).

    Draft i is kept while ``uniforms[b, i] * draft[b, i, token] < target[b, i,
    token]``.  The next token is the first one at which the running sum of the
    weights passes ``uniforms[b, drafts]`` times their sum, the weights being
    ``max(target - draft, 0)`` at the first draft that was not kept (the target's
    alone where these are all 0), or the target's after the last draft.  Sums are
    64 bits.  Weights that are NaN or negative count as 0; where none is left the
    token is -1.

    Returns ``out`` int64 [batch, drafts + 1], the kept drafts, the next token,
    then -1, and ``kept`` int32 [batch].  ``counts`` (int32 [batch]): sequence b
    has only its first ``counts[b]`` drafts.  ``lengths`` (int32 [batch]) is
    changed in place where given: ``lengths[b]`` loses the drafts that were not
    kept, which is what is then left of the cached tokens (``KVPages.lengths``).
    It has to hold them before: of a sequence that ``kv_pages_step`` refused no
    draft is in the cache, which ``counts=(step.taken - 1).clamp(min=0)`` says
    where a step takes a token and its drafts; its row of ``out`` is to be ignored.
    """
    torch = _torch()
    index = target.get_device()
    for t in (draft, tokens, uniforms, counts, lengths):
        if index < 0 or (t is not None and t.get_device() != index):
            _require_device(torch, {"target": target, "draft": draft, "tokens": tokens, "uniforms": uniforms,
                                    "counts": counts, "lengths": lengths})
    if stream is not None:
        with _on_stream(torch, target, stream):
            return verify_draft(target, draft, tokens, uniforms, counts=counts, lengths=lengths)
    kind = _row_type(torch, "target", target.dtype)
    if tokens.dtype != torch.int64 and tokens.dtype != torch.int32:
        raise ValueError(f"tokens must have dtype torch.int64 or torch.int32; got {tokens.dtype}")
    if tokens.ndim != 2 or not tokens.is_contiguous():
        raise ValueError(f"tokens must be contiguous with shape (batch, drafts); got {tuple(tokens.shape)}")
    batch, drafts = tokens.shape
    if drafts > MOST_DRAFTS:
        raise ValueError(f"verify_draft takes up to {MOST_DRAFTS} drafts a sequence; got {drafts}")
    if target.ndim != 3 or target.shape[:2] != (batch, drafts + 1) or target.shape[2] < 1:
        raise ValueError(f"target must have shape ({batch}, {drafts + 1}, vocab); got {tuple(target.shape)}")
    vocab = int(target.shape[2])
    if target.stride(2) != 1 and vocab > 1:
        raise ValueError("target must be contiguous along the vocabulary")
    d_at = (0, 0, 0)
    if draft is not None:
        if draft.dtype != target.dtype or draft.shape != (batch, drafts, vocab):
            raise ValueError(f"draft must have shape {(batch, drafts, vocab)} and dtype {target.dtype}; got "
                             f"{tuple(draft.shape)} and {draft.dtype}")
        if draft.stride(2) != 1 and vocab > 1:
            raise ValueError("draft must be contiguous along the vocabulary")
        if drafts:
            d_at = (draft.data_ptr(), draft.stride(0), draft.stride(1))
    if uniforms.dtype != torch.float32 or uniforms.shape != (batch, drafts + 1) or not uniforms.is_contiguous():
        raise ValueError(f"uniforms must be contiguous with shape {(batch, drafts + 1)} and dtype torch.float32; got "
                         f"{tuple(uniforms.shape)} and {uniforms.dtype}")
    for name, t in (("counts", counts), ("lengths", lengths)):
        if t is not None and (t.dtype != torch.int32 or t.shape != (batch,) or not t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous torch.int32 tensor of shape ({batch},); got {t.dtype} "
                             f"{tuple(t.shape)}")
    out = torch.empty((batch, drafts + 1), dtype=torch.int64, device=target.device)
    kept = torch.empty(batch, dtype=torch.int32, device=target.device)
    if batch:
        def args(at: int, nbytes: int) -> bytes:
            return _VERIFY.pack(target.data_ptr(), target.stride(0), target.stride(1), *d_at, kind, batch, drafts,
                                vocab, tokens.data_ptr(), tokens.element_size(), uniforms.data_ptr(),
                                0 if counts is None else counts.data_ptr(), out.data_ptr(), kept.data_ptr(),
                                0 if lengths is None else lengths.data_ptr(), at, nbytes)

        lib = _verified_library()
        nbytes = _WORKSPACES.get((batch, vocab))
        if nbytes is None:
            nbytes = lib.amd_strix_halo_kernels_verify_workspace(args(0, 0))
            if nbytes < 0:
                _check(lib, 1)
            if len(_WORKSPACES) < 4096:
                _WORKSPACES[batch, vocab] = nbytes
        work = torch.empty(nbytes, dtype=torch.uint8, device=target.device) if nbytes else None
        _check(lib, lib.amd_strix_halo_kernels_verify(index, _current_stream(torch, index),
                                                      args(work.data_ptr() if nbytes else 0, nbytes)))
    return out, kept
