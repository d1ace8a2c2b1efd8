"""Pages of the cache's sequences, handed out and taken back on the device.

No counterpart in the reference.  ``KVPages`` holds which pages of a pool belong
to which sequence; ``kv_pages_step`` turns the numbers of new tokens of a batch
into the slots and positions that ``kv_cache_write`` and ``rotate_qk`` take and
the table that ``kv_cache_attention`` reads.  Nothing is read back to the host, so
a step can be captured into a graph with the rest of its layer.  One pool serves
all layers whose caches have the same pages.
"""

from __future__ import annotations

import struct
from dataclasses import dataclass
from typing import Any, NamedTuple

from .native import _check, _current_stream, _on_stream, _require_device, _torch, _verified_library

KV_PLAN_BATCH = 4096

# shk_kv_plan of include/strix_halo_gfx950.h: every field is 8 bytes
_PLAN = struct.Struct("=17q")

_PARTS = ("page_table", "lengths", "owned", "free_pages", "free_count")


@dataclass(frozen=True, eq=False)
class KVPages:
    """The pages of a batch's sequences; ``new_kv_pages`` makes it.

    All are contiguous int32 tensors of one device.  Sequence b holds
    ``lengths[b]`` tokens and owns the first ``owned[b]`` pages of
    ``page_table[b]`` ([batch, width], batch up to 4096; what lies behind them is
    not read).  ``free_pages[:free_count[0]]`` is a stack of unused pages; it has a
    place for every page that may come back.  page_size is a power of two from 16
    to 1024.  A caller may shorten ``lengths`` between steps (tokens that were not
    kept): the pages stay with the sequence.
    """

    page_table: Any
    lengths: Any
    owned: Any
    free_pages: Any
    free_count: Any
    page_size: int

    def __post_init__(self) -> None:
        torch = _torch()
        table = self.page_table
        if table.ndim != 2:
            raise ValueError(f"page_table must have shape (batch, width); got {tuple(table.shape)}")
        batch = int(table.shape[0])
        for name, shape in (("page_table", table.shape), ("lengths", (batch,)), ("owned", (batch,)),
                            ("free_pages", (self.free_pages.numel(),)), ("free_count", (1,))):
            t = getattr(self, name)
            if t.dtype != torch.int32 or tuple(t.shape) != tuple(shape) or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous torch.int32 tensor of shape {tuple(shape)}; got "
                                 f"{t.dtype} {tuple(t.shape)}")
            if t.device != table.device:
                raise ValueError(f"{name} is on {t.device}, expected {table.device}")
        if not 1 <= batch <= KV_PLAN_BATCH or table.shape[1] < 1:
            raise ValueError(f"page_table needs 1 to {KV_PLAN_BATCH} sequences and at least one page each; got "
                             f"{tuple(table.shape)}")
        size = self.page_size
        if isinstance(size, bool) or not isinstance(size, int) or not 16 <= size <= 1024 or size & (size - 1):
            raise ValueError(f"page_size must be a power of two from 16 to 1024; got {size!r}")
        object.__setattr__(self, "_ticket", torch.zeros(1, dtype=torch.int32, device=table.device))

    def __reduce__(self) -> Any:
        # copies and loaded pools are made of their own tensors
        return KVPages, (*(getattr(self, n) for n in _PARTS), self.page_size)


def new_kv_pages(batch: int, width: int, pages: int, page_size: int, *, first: int = 0,
                 device: Any = "cuda") -> KVPages:
    """``batch`` empty sequences of up to ``width`` pages each, and the pages
    ``first`` .. ``pages - 1`` free (those before ``first`` are the caller's, a
    shared prefix for instance)."""
    torch = _torch()
    if not 0 <= first <= pages:
        raise ValueError(f"first must be from 0 to {pages}; got {first}")
    made = {"dtype": torch.int32, "device": device}
    free = torch.arange(pages - 1, first - 1, -1, **made)  # handed out in rising order
    return KVPages(torch.zeros((batch, width), **made), torch.zeros(batch, **made), torch.zeros(batch, **made), free,
                   torch.full((1,), pages - first, **made), page_size)


class KVStep(NamedTuple):
    """Where a step's tokens go: ``slots`` (int64), ``positions`` and
    ``sequences`` (int32) [capacity], ``starts`` [batch + 1] and ``taken``
    [batch] (int32)."""

    slots: Any
    positions: Any
    sequences: Any
    starts: Any
    taken: Any


def kv_pages_step(pages: KVPages, new_tokens: Any, capacity: int, *, stream: Any | None = None) -> KVStep:
    """Makes room for ``new_tokens[b]`` (int32 [batch]) tokens of each sequence.

    A negative number ends the sequence: its pages are free again, for this step
    too.  The others' tokens are numbered through in order of the sequences, up
    to ``capacity`` of them; ``starts[b]`` is the first of sequence b.  Token i has
    ``positions[i]`` in its sequence ``sequences[i]`` and belongs into
    ``slots[i]``; behind the last one they are 0, -1 and -1.  A sequence that
    would not fit its row of the table, the capacity, or the free pages (asked
    for in order of the sequences: a sequence that asks for any behind the first
    one that cannot be served is not served either) is refused: its slots are
    -1, its length and pages stay, and ``taken[b]`` is 0 instead of
    ``new_tokens[b]``.  Nothing of it is in the cache then: what a later call takes
    off the lengths (``verify_draft``) is to leave it out.

    Updates ``pages`` in place: lengths, owned, page_table and the free stack.
    Steps of one pool must follow each other.
    """
    torch = _torch()
    table = pages.page_table
    index = table.get_device()
    if index < 0 or new_tokens.get_device() != index:
        _require_device(torch, {"pages": table, "new_tokens": new_tokens})
    if stream is not None:
        with _on_stream(torch, table, stream):
            return kv_pages_step(pages, new_tokens, capacity)
    batch, width = table.shape
    if pages.lengths.shape[0] != batch or pages.owned.shape[0] != batch or not table.is_contiguous():
        pages.__post_init__()  # a tensor was given other memory: says what is wrong
    if new_tokens.dtype != torch.int32 or new_tokens.shape != (batch,) or not new_tokens.is_contiguous():
        raise ValueError(f"new_tokens must be a contiguous torch.int32 tensor of shape ({batch},); got "
                         f"{new_tokens.dtype} {tuple(new_tokens.shape)}")
    if isinstance(capacity, bool) or not isinstance(capacity, int) or not 0 <= capacity < 2**31:
        raise ValueError(f"capacity must be an int from 0 to {2**31 - 1}; got {capacity!r}")
    # one allocation, the 8-byte slots first
    work = torch.empty(4 * capacity + 2 * batch + 1, dtype=torch.int32, device=table.device)
    slots, positions, sequences, starts, taken = work.split_with_sizes(
        (2 * capacity, capacity, capacity, batch + 1, batch))
    step = KVStep(slots.view(torch.int64), positions, sequences, starts, taken)
    lib = _verified_library()
    _check(lib, lib.amd_strix_halo_kernels_kv_plan(
        index, _current_stream(torch, index),
        _PLAN.pack(table.data_ptr(), batch, width, pages.lengths.data_ptr(), pages.owned.data_ptr(),
                   pages.free_pages.data_ptr(), pages.free_pages.shape[0], pages.free_count.data_ptr(),
                   pages.page_size, new_tokens.data_ptr(), capacity, step.slots.data_ptr(), positions.data_ptr(),
                   sequences.data_ptr(), starts.data_ptr(), taken.data_ptr(), pages._ticket.data_ptr())))
    return step
