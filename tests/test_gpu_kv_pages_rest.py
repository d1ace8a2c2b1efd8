"""Pages of sequences whose lengths a caller has set: those without new tokens, and sums past 32 bits."""

from __future__ import annotations

import random

import pytest

torch = pytest.importorskip("torch")

import amd_strix_halo_kernels as shk  # noqa: E402
from tests import _step_ref as ref  # noqa: E402

pytestmark = pytest.mark.gpu


def _state(pages):
    return {"page_table": pages.page_table.tolist(), "lengths": pages.lengths.tolist(), "owned": pages.owned.tolist(),
            "free": pages.free_pages.tolist()[:int(pages.free_count)]}


def _step(pool, new, capacity, device):
    state = _state(pool)
    want = ref.step(state, new, capacity, pool.page_size)
    got = shk.kv_pages_step(pool, torch.tensor(new, dtype=torch.int32, device=device), capacity)
    for name, w in zip(("slots", "positions", "sequences", "starts", "taken"), want):
        assert getattr(got, name).tolist() == w, name
    now = _state(pool)
    assert now["lengths"] == state["lengths"] and now["owned"] == state["owned"] and now["free"] == state["free"]
    for row, w, n in zip(now["page_table"], state["page_table"], state["owned"]):
        assert row[:n] == w[:n]
    return now


@pytest.mark.parametrize("batch,width,pages,capacity", [(5, 8, 40, 0), (5, 8, 40, 64), (700, 12, 4000, 9000),
                                                        (40, 200, 8000, 30000)])
def test_lengths_past_the_owned_pages(device, batch, width, pages, capacity):
    """A sequence whose length needs pages that it does not own gets them with its next step, new tokens or none:
    no page is lost and none is in two places."""
    rng = random.Random(batch)
    pool = shk.new_kv_pages(batch, width, pages, 16, device=device)
    pool.page_table.fill_(-7)
    for n in range(5):
        grown = [min(16 * width, x + rng.choice([0, 0, rng.randint(0, 60)])) for x in pool.lengths.tolist()]
        pool.lengths.copy_(torch.tensor(grown, dtype=torch.int32))
        new = [rng.choice([0, 0, -1, rng.randint(1, 20)]) for _ in range(batch)]
        now = _step(pool, new, capacity, device)
        held = [p for row, k in zip(now["page_table"], now["owned"]) for p in row[:k]]
        assert sorted(held + now["free"]) == list(range(pages))
    # (behind a token that passes the capacity all are refused, those without tokens too)
    assert capacity == 0 or max(now["owned"]) > 1


def test_pages_for_sequences_without_tokens_run_out(device):
    pool = shk.new_kv_pages(4, 8, 6, 16, device=device)
    pool.lengths.copy_(torch.tensor([40, 33, 5, 0], dtype=torch.int32))
    now = _step(pool, [0, 0, 0, 0], 8, device)
    assert now["owned"] == [3, 3, 0, 0] and now["free"] == []
    assert sorted(now["page_table"][0][:3] + now["page_table"][1][:3]) == [0, 1, 2, 3, 4, 5]
