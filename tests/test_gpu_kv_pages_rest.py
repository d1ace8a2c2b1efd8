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


def test_sums_of_pages_past_32_bits(device):
    """Sequences behind 2^31 pages that are asked for and not there are refused, with and without new tokens."""
    batch, width = 4096, 2**19 + 1024  # 8.6 GB of table, of which nothing is read
    table = torch.empty((batch, width), dtype=torch.int32, device=device)
    zeros = lambda n: torch.zeros(n, dtype=torch.int32, device=device)  # noqa: E731
    pool = shk.KVPages(table, zeros(batch), zeros(batch), torch.arange(8, dtype=torch.int32, device=device),
                       torch.full((1,), 8, dtype=torch.int32, device=device), 16)
    pool.lengths.fill_(16 * width - 1)
    pool.lengths[0] = pool.lengths[-1] = 20
    pool.owned[-1] = 2  # the last one's new token asks for no page
    table[-1, :2] = torch.tensor([50, 51], dtype=torch.int32)
    new = torch.ones(batch, dtype=torch.int32, device=device)
    new[1::2] = 0
    new[-1] = 1
    step = shk.kv_pages_step(pool, new, batch)
    taken = step.taken.tolist()
    assert taken[0] == taken[-1] == 1 and not any(taken[1:-1])
    assert pool.lengths.tolist() == [21] + [16 * width - 1] * (batch - 2) + [21]
    assert pool.owned.tolist() == [2] + [0] * (batch - 2) + [2] and pool.free_count.item() == 6
    slots, total = step.slots.tolist(), int(new.sum())
    assert slots[0] == 6 * 16 + 4 and slots[total - 1] == 51 * 16 + 4
    assert set(slots[1:total - 1]) == {-1} and set(slots[total:]) == {-1}
