"""Pages of a step against the same rules on Python lists, whole numbers all."""

from __future__ import annotations

import random

import pytest

torch = pytest.importorskip("torch")

import amd_strix_halo_kernels as shk  # noqa: E402
from tests import _step_ref as ref  # noqa: E402

pytestmark = pytest.mark.gpu


def _state(pages):
    free = pages.free_pages.tolist()[:int(pages.free_count)]
    return {"page_table": pages.page_table.tolist(), "lengths": pages.lengths.tolist(), "owned": pages.owned.tolist(),
            "free": free}


def _compare(pages, got, state, want):
    for name, w in zip(("slots", "positions", "sequences", "starts", "taken"), want):
        assert getattr(got, name).tolist() == w, name
    now = _state(pages)
    assert now["lengths"] == state["lengths"] and now["owned"] == state["owned"] and now["free"] == state["free"]
    for row, w, n in zip(now["page_table"], state["page_table"], state["owned"]):
        assert row[:n] == w[:n]


@pytest.mark.parametrize("batch,width,pages,page,most", [(1, 4, 6, 16, 30), (3, 8, 12, 16, 40), (64, 20, 700, 32, 70),
                                                         (65, 9, 300, 16, 50), (700, 6, 2500, 64, 100),
                                                         (4096, 3, 6000, 16, 12)])
def test_steps(device, batch, width, pages, page, most):
    """Sequences grow, are shortened, end and are refused, step after step."""
    rng = random.Random(batch)
    pool = shk.new_kv_pages(batch, width, pages, page, device=device)
    state = _state(pool)
    refused = 0
    for n in range(8):
        new = [rng.choice([0, 1, 1, rng.randint(0, most), rng.randint(0, most), -1]) for _ in range(batch)]
        capacity = max(0, sum(max(0, x) for x in new) + rng.choice([0, 0, 5, -3]))
        want = ref.step(state, new, capacity, page)
        got = shk.kv_pages_step(pool, torch.tensor(new, dtype=torch.int32, device=device), capacity)
        torch.cuda.synchronize()
        _compare(pool, got, state, want)
        refused += sum(x > 0 and t == 0 for x, t in zip(new, want[4]))
        # tokens that were not kept
        cut = [rng.randint(0, min(x, 5)) if rng.random() < 0.5 else 0 for x in state["lengths"]]
        state["lengths"] = [x - c for x, c in zip(state["lengths"], cut)]
        pool.lengths.sub_(torch.tensor(cut, dtype=torch.int32, device=device))
        held = [p for row, n in zip(state["page_table"], state["owned"]) for p in row[:n]]
        assert sorted(held + state["free"]) == list(range(pages))  # no page twice, none lost
    assert refused or batch < 3


def test_refusals_of_a_step(device):
    """The table's width, the capacity and the free pages, each at its limit and one past it."""
    def once(new, capacity, *, width=4, pages=8, lengths=None):
        pool = shk.new_kv_pages(len(new), width, pages, 16, device=device)
        state = _state(pool)
        if lengths:
            first = torch.tensor(lengths, dtype=torch.int32, device=device)
            shk.kv_pages_step(pool, first, 4096)
            ref.step(state, lengths, 4096, 16)
        want = ref.step(state, new, capacity, 16)
        got = shk.kv_pages_step(pool, torch.tensor(new, dtype=torch.int32, device=device), capacity)
        _compare(pool, got, state, want)
        return got.taken.tolist()

    assert once([64], 64) == [64]
    assert once([65], 65) == [0]                         # five pages in a table of four
    assert once([10, 10], 19) == [10, 0]                 # the second passes the capacity
    assert once([64, 64], 128) == [64, 64]               # all eight pages
    assert once([64, 49, 16], 129, pages=8) == [64, 49, 0]
    assert once([64, 17, 49, 1], 131, pages=7) == [64, 17, 0, 0]  # behind one that is refused none is served
    assert once([64, 64, 3], 131, pages=9, lengths=[0, 0, 5]) == [64, 64, 3]  # asks for no page
    assert once([0, 0], 0) == [0, 0]
    assert once([-1, 64], 64, pages=6, lengths=[50, 20]) == [0, 0]  # 84 tokens in a table of 64
    assert once([-1, 40], 64, pages=6, lengths=[50, 20]) == [0, 40]  # on the pages that the first gave back


def test_large_steps(device):
    """Many workgroups: prompts of thousands of tokens, pages handed out and taken back at once."""
    batch, width, page = 37, 600, 16
    pool = shk.new_kv_pages(batch, width, 20000, page, first=7, device=device)
    state = _state(pool)
    assert min(state["free"]) == 7
    rng = random.Random(3)
    for n in range(3):
        new = [rng.randint(0, 4500) if rng.random() < 0.8 else -1 for _ in range(batch)]
        capacity = sum(max(0, x) for x in new) + 77
        want = ref.step(state, new, capacity, page)
        got = shk.kv_pages_step(pool, torch.tensor(new, dtype=torch.int32, device=device), capacity)
        _compare(pool, got, state, want)


def test_replays(device):
    """A captured step goes on from where the pool is, and on another stream."""
    eager, captured = (shk.new_kv_pages(9, 40, 200, 16, device=device) for _ in range(2))
    new = torch.ones(9, dtype=torch.int32, device=device)
    side, graph = torch.cuda.Stream(device), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        got = shk.kv_pages_step(captured, new, 64)
    rng = random.Random(1)
    for n in range(12):
        new.copy_(torch.tensor([rng.choice([1, 7, 0, 3, -1]) for _ in range(9)], dtype=torch.int32))
        want = shk.kv_pages_step(eager, new, 64, stream=side if n % 2 else None)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert torch.equal(g, w)
        assert _state(eager) == _state(captured)


def test_refused_arguments(device):
    pool = shk.new_kv_pages(3, 4, 12, 16, device=device)
    new = torch.ones(3, dtype=torch.int32, device=device)
    for bad, capacity, match in ((new.long(), 8, "new_tokens"), (new[:2], 8, "new_tokens"), (new, -1, "capacity"),
                                 (new, 2.0, "capacity"), (new, True, "capacity"), (new, 2**31, "capacity")):
        with pytest.raises(ValueError, match=match):
            shk.kv_pages_step(pool, bad, capacity)
    with pytest.raises((RuntimeError, ValueError), match="CUDA/HIP|expected"):
        shk.kv_pages_step(pool, new.cpu(), 8)
    assert pool.lengths.tolist() == [0, 0, 0] and int(pool.free_count) == 12


def test_counts_past_any_capacity(device):
    """Numbers that no table holds are refused, their sum saturates, and what fits before them is served."""
    pool = shk.new_kv_pages(4, 4, 16, 16, device=device)
    new = torch.tensor([20, 2**31 - 1, 2**31 - 1, 5], dtype=torch.int32, device=device)
    step = shk.kv_pages_step(pool, new, 30)
    assert step.taken.tolist() == [20, 0, 0, 0] and pool.lengths.tolist() == [20, 0, 0, 0]
    assert step.slots[:20].tolist() == list(range(20)) and step.slots[20:].tolist() == [-1] * 10
    assert step.sequences.tolist() == [0] * 20 + [1] * 10
    assert step.starts.tolist() == [0, 20, 2**31 - 1, 2**31 - 1, 2**31 - 1]
