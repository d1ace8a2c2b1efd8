"""examples/draft_step.py while the pool runs out: a sequence that gets no places sits the step out."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

from tests import _step_ref  # noqa: E402

ROOT = Path(__file__).resolve().parents[1]
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("draft_step", ROOT / "examples" / "draft_step.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("spare", [0, 2, 3])
def test_sequences_without_places_keep_their_tokens(example, device, spare):
    batch, drafts = 6, 3
    layer = example.DraftLayer(hidden=256, heads=8, kv_heads=2, head_dim=64, vocab=500, batch=batch, drafts=drafts,
                               most=96, page=16, device=device)
    layer.pages.free_count.fill_(batch + spare)  # a page each, and some of them a second one
    pool = {"page_table": layer.pages.page_table.tolist(), "lengths": [0] * batch, "owned": [0] * batch,
            "free": layer.pages.free_pages.tolist()[:batch + spare]}
    g = torch.Generator(device=device).manual_seed(spare)
    refused = 0
    for _ in range(16):
        last = torch.randint(0, 500, (batch,), device=device, generator=g)
        drafted, draft = example.propose(layer, last, g)
        uniforms = torch.randint(0, 256, (batch, 1 + drafts), device=device, generator=g).float() / 256
        out, kept, parts = layer.step(torch.cat((last[:, None], drafted), dim=1), draft, uniforms)
        taken = _step_ref.step(pool, [1 + drafts] * batch, batch * (1 + drafts), 16)[4]
        assert parts["step"].taken.tolist() == taken
        for b, (row, k) in enumerate(zip(out.tolist(), kept.tolist())):
            if taken[b]:
                pool["lengths"][b] -= drafts - k
                assert row[:k] == drafted[b, :k].tolist() and row[k] >= 0
            else:
                refused += 1
                assert k == 0 and row == [-1] * (1 + drafts)
        assert layer.pages.lengths.tolist() == pool["lengths"]
        assert layer.pages.owned.tolist() == pool["owned"]
    assert refused and min(pool["lengths"]) > 10
