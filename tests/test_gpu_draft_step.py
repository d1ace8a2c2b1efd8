"""examples/draft_step.py: the operators of a step with drafted tokens one after
the other, each against its definition on what the step gave it, and a captured
step against the eager one."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

import amd_strix_halo_kernels as shk  # noqa: E402
from tests import _decode_ref, _fp8_ref, _step_ref  # noqa: E402

ROOT = Path(__file__).resolve().parents[1]
pytestmark = pytest.mark.gpu

SMALL = dict(hidden=256, heads=8, kv_heads=2, head_dim=64, vocab=500, batch=6, drafts=3, most=96, page=16)


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("draft_step", ROOT / "examples" / "draft_step.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _inputs(example, layer, g, device):
    last = torch.randint(0, 500, (layer.batch,), device=device, generator=g)
    drafted, draft = example.propose(layer, last, g)
    uniforms = torch.randint(0, 256, (layer.batch, 1 + layer.drafts), device=device, generator=g).float() / 256
    return torch.cat((last[:, None], drafted), dim=1), draft, uniforms


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("rotated", [64, 32])
def test_each_operator_of_a_step(example, device, bits, rotated):
    layer = example.DraftLayer(**SMALL, bits=bits, rotated=rotated, seed=bits, device=device)
    g = torch.Generator(device=device).manual_seed(bits)
    pool = {"page_table": layer.pages.page_table.tolist(), "lengths": [0] * 6, "owned": [0] * 6,
            "free": layer.pages.free_pages.tolist()}
    total = 0
    for n in range(7):
        tokens, draft, uniforms = _inputs(example, layer, g, device)
        out, kept, parts = layer.step(tokens, draft, uniforms)
        # pages
        want = _step_ref.step(pool, [4] * 6, 24, 16)
        for got, w in zip(parts["step"], want):
            assert got.tolist() == w
        assert parts["lengths"].tolist() == pool["lengths"]
        # drafts: what was kept, the next token, and the lengths without the others
        target = parts["target"].cpu()
        run = target.double().cumsum(-1)
        for b in range(6):
            exact = _step_ref.verified(target[b].tolist(), draft[b].tolist(), tokens[b, 1:].tolist(),
                                       uniforms[b].tolist(), 3)
            assert int(kept[b]) == exact[1] and out[b].tolist()[:exact[1]] == exact[0][:exact[1]]
            # the drawn token, unless the share falls within 2^-40 of a running sum
            assert out[b].tolist() == exact[0] or float((run[b] - float(uniforms[b, -1])).abs().min()) < 2.0**-40
        pool["lengths"] = [x - 3 + int(k) for x, k in zip(pool["lengths"], kept.tolist())]
        assert layer.pages.lengths.tolist() == pool["lengths"]
        total += int(kept.sum())
    assert 0 < total < 7 * 18
    # heads and attention of the last step
    p = {k: v.cpu() for k, v in parts.items() if k != "step"}
    positions = parts["step"].positions.cpu()
    frequencies, amplitude = shk.rotary_frequencies(rotated, scaling="yarn", factor=4.0, trained=2048)
    want, bound = _step_ref.rotated(p["qkv"][:, :8], layer.norms[0].cpu(), 1e-6, positions, frequencies, amplitude,
                                    False, torch.bfloat16)
    assert ((p["q"].reshape(24, 8, 64).double() - want).abs() <= bound).all()
    c = layer.cache
    cache = [t.cpu() for t in (c.key_codes, c.value_codes, c.key_scales, c.value_scales)]
    want = _decode_ref.attention(p["q"], cache, layer.pages.page_table.cpu(), p["lengths"])
    bound, _ = _decode_ref.attention_bounds(torch.bfloat16, 64, 96, *want)
    assert ((p["seen"].double() - want[0]).abs() <= bound).all()
    # the head's product
    codes, scales = (t.cpu() for t in shk.quantize_fp8(example._norm(parts["y"])))
    want, bound = _fp8_ref.product(codes, layer.head.codes.cpu(), scales, layer.head.scales.cpu(), torch.float32)
    assert ((p["logits"].double() - want).abs() <= bound).all()


def test_captured_steps(example, device):
    """Replays equal the eager steps, token for token."""
    eager, captured = (example.DraftLayer(**SMALL, device=device) for _ in range(2))
    g = torch.Generator(device=device).manual_seed(8)
    held = _inputs(example, captured, g, device)
    side, graph = torch.cuda.Stream(device), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        captured.step(*held)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        out, kept, _ = captured.step(*held)
    eager.step(*held)
    for n in range(6):
        fresh = _inputs(example, eager, g, device)
        for h, f in zip(held, fresh):
            h.copy_(f)
        want, count, _ = eager.step(*fresh)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(kept, count)
        for name in ("lengths", "owned", "free_count"):
            assert torch.equal(getattr(eager.pages, name), getattr(captured.pages, name))


def test_example_runs(example, device, capsys):
    example.main(steps=3, batch=4)
    assert "3 steps of 4 sequences" in capsys.readouterr().out
