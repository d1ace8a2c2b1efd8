"""examples/decode_step.py: the decode operators one after the other, each
against its 64-bit definition on what the step gave it, and a captured step
against the eager one."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

from tests import _decode_ref as ref  # noqa: E402

ROOT = Path(__file__).resolve().parents[1]
pytestmark = pytest.mark.gpu

SMALL = dict(hidden=256, heads=8, kv_heads=2, head_dim=64, experts=4, inner=96, top=2, batch=16, most=64, page=16)


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("decode_step", ROOT / "examples" / "decode_step.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("prefix", [0, 50])
def test_each_operator_of_a_step(example, device, bits, prefix):
    layer = example.DecoderLayer(**SMALL, bits=bits, prefix=prefix, seed=bits, device=device)
    g = torch.Generator().manual_seed(5)
    for n in range(1, 19):
        x = torch.randn((16, 256), generator=g).to(torch.bfloat16).to(device)
        y, parts = layer.step(x)
    c, p = layer.cache, {k: v.cpu() for k, v in parts.items()}
    assert y.shape == (16, 256) and torch.isfinite(y).all() and (layer.lengths == n).all()
    cache = [t.cpu() for t in (c.key_codes, c.value_codes, c.key_scales, c.value_scales)]
    want = ref.attention(p["q"][:, None], cache, layer.table.cpu(), layer.lengths.cpu(), layer.prefix_pages.cpu(),
                         prefix)
    bound, _ = ref.attention_bounds(torch.bfloat16, 64, n + prefix, *want)
    assert ((p["seen"].double() - want[0][:, 0]).abs() <= bound[:, 0]).all()
    want, bound = ref.moe(p["y"], layer.up_gate.cpu(), layer.down.cpu(), p["ids"], p["share"],
                          layer.up_gate_scale.cpu(), layer.down_scale.cpu(), 0, "nn")
    assert ((p["out"].double() - want).abs() <= bound).all()


def test_captured_steps(example, device):
    """Replays equal the eager steps on the same inputs, token for token."""
    eager = example.DecoderLayer(**SMALL, prefix=50, device=device)
    captured = example.DecoderLayer(**SMALL, prefix=50, device=device)
    g = torch.Generator().manual_seed(6)
    x = torch.zeros((16, 256), dtype=torch.bfloat16, device=device)
    side, graph = torch.cuda.Stream(device), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        captured.step(x)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        y, _ = captured.step(x)
    captured.lengths.zero_()
    for _ in range(6):
        x.copy_(torch.randn((16, 256), generator=g).to(torch.bfloat16))
        want, _ = eager.step(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
