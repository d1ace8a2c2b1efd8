"""Verification of drafts against exact fractions."""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

import amd_strix_halo_kernels as shk  # noqa: E402
from tests import _step_ref as ref  # noqa: E402
from tests._util import stable_seed  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _coarse(g, *shape):
    """Probabilities that are whole multiples of 2^-10: every sum of them is exact,
    and shares fall on running sums."""
    return torch.randint(0, 40, shape, generator=g).float() * (torch.rand(shape, generator=g) < 0.4) / 1024


def _check(device, target, draft, tokens, uniforms, counts=None):
    dev = [None if t is None else t.to(device) for t in (target, draft, tokens, uniforms)]
    lengths = torch.arange(100, 100 + len(tokens), dtype=torch.int32, device=device)
    given = None if counts is None else counts.to(device)
    out, kept = shk.verify_draft(*dev, counts=given, lengths=lengths)
    for b in range(tokens.shape[0]):
        count = tokens.shape[1] if counts is None else int(counts[b])
        want = ref.verified(target[b].tolist(), None if draft is None else draft[b].tolist(), tokens[b].tolist(),
                            uniforms[b].tolist(), count)
        assert (out[b].tolist(), int(kept[b])) == want, b
        assert int(lengths[b]) == 100 + b - (count - want[1])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("greedy", [False, True])
@pytest.mark.parametrize("batch,drafts,vocab", [(1, 1, 1), (1, 5, 300), (9, 0, 77), (7, 3, 1000), (33, 5, 257),
                                                (2, 8, 5003), (3, 63, 40), (300, 2, 16), (5, 4, 2048), (4, 2, 20011)])
def test_coarse(device, batch, drafts, vocab, dtype, greedy):
    g = torch.Generator().manual_seed(stable_seed("coarse", batch, drafts, vocab, greedy))
    target = _coarse(g, batch, drafts + 1, vocab).to(dtype)
    draft = None if greedy else _coarse(g, batch, drafts, vocab).to(dtype)
    tokens = torch.randint(0, vocab, (batch, drafts), generator=g)
    if drafts and vocab > 1:  # drafts that are mostly kept
        likely = (target[:, :drafts] - (0 if greedy else draft)).argmax(dim=-1)
        tokens = torch.where(torch.rand((batch, drafts), generator=g) < 0.8, likely, tokens)
    uniforms = torch.randint(0, 256, (batch, drafts + 1), generator=g).float() / 256
    if greedy:
        uniforms[:, :drafts] /= 64
    _check(device, target, draft, tokens, uniforms)
    counts = torch.randint(0, drafts + 1, (batch,), generator=g).to(torch.int32)
    _check(device, target, draft, tokens.to(torch.int32), uniforms, counts)


@pytest.mark.parametrize("greedy", [False, True])
@pytest.mark.parametrize("vocab", [2047, 2048, 2049, 8192, 8193, 16384, 16385, 24001, 32767, 32768, 32769, 65537])
def test_sizes_around_a_workgroup(device, vocab, greedy):
    """Where another form of the kernel begins: shares at the start, on running sums, and at the end."""
    g = torch.Generator().manual_seed(stable_seed("around", vocab, greedy))
    target = _coarse(g, 5, 2, vocab)
    draft = None if greedy else _coarse(g, 5, 1, vocab)
    target[3, :, : vocab - 1] = 0.0  # one weight, the last
    target[3, :, vocab - 1] = 0.25
    target[4, :, 1:] = 0.0  # one, the first
    target[4, :, 0] = 0.25
    tokens = torch.randint(0, vocab, (5, 1), generator=g)
    uniforms = torch.tensor([[1.0, 0.0], [1.0, 0.5], [1.0, 255 / 256], [1.0, 0.75], [1.0, 0.75]])
    _check(device, target, draft, tokens, uniforms)


@pytest.mark.parametrize("batch,vocab", [(3, 131072), (70, 32001)])
def test_fine(device, batch, vocab):
    """Real probabilities: the drawn token's running sum passes the share, the one before does not, to
    2^-40 of the sum (the order of adding in 64 bits moves it by less)."""
    g = torch.Generator().manual_seed(batch)
    logits = 3 * torch.randn((batch, 3, vocab), generator=g)
    target = torch.softmax(logits, -1)
    draft = torch.softmax(logits[:, :2] + torch.randn((batch, 2, vocab), generator=g), -1)
    tokens = draft.argmax(dim=-1)
    uniforms = torch.rand((batch, 3), generator=g)
    out, kept = shk.verify_draft(target.to(device), draft.to(device), tokens.to(device), uniforms.to(device))
    out, kept = out.cpu(), kept.cpu().long()
    assert len(set(kept.tolist())) > 1 or batch < 10
    for b in range(batch):
        k = int(kept[b])
        for i in range(min(k + 1, 2)):
            t = tokens[b, i]
            assert (float(uniforms[b, i]) * float(draft[b, i, t]) < float(target[b, i, t])) == (i < k)
        weights = target[b, k].double() - (draft[b, k].double() if k < 2 else 0.0)
        run = weights.clamp(min=0).cumsum(0)
        token, share = int(out[b, k]), float(uniforms[b, 2]) * float(run[-1])
        slack = 2.0**-40 * float(run[-1])
        assert weights[token] > 0 and run[token] > share - slack
        assert token == 0 or run[token - 1] <= share + slack
        assert out[b].tolist() == tokens[b, :k].tolist() + [token] + [-1] * (2 - k)


def test_borders(device):
    """Equality keeps no draft and draws the next token; zero weights are never drawn."""
    target = torch.tensor([[[0.0, 0.25, 0.0, 0.25, 0.5, 0.0], [0.5, 0.0, 0.0, 0.0, 0.0, 0.5]]])
    draft = torch.tensor([[[0.0, 0.5, 0.0, 0.25, 0.25, 0.0]]])
    for token in range(6):
        for u in (0.0, 0.25, 0.5, 0.75, 1 - 2.0**-24):
            for v in (0.0, 0.25, 0.5, 0.75, 1 - 2.0**-24, 1.0, 2.0):
                t = torch.tensor([[token]])
                uniforms = torch.tensor([[u, v]])
                got, kept = shk.verify_draft(target.to(device), draft.to(device), t.to(device), uniforms.to(device))
                if v < 1.0:
                    want = ref.verified(target[0].tolist(), draft[0].tolist(), t[0].tolist(), uniforms[0].tolist(), 1)
                    assert (got[0].tolist(), int(kept)) == want
                else:  # a share that no running sum passes: the last token with a weight
                    assert got[0, int(kept)] == (5 if int(kept) else 4)


def test_rows_without_weights_and_bad_values(device):
    zero, nan, inf = [0.0] * 4, [math.nan, 0.5, -1.0, 0.25], [0.25] * 4
    same = [0.25, 0.25, 0.25, 0.25]
    target = torch.tensor([[zero, inf], [nan, inf], [same, inf], [same, zero], [same, same], [same, same]])
    draft = torch.tensor([[same], [[0.0, 0.25, 0.0, 0.25]], [same], [[0.125] * 4], [same], [same]])
    tokens = torch.tensor([[1], [2], [1], [1], [-1], [4]])
    uniforms = torch.tensor([[0.5, 0.5], [0.5, 0.5], [1.0, 0.5], [0.5, 0.5], [0.0, 0.75], [0.0, 0.25]])
    _check(device, target, draft, tokens, uniforms)
    out, kept = shk.verify_draft(target.to(device), draft.to(device), tokens.to(device), uniforms.to(device))
    assert out.tolist() == [[-1, -1], [1, -1], [2, -1], [1, -1], [3, -1], [1, -1]] and kept.tolist() == [0, 0, 0, 1, 0, 0]


def test_strides_stream_and_graph(device):
    g = torch.Generator().manual_seed(9)
    base = _coarse(g, 6, 7, 301).to(BF16)
    store = base.to(device)
    target, draft = store[::2, 1:5, 1:], store[1::2, 1:4, :300]  # rows off any alignment
    tokens = torch.randint(0, 300, (3, 3), generator=g).to(device)
    uniforms = (torch.randint(0, 256, (3, 4), generator=g).float() / 512).to(device)
    _check(device, base[::2, 1:5, 1:], base[1::2, 1:4, :300], tokens.cpu(), uniforms.cpu())
    want = shk.verify_draft(target, draft, tokens, uniforms)
    whole = shk.verify_draft(target.contiguous(), draft.contiguous(), tokens, uniforms)
    side = torch.cuda.Stream(device)
    torch.cuda.synchronize()
    other = shk.verify_draft(target, draft, tokens, uniforms, stream=side)
    side.synchronize()
    for got in (whole, other):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = shk.verify_draft(target, draft, tokens, uniforms)
    for n in range(4):
        uniforms.copy_(torch.randint(0, 256, (3, 4), generator=g).float() / 512)
        want = shk.verify_draft(target, draft, tokens, uniforms)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_no_sequences(device):
    out, kept = shk.verify_draft(torch.empty((0, 3, 10), device=device), None,
                                 torch.empty((0, 2), dtype=torch.int64, device=device), torch.empty((0, 3), device=device))
    assert out.shape == (0, 3) and kept.shape == (0,)


def test_kept_tokens_are_distributed_as_the_targets(device):
    """20000 sequences over five tokens: each first token's share within 5 standard deviations of the target's."""
    n = 20000
    p = torch.tensor([0.1, 0.4, 0.05, 0.25, 0.2])
    q = torch.tensor([0.3, 0.1, 0.2, 0.2, 0.2])
    g = torch.Generator().manual_seed(2)
    tokens = torch.multinomial(q, n, replacement=True, generator=g)[:, None]
    out, _ = shk.verify_draft(p.expand(n, 2, 5).to(device), q.expand(n, 1, 5).to(device), tokens.to(device),
                              torch.rand((n, 2), generator=g).to(device))
    share = torch.bincount(out[:, 0].cpu(), minlength=5).double() / n
    assert ((share - p).abs() <= 5 * (p * (1 - p) / n).sqrt()).all()


def test_refusals(device):
    target, draft = torch.zeros((2, 4, 50), device=device), torch.zeros((2, 3, 50), device=device)
    tokens, u = torch.zeros((2, 3), dtype=torch.int64, device=device), torch.zeros((2, 4), device=device)
    counts = torch.zeros(2, dtype=torch.int32, device=device)
    for args, kw, match in (((target.double(), None, tokens, u), {}, "target must have dtype"),
                            ((target[:, :3], None, tokens, u), {}, "target must have shape"),
                            ((target[..., ::2], None, tokens, u), {}, "target must be contiguous"),
                            ((target, draft.half(), tokens, u), {}, "draft must have shape"),
                            ((target, draft[..., :49], tokens, u), {}, "draft must have shape"),
                            ((target, draft, tokens.float(), u), {}, "tokens must have dtype"),
                            ((target, draft, tokens[0], u), {}, "tokens must be contiguous"),
                            ((target, draft, tokens, u[:, :3]), {}, "uniforms must be contiguous"),
                            ((target, draft, tokens, u.half()), {}, "uniforms must be contiguous"),
                            ((target, draft, tokens, u), {"counts": counts.long()}, "counts must be"),
                            ((target, draft, tokens, u), {"lengths": counts[:1]}, "lengths must be"),
                            ((torch.zeros((1, 65, 4), device=device), None, torch.zeros((1, 64), dtype=torch.int64, device=device),
                              torch.zeros((1, 65), device=device)), {}, "up to 63 drafts")):
        with pytest.raises(ValueError, match=match):
            shk.verify_draft(*args, **kw)
    with pytest.raises((RuntimeError, ValueError), match="CUDA/HIP|expected"):
        shk.verify_draft(target, draft, tokens.cpu(), u)


@pytest.mark.parametrize("vocab", [524288, 600001])
def test_vocabularies_of_several_steps_a_piece(device, vocab):
    """Weights that are whole multiples of 2^-20, so that the order of adding does not show."""
    g = torch.Generator().manual_seed(vocab)
    target = (torch.randint(0, 9, (2, 1, vocab), generator=g).float() * 2.0**-20)
    target[1, 0, : vocab - 3] = 0.0
    uniforms = torch.tensor([[0.734375], [0.5]])
    out, _ = shk.verify_draft(target.to(device), None, torch.empty((2, 0), dtype=torch.int64, device=device),
                              uniforms.to(device))
    run = target[:, 0].double().cumsum(-1)
    assert out[:, 0].tolist() == [int((run[b] <= float(uniforms[b, 0]) * float(run[b, -1])).sum()) for b in range(2)]
