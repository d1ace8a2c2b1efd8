"""Norm and rotation of query and key heads, against float64 and, for keys and
values that go into a cache, bit for bit against the two calls they replace."""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

import amd_strix_halo_kernels as shk  # noqa: E402
from tests import _step_ref as ref  # noqa: E402
from tests._util import stable_seed  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _case(*parts, tokens, heads, kv_heads, dim, dtype, first=0):
    g = torch.Generator().manual_seed(stable_seed(*parts))
    x = torch.randn((tokens, heads + 2 * kv_heads, dim), generator=g) * torch.exp(
        torch.randn((tokens, heads + 2 * kv_heads, 1), generator=g))
    positions = first + torch.randint(0, 5000, (tokens,), generator=g)
    weights = 0.5 + torch.rand((2, dim), generator=g)
    return x.to(dtype), positions, weights


def _check(got, x, weight, positions, frequencies, amplitude, interleaved, eps=1e-6):
    want, bound = ref.rotated(x, weight, eps, positions, frequencies, amplitude, interleaved, x.dtype)
    off = (got.cpu().double() - want).abs()
    assert got.dtype == x.dtype and bool((off <= bound).all()), float((off / bound).max())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [None, "own", "f32"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dim,rotated", [(64, 64), (128, 128), (128, 32), (256, 64), (80, 40), (96, 48), (192, 192),
                                         (2, 2), (6, 4), (10, 0), (250, 250), (36, 18), (128, 16)])
def test_heads(device, dtype, norm, interleaved, dim, rotated):
    x, positions, weights = _case("heads", dtype, norm, interleaved, dim, rotated, tokens=19, heads=6, kv_heads=2,
                                  dim=dim, dtype=dtype)
    frequencies = ref.half_turns(rotated // 2)
    rotary = shk.new_rotary(frequencies, amplitude=1.25, interleaved=interleaved, device=device)
    w = None if norm is None else weights.to(F32 if norm == "f32" else dtype)
    dev = x.to(device)
    q, k = shk.rotate_qk(dev[:, :6], dev[:, 6:8], positions.to(device), rotary,
                         q_weight=None if w is None else w[0].to(device),
                         k_weight=None if w is None else w[1].to(device))
    _check(q, x[:, :6], None if w is None else w[0], positions, frequencies, 1.25, interleaved)
    _check(k, x[:, 6:8], None if w is None else w[1], positions, frequencies, 1.25, interleaved)


@pytest.mark.parametrize("tokens,heads,kv_heads,dim", [(1, 1, 1, 128), (1, 32, 8, 128), (3, 1, 1, 64), (700, 32, 8, 128),
                                                       (2100, 5, 3, 64), (515, 64, 1, 256), (4000, 1, 1, 64),
                                                       (900, 8, 8, 192)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_sizes(device, tokens, heads, kv_heads, dim, interleaved):
    x, positions, w = _case("sizes", tokens, heads, kv_heads, dim, interleaved, tokens=tokens, heads=heads,
                            kv_heads=kv_heads, dim=dim, dtype=BF16)
    frequencies = ref.half_turns(dim // 2)
    rotary = shk.new_rotary(frequencies, interleaved=interleaved, device=device)
    dev, w = x.to(device), w.to(BF16)
    q, k = shk.rotate_qk(dev[:, :heads], dev[:, heads:heads + kv_heads], positions.to(device, torch.int32), rotary,
                         q_weight=w[0].to(device), k_weight=w[1].to(device))
    _check(q, x[:, :heads], w[0], positions, frequencies, 1.0, interleaved)
    _check(k, x[:, heads:heads + kv_heads], w[1], positions, frequencies, 1.0, interleaved)


@pytest.mark.parametrize("first", [-5000, 131072, 2**24 + 1, 2**31 - 6000, 2**40])
def test_far_positions(device, first):
    x, positions, _ = _case("far", first, tokens=40, heads=2, kv_heads=1, dim=64, dtype=F32, first=first)
    frequencies, amplitude = shk.rotary_frequencies(64, scaling="yarn", factor=8.0, trained=4096)
    rotary = shk.new_rotary(frequencies, amplitude=amplitude, device=device)
    dev = x.to(device)
    q, k = shk.rotate_qk(dev[:, :2], dev[:, 2:3], positions.to(device), rotary)
    _check(q, x[:, :2], None, positions, frequencies, amplitude, False)
    _check(k, x[:, 2:3], None, positions, frequencies, amplitude, False)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dim,tokens,heads,kv_heads", [(64, 70, 4, 2), (128, 9, 32, 8), (256, 33, 2, 1), (128, 1500, 8, 8)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_into_the_cache(device, bits, dtype, dim, tokens, heads, kv_heads, interleaved):
    x, positions, w = _case("cache", bits, dtype, dim, tokens, interleaved, tokens=tokens, heads=heads,
                            kv_heads=kv_heads, dim=dim, dtype=dtype)
    x[0, heads] = 0.0
    x[0, -1] = math.inf
    rotary = shk.new_rotary(ref.half_turns(dim // 4), interleaved=interleaved, device=device)
    dev, positions, w = x.to(device), positions.to(device), w.to(device)
    q, k, v = dev[:, :heads], dev[:, heads:heads + kv_heads], dev[:, heads + kv_heads:]
    pages = -(-tokens // 16) + 2
    slots = torch.randperm(pages * 16, generator=torch.Generator().manual_seed(1))[:tokens].to(device)
    if tokens > 2:
        slots[1], slots[2] = -1, pages * 16  # padding, and outside the cache
    one, two = (shk.new_kv_cache(pages, 16, kv_heads, dim, bits=bits, device=device) for _ in range(2))
    how = {"q_weight": w[0], "k_weight": w[1]}
    q1, k1 = shk.rotate_qk(q, k, positions, rotary, **how)
    shk.kv_cache_write(one, k1, v, slots)
    q2 = shk.rotate_qk(q, k, positions, rotary, cache=two, values=v, slots=slots.to(torch.int32), **how)
    assert torch.equal(q1, q2)
    for name in ("key_codes", "value_codes", "key_scales", "value_scales"):
        a, b = (getattr(c, name) for c in (one, two))
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), name


@pytest.mark.parametrize("offset", [0, 1, 4])
@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place_and_off_alignment(device, offset, interleaved):
    """Rows that start on 16 bytes, on 2 and on 8; results over the inputs."""
    x, positions, w = _case("place", offset, interleaved, tokens=50, heads=4, kv_heads=2, dim=64, dtype=BF16)
    buffer = torch.zeros((50, 9 * 64), dtype=BF16, device=device)
    dev = buffer[:, offset:offset + 6 * 64].view(50, 6, 64) if offset == 0 else buffer.as_strided(
        (50, 6, 64), (9 * 64, 64, 1), offset)
    dev.copy_(x[:, :6])
    frequencies = ref.half_turns(32)
    rotary = shk.new_rotary(frequencies, interleaved=interleaved, device=device)
    w = w.to(BF16)
    q, k = dev[:, :4], dev[:, 4:6]
    got = shk.rotate_qk(q, k, positions.to(device), rotary, q_weight=w[0].to(device), k_weight=w[1].to(device),
                        q_out=q, k_out=k)
    assert got[0] is q and got[1] is k
    _check(q, x[:, :4], w[0], positions, frequencies, 1.0, interleaved)
    _check(k, x[:, 4:6], w[1], positions, frequencies, 1.0, interleaved)
    buffer.as_strided((50, 6 * 64), (9 * 64, 1), offset).zero_()
    assert not buffer.any()


def test_rows_with_bad_values_stay_alone(device):
    x, positions, w = _case("bad", tokens=8, heads=4, kv_heads=4, dim=128, dtype=BF16)
    rotary = shk.new_rotary(ref.half_turns(64), device=device)
    how = {"q_weight": w[0].to(BF16).to(device), "k_weight": w[1].to(BF16).to(device)}
    clean = x.to(device)
    good = shk.rotate_qk(clean[:, :4], clean[:, 4:8], positions.to(device), rotary, **how)
    dirty = clean.clone()
    dirty[2, 1, 5], dirty[3, 6, 100] = math.nan, math.inf
    got = shk.rotate_qk(dirty[:, :4], dirty[:, 4:8], positions.to(device), rotary, **how)
    mask = torch.ones((8, 8), dtype=torch.bool)
    mask[2, 1] = mask[3, 6] = False
    for g, want, part in zip(got, good, (mask[:, :4], mask[:, 4:])):
        assert torch.equal(g[part.to(device)], want[part.to(device)])
    assert got[0][2, 1].isnan().all() and got[1][3, 2].isnan().any()


def test_no_tokens(device):
    rotary = shk.new_rotary(ref.half_turns(32), device=device)
    x = torch.empty((0, 3, 64), dtype=BF16, device=device)
    q, k = shk.rotate_qk(x[:, :2], x[:, 2:], torch.empty(0, dtype=torch.int64, device=device), rotary)
    assert q.shape == (0, 2, 64) and k.shape == (0, 1, 64)


def test_stream_graph_and_gradient(device):
    x, positions, w = _case("graph", tokens=20, heads=4, kv_heads=2, dim=64, dtype=BF16)
    rotary = shk.new_rotary(ref.half_turns(32), device=device)
    dev, positions = x.to(device), positions.to(device)
    want = shk.rotate_qk(dev[:, :4], dev[:, 4:6], positions, rotary)
    side = torch.cuda.Stream(device)
    torch.cuda.synchronize()
    got = shk.rotate_qk(dev[:, :4], dev[:, 4:6], positions, rotary, stream=side)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = shk.rotate_qk(dev[:, :4], dev[:, 4:6], positions, rotary)
    for i in range(4):
        dev.copy_(torch.roll(x, i, 0))
        positions += 1
        want = shk.rotate_qk(dev[:, :4], dev[:, 4:6], positions, rotary)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    q = dev[:, :4].clone().requires_grad_()
    out = shk.rotate_qk(q, dev[:, 4:6], positions, rotary)
    with pytest.raises(RuntimeError, match="rotate_qk has no gradient"):
        out[0].float().sum().backward()


def test_refusals(device):
    rotary = shk.new_rotary(ref.half_turns(32), device=device)
    x = torch.zeros((5, 6, 64), dtype=BF16, device=device)
    q, k, v = x[:, :4], x[:, 4:5], x[:, 5:]
    at = torch.arange(5, device=device)
    w = torch.ones(64, dtype=BF16, device=device)
    cache = shk.new_kv_cache(4, 16, 1, 64, device=device)
    into = {"cache": cache, "values": v, "slots": at}
    for args, kw, match in (
        ((q.double(), k.double(), at, rotary), {}, "q must have dtype"), ((q, k.half(), at, rotary), {}, "dtype of q"),
        ((q[0], k, at, rotary), {}, "q must have shape"), ((q, k[:4], at, rotary), {}, "k must have shape"),
        ((q, k[..., :32], at, rotary), {}, "k must have shape"),
        ((x.transpose(1, 2), k, at, rotary), {}, "contiguous along head_dim"),
        ((q[..., :32], k[..., :32], at, rotary), {}, "rotary turns 64"),
        ((q, k, at.float(), rotary), {}, "positions must have dtype"),
        ((q, k, at[:4], rotary), {}, "positions must be contiguous"),
        ((q, k, at, rotary), {"q_weight": w}, "both or neither"),
        ((q, k, at, rotary), {"q_weight": w, "k_weight": w.float()}, "both the same"),
        ((q, k, at, rotary), {"q_weight": w.half(), "k_weight": w.half()}, "must have dtype"),
        ((q, k, at, rotary), {"q_weight": w[:32], "k_weight": w[:32]}, "q_weight must be contiguous"),
        ((q, k, at, rotary), {"eps": -1.0}, "eps"), ((q, k, at, rotary), {"eps": math.nan}, "eps"),
        ((q, k, at, rotary), {"values": v}, "need a cache"), ((q, k, at, rotary), {"slots": at}, "need a cache"),
        ((q, k, at, rotary), {"q_out": q.float()}, "q_out must have dtype"),
        ((q, k, at, rotary), {"k_out": q}, "k_out must have shape"),
        ((q, k, at, rotary), into | {"k_out": k}, "no other result"),
        ((q, k, at, rotary), into | {"values": None}, "needs values and slots"),
        ((q, k, at, rotary), into | {"values": v.float()}, "values must have the dtype"),
        ((q, k, at, rotary), into | {"slots": at[:3]}, "slots must have shape"),
        ((q, x[:, 4:], at, rotary), into, "k must have shape"),
    ):
        with pytest.raises(ValueError, match=match):
            shk.rotate_qk(*args, **kw)
    with pytest.raises((RuntimeError, ValueError), match="CUDA/HIP|expected"):
        shk.rotate_qk(q, k, at.cpu(), rotary)


def test_offsets_past_32_bits(device):
    """Tokens 18 MB apart."""
    store = torch.zeros((300, 9_000_000), dtype=BF16, device=device)
    x = torch.randn((300, 3, 128), generator=torch.Generator().manual_seed(1)).to(BF16)
    far = store.as_strided((300, 3, 128), (9_000_000, 128, 1), 8_999_000)
    far.copy_(x)
    rotary = shk.new_rotary(ref.half_turns(64), device=device)
    at = torch.arange(300, device=device)
    near = x.to(device)
    want = shk.rotate_qk(near[:, :2], near[:, 2:], at, rotary)
    got = shk.rotate_qk(far[:, :2], far[:, 2:], at, rotary)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
