"""The gated mixture-of-experts layer for a few tokens, on the GPU, against
the layer in float64 within bounds derived from its arithmetic (_decode_ref)."""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

import amd_strix_halo_kernels as shk  # noqa: E402
from tests import _decode_ref as ref  # noqa: E402
from tests._util import spec_of, stable_seed  # noqa: E402

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _case(seed, tokens, experts, top, hidden, inner, *, group=0, layout="nn", dtype="bf16"):
    g = torch.Generator().manual_seed(seed)

    def weight(k, n):
        codes = ref.pack(torch.randint(-8, 8, (experts, n, k + k % 2), generator=g), 4)
        rows = (experts, n) if not group else (experts, -(-k // group), n)
        s = ((0.5 + torch.rand(rows, generator=g)) * 0.2 / math.sqrt(k)).bfloat16()
        return (codes if layout == "nt" else codes.transpose(1, 2).contiguous()), s

    up_gate, up_scale = weight(hidden, 2 * inner)
    down, down_scale = weight(inner, hidden)
    x = torch.randn((tokens, hidden), generator=g).to(DTYPES[dtype])
    ids = torch.stack([torch.randperm(experts, generator=g)[:top] for _ in range(tokens)]) if tokens else torch.zeros(
        (0, top), dtype=torch.int64)
    share = torch.rand((tokens, top), generator=g)
    return [x, up_gate, down, ids, share, up_scale, down_scale, group, layout]


def _run(case, device, **kw):
    x, up_gate, down, ids, share, up_scale, down_scale, group, layout = case
    d = [t.to(device) for t in (x, up_gate, down, ids, share, up_scale, down_scale)]
    return shk.moe_swiglu_int4(*d[:5], up_gate_scale=d[5], down_scale=d[6], scale=spec_of(group),
                               layout=shk.GemmLayout(layout), **kw)


def _check(got, case):
    want, bound = ref.moe(*case)
    off = (got.cpu().double() - want).abs()
    assert got.dtype == case[0].dtype and torch.isfinite(got).all()
    assert (off <= bound).all(), f"off by {float(off.max())}, {float((off - bound).max())} over its bound"


@pytest.mark.parametrize("layout", ["nn", "nt"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("group", [0, 32, 64, 128, 256])
@pytest.mark.parametrize("tokens,experts,top,hidden,inner", [(1, 4, 2, 256, 192), (5, 3, 1, 320, 64),
                                                             (16, 8, 3, 128, 320),
                                                             (17, 2, 2, 288, 96), (64, 4, 2, 160, 128)])
def test_layer(layout, dtype, group, tokens, experts, top, hidden, inner, device):
    print(f"case moe {layout} {dtype} group {group} {tokens} tokens {experts} experts {hidden}x{inner}", flush=True)
    case = _case(stable_seed("moe", layout, dtype, group, tokens, experts, top, hidden, inner), tokens, experts, top,
                 hidden, inner, group=group, layout=layout, dtype=dtype)
    _check(_run(case, device), case)


@pytest.mark.parametrize("layout", ["nn", "nt"])
@pytest.mark.parametrize("group", [0, 32, 128])
@pytest.mark.parametrize("hidden,inner", [(1, 1), (2, 3), (7, 65), (33, 31), (65, 130), (257, 127), (130, 66)])
def test_odd_sizes(layout, group, hidden, inner, device):
    """Rows of any length and alignment, an odd K whose last nibble is padding
    (here: any value)."""
    print(f"case moe odd {layout} group {group} {hidden}x{inner}", flush=True)
    for dtype in DTYPES:
        case = _case(stable_seed("odd", layout, group, hidden, inner, dtype), 3, 5, 2, hidden, inner, group=group,
                     layout=layout, dtype=dtype)
        _check(_run(case, device), case)


def _waves(grid, k, two_below):
    """Waves of a product's workgroups, which share K."""
    return 8 if grid <= 256 else 2 if k < two_below and grid > 1024 else 4


def _up(n, to):
    return -(-n // to) * to


@pytest.mark.parametrize("layout", ["nn", "nt"])
@pytest.mark.parametrize("group", [0, 64, 128, 256])
@pytest.mark.parametrize("tokens,top,experts,hidden,inner,waves", [
    (54, 1, 54, 808, 1290, (2, 4)), (33, 2, 60, 2600, 810, (4, 2)), (33, 2, 60, 4200, 1290, (4, 2)),
    (2, 2, 3, 3208, 200, (8, 8)), (2, 2, 3, 200, 3208, (8, 8))])
def test_several_pieces_of_k_a_wave(layout, group, tokens, top, experts, hidden, inner, waves, device):
    """Each number of waves, with three pieces of 128 or more for each in one of
    the two products, and an end that is none.  Most choices are padding."""
    print(f"case moe waves {waves} {layout} group {group} {hidden}x{inner}", flush=True)
    pairs = tokens * top
    most = min(pairs, experts)
    hit = most + (pairs - most) // 16
    grids = _up(-(-_up(inner, 128) // 64), 8) * hit, _up(-(-hidden // 128), 8) * hit
    assert waves == (_waves(grids[0], hidden, 4096 if group else 1536), _waves(grids[1], inner, 4096))
    dtype = "f16" if group == 64 else "bf16"
    case = _case(stable_seed("waves", layout, group, hidden, inner), tokens, 3, min(top, 2), hidden, inner, group=group,
                 layout=layout, dtype=dtype)
    g = torch.Generator().manual_seed(hidden + group)
    ids = torch.full((tokens, top), -1)
    ids.view(-1)[torch.randperm(pairs, generator=g)[:12]] = torch.randint(0, experts, (12,), generator=g)[:pairs]
    if pairs > 40:
        ids[:19, 0] = experts - 1  # two workgroups' rows
    case[3], case[4] = ids, torch.rand((tokens, top), generator=g)
    whole = [case[i][torch.arange(experts) % 3] for i in (1, 2, 5, 6)]
    x, share = case[0].to(device), case[4].to(device)
    got = shk.moe_swiglu_int4(x, whole[0].to(device), whole[1].to(device), ids.to(device), share,
                              up_gate_scale=whole[2].to(device), down_scale=whole[3].to(device), scale=spec_of(group),
                              layout=shk.GemmLayout(layout))
    # the three experts that all others repeat
    case[3] = torch.where(ids >= 0, ids % 3, ids)
    _check(got, case)


def test_refusals(device):
    x, up_gate, down, ids, share, up_scale, down_scale, _, _ = _case(3, 3, 4, 2, 64, 32)
    good = {n: t.to(device) for n, t in (("x", x), ("up_gate", up_gate), ("down", down), ("expert_ids", ids),
                                         ("expert_weights", share), ("up_gate_scale", up_scale),
                                         ("down_scale", down_scale))}
    for name, bad, match in (
        ("x", good["x"].float(), "x must have dtype"), ("x", good["x"][0], "x must have shape"),
        ("x", good["x"].t().contiguous().t(), "rows of x must be contiguous"), ("x", x, "CUDA/HIP"),
        ("up_gate", good["up_gate"][..., :63], "even number"),
        ("up_gate", good["up_gate"][:, :31], "up_gate must have shape"),
        ("up_gate", good["up_gate"][0], "up_gate must have shape"), ("down", good["down"][:3], "down must have shape"),
        ("down", good["down"].to(torch.int8), "down must have dtype"),
        ("down", good["down"].transpose(1, 2).contiguous().transpose(1, 2), "down must be contiguous"),
        ("up_gate_scale", good["up_gate_scale"].float(), "up_gate_scale must have dtype"),
        ("down_scale", good["down_scale"][:, :63], "down_scale must have shape"),
        ("expert_ids", good["expert_ids"][:2], "expert_ids must have shape"),
        ("expert_ids", good["expert_ids"].float(), "expert_ids must have dtype"),
        ("expert_ids", good["expert_ids"].t().contiguous().t(), "expert_ids must be contiguous"),
        ("expert_weights", good["expert_weights"].half(), "expert_weights must have dtype"),
        ("out", torch.empty_like(good["x"]).half(), "out must have dtype"),
        ("scale", spec_of(32), "up_gate_scale must have shape"),
        ("layout", shk.GemmLayout.NT, "up_gate must have shape|even number"),
    ):
        with pytest.raises((ValueError, RuntimeError), match=match):
            shk.moe_swiglu_int4(**{**good, name: bad})
    case = _case(3, 65, 4, 2, 64, 32)
    with pytest.raises(ValueError, match="up to 64 tokens"):
        _run(case, device)
    shk.moe_swiglu_int4(**good)


@pytest.mark.parametrize("layout", ["nn", "nt"])
def test_every_end_of_a_row(layout, device):
    """hidden takes every residue of eight values; rows past x's are not read."""
    for hidden in range(137, 153):
        case = _case(stable_seed("end", layout, hidden), 5, 3, 2, hidden, 70, layout=layout, dtype="f16")
        wide = torch.full((5, hidden + 3), math.nan, dtype=torch.float16)
        wide[:, :hidden] = case[0]
        case[0] = wide[:, :hidden]
        x = wide.to(device)[:, :hidden]
        d = [t.to(device) for t in case[1:7]]
        got = shk.moe_swiglu_int4(x, *d[:4], up_gate_scale=d[4], down_scale=d[5], layout=shk.GemmLayout(layout))
        _check(got, case)


def test_experts_with_many_rows_and_none(device):
    """All tokens through one expert of several, a token twice through the
    same one, and most experts idle."""
    case = _case(5, 64, 70, 2, 192, 64)
    case[3][:] = 69
    _check(_run(case, device), case)
    case = _case(6, 1, 1000, 1, 64, 64)
    case[3][:] = 999
    _check(_run(case, device), case)


def test_many_pairs(device):
    case = _case(7, 64, 40, 16, 64, 64)
    _check(_run(case, device), case)


def test_ids_outside_the_experts_add_nothing(device):
    case = _case(8, 6, 4, 2, 128, 64)
    case[3][0] = -1
    case[3][1, 0] = 4
    case[3][2, 1] = -(2**40)
    case[4][0] = math.nan  # a padded token's share is not read into anything
    got = _run(case, device)
    assert (got[0] == 0).all()
    case[4][0] = 0.0
    _check(got, case)
    case[3] = case[3].clamp(-1, 4).to(torch.int32)
    assert torch.equal(_run(case, device), got)


def test_zero_scales_and_strided_x(device):
    case = _case(9, 4, 3, 2, 256, 128, group=64)
    case[5][:, 1] = 0.0
    case[6][:, 0] = 0.0
    wide = torch.full((4, 600), math.nan, dtype=torch.bfloat16)
    wide[:, 33:33 + 256] = case[0]
    got = shk.moe_swiglu_int4(wide.to(device)[:, 33:33 + 256], *(t.to(device) for t in case[1:5]),
                              up_gate_scale=case[5].to(device), down_scale=case[6].to(device), scale=spec_of(64))
    _check(got, case)


def test_no_tokens_and_no_choices(device):
    case = _case(10, 0, 3, 2, 64, 64)
    assert _run(case, device).shape == (0, 64)
    case = _case(11, 3, 3, 0, 64, 64)
    case[3], case[4] = torch.zeros((3, 0), dtype=torch.int64), torch.zeros((3, 0))
    assert (_run(case, device) == 0).all()


def test_nan_stays_in_its_token(device):
    case = _case(12, 3, 2, 2, 128, 64)
    case[0][1, 5] = math.nan
    got = _run(case, device)
    assert torch.isnan(got[1]).all()
    case[0][1, 5] = 0.0
    want, bound = ref.moe(*case)
    off = (got.cpu().double() - want).abs()
    assert (off[[0, 2]] <= bound[[0, 2]]).all()


@pytest.mark.parametrize("which", [0, 4, 5, 6])
def test_no_gradient_is_said(which, device):
    for tokens in (3, 0):
        case = _case(17, tokens, 2, 2, 128, 64)
        d = [t.to(device) for t in case[:7]]
        d[which].requires_grad_()
        got = shk.moe_swiglu_int4(*d[:5], up_gate_scale=d[5], down_scale=d[6])
        if tokens:
            _check(got.detach(), case)
        with pytest.raises(RuntimeError, match="moe_swiglu_int4 has no gradient"):
            got.sum().backward()
        with torch.no_grad():
            assert not shk.moe_swiglu_int4(*d[:5], up_gate_scale=d[5], down_scale=d[6]).requires_grad


def test_repeated_calls_streams_and_out(device):
    case = _case(13, 20, 6, 2, 320, 192)
    first = _run(case, device)
    for _ in range(3):
        assert torch.equal(_run(case, device), first)
    stream, out = torch.cuda.Stream(device), torch.zeros_like(first)
    d = [t.to(device) for t in case[:7]]
    torch.cuda.synchronize()
    got = shk.moe_swiglu_int4(*d[:5], up_gate_scale=d[5], down_scale=d[6], out=out, stream=stream)
    stream.synchronize()
    assert got is out and torch.equal(out, first)


def test_other_stream_takes_no_block_of_this_one(device):
    case = _case(15, 20, 6, 2, 320, 192)
    want = _run(case, device)
    d = [t.to(device) for t in case[:7]]
    stream = torch.cuda.Stream(device)
    work = 4 * (20 * 2 * (256 + 320) + 3)
    torch.cuda.synchronize()
    blocks = [torch.full((n,), 7, dtype=torch.uint8, device=device) for n in (2 * want.numel(), work) for _ in range(4)]
    torch.cuda._sleep(20_000_000)
    copies = [b.clone() for b in blocks]
    del blocks
    got = shk.moe_swiglu_int4(*d[:5], up_gate_scale=d[5], down_scale=d[6], stream=stream)
    torch.cuda.synchronize()
    assert all((c == 7).all() for c in copies) and torch.equal(got, want)


def test_graph_of_the_layer(device):
    case = _case(14, 4, 6, 2, 320, 192)
    d = [t.to(device) for t in case[:7]]
    out = torch.zeros_like(d[0])

    def step():
        shk.moe_swiglu_int4(*d[:5], up_gate_scale=d[5], down_scale=d[6], out=out)

    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(device).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    g = torch.Generator().manual_seed(3)
    for _ in range(4):
        case[0] = torch.randn((4, 320), generator=g).bfloat16()
        case[3] = torch.stack([torch.randperm(6, generator=g)[:2] for _ in range(4)])
        d[0].copy_(case[0])
        d[3].copy_(case[3])
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        step()
        assert torch.equal(got, out)
        _check(got, case)


def test_weights_past_32_bits(device):
    """The last expert of a weight of more than 4 GiB."""
    hidden, inner = 512, 16384
    case = _case(15, 2, 1, 1, hidden, inner)
    experts = 2**32 // (hidden * inner) + 2
    up_gate = torch.zeros((experts, hidden // 2, 2 * inner), dtype=torch.uint8, device=device)
    assert up_gate.numel() > 2**32
    down = torch.zeros((experts, inner // 2, hidden), dtype=torch.uint8, device=device)
    up_scale = torch.zeros((experts, 2 * inner), dtype=torch.bfloat16, device=device)
    down_scale = torch.zeros((experts, hidden), dtype=torch.bfloat16, device=device)
    for whole, part in ((up_gate, case[1]), (down, case[2]), (up_scale, case[5]), (down_scale, case[6])):
        whole[-1] = part[0].to(device)
    ids = torch.full((2, 1), experts - 1, device=device)
    got = shk.moe_swiglu_int4(case[0].to(device), up_gate, down, ids, case[4].to(device), up_gate_scale=up_scale,
                              down_scale=down_scale)
    _check(got, case)
