"""8-bit floating-point products with a scale for each block of 128, and the
conversion that feeds them, against their 64-bit definitions."""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

import amd_strix_halo_kernels as shk  # noqa: E402
from tests import _fp8_ref as ref  # noqa: E402
from tests._util import stable_seed  # noqa: E402

pytestmark = pytest.mark.gpu

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _gen(*parts):
    return torch.Generator().manual_seed(stable_seed(*parts))


def _codes(g, rows, cols, kind):
    """Codes over the type's whole range, zeros and subnormal values among them."""
    x = torch.randn((rows, cols), generator=g) * torch.exp2(torch.randint(-9, 8, (rows, cols), generator=g).float())
    return x.clamp(-ref.LARGEST[kind], ref.LARGEST[kind]).to(kind)


def _scales(g, rows, cols):
    return torch.exp2(2 * torch.randn((rows, cols), generator=g)) * 1e-3


def _case(g, m, n, k, b_rows=128, a_kind=E4M3, b_kind=E4M3):
    a, b = _codes(g, m, k, a_kind), _codes(g, n, k, b_kind)
    return a, b, _scales(g, m, -(-k // 128)), _scales(g, -(-n // b_rows), -(-k // 128))


def _check(got, a, b, sa, sb):
    want, bound = ref.product(a, b, sa, sb, got.dtype)
    off = (got.double().cpu() - want).abs()
    assert bool((off <= bound).all()), (float((off / bound).max()), int((off > bound).sum()))


# every tile, its edges and its neighbours; K below, at and past a block
SIZES = [(1, 1, 1), (1, 64, 128), (1, 4097, 640), (5, 100, 300), (16, 1000, 2048), (17, 130, 129), (32, 640, 1024),
         (33, 257, 127), (64, 512, 4096), (65, 128, 256), (128, 128, 128), (200, 333, 1000), (257, 500, 144),
         (1, 7, 16384), (70, 1, 130), (40, 5000, 300), (20, 5000, 200), (16, 9000, 260), (64, 13000, 130), (70, 90, 5000),
         (100, 500, 4200)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("b_rows", [1, 128])
def test_product(device, m, n, k, b_rows):
    a, b, sa, sb = _case(_gen("product", m, n, k, b_rows), m, n, k, b_rows)
    got = shk.mm_fp8(a.to(device), b.to(device), a_scale=sa.to(device), b_scale=sb.to(device))
    assert got.dtype == BF16 and got.shape == (m, n)
    _check(got, a, b, sa, sb)


# 64 x 64 tiles by one group of waves, by two (an odd and an even number of blocks,
# with and without an end, K whole and in parts, the last of one block), and both
# sides of where few rows give way to tiles
GROUPS = [(700, 1900, 100), (700, 1900, 900), (65, 200, 129), (65, 200, 256), (65, 200, 300), (130, 70, 384), (66, 200, 640),
          (65, 200, 2944), (65, 200, 3100), (65, 200, 9324), (16, 600, 10240), (16, 600, 10300), (32, 600, 5120),
          (32, 600, 5200), (20, 8300, 2048), (20, 8300, 2100), (60, 300, 2048), (60, 300, 2060)]


@pytest.mark.parametrize("out_dtype", [BF16, F32])
@pytest.mark.parametrize("m,n,k", GROUPS)
def test_groups_of_waves(device, m, n, k, out_dtype):
    a, b, sa, sb = _case(_gen("groups", m, n, k), m, n, k, 1)
    dev = [t.to(device) for t in (a, b, sa, sb)]
    got = shk.mm_fp8(*dev[:2], a_scale=dev[2], b_scale=dev[3], out_dtype=out_dtype)
    rows = torch.arange(0, m, 1 if m < 100 else 7)
    _check(got[rows.to(device)], a[rows], b, sa[rows], sb)
    again = shk.mm_fp8(*dev[:2], a_scale=dev[2], b_scale=dev[3], out_dtype=out_dtype)
    assert torch.equal(got, again)


# tiles of 64 x 128, of 256 x 256 (K of no whole block, one, an odd and an even
# number, with and without an end), and the f32 results' own of 128 x 128
LARGE = [(1000, 3000, 200), (2500, 2700, 100), (2600, 2560, 128), (2500, 2505, 384), (2304, 2568, 300),
         (2400, 2512, 256), (4100, 1300, 777)]


@pytest.mark.parametrize("out_dtype", [BF16, F16, F32])
@pytest.mark.parametrize("b_rows", [1, 128])
@pytest.mark.parametrize("m,n,k", LARGE)
def test_large_tiles(device, m, n, k, b_rows, out_dtype):
    """Rows and columns of every tile and its edges: sampled rows against the definition, and all
    of them against the same rows multiplied few at a time."""
    a, b, sa, sb = _case(_gen("large", m, n, k, b_rows), m, n, k, b_rows)
    dev = [t.to(device) for t in (a, b, sa, sb)]
    got = shk.mm_fp8(*dev[:2], a_scale=dev[2], b_scale=dev[3], out_dtype=out_dtype)
    rows = torch.unique(torch.cat((torch.arange(0, m, 97), torch.tensor([0, 15, 16, 63, 64, 127, 128, 255, 256, m - 1]))))
    _check(got[rows.to(device)], a[rows], b, sa[rows], sb)
    wide = [shk.mm_fp8(dev[0][i:i + 32], dev[1], a_scale=dev[2][i:i + 32], b_scale=dev[3], out_dtype=F32)
            for i in range(0, m, 32)]
    off = (got.double() - torch.cat(wide).double()).abs().amax(dim=1).cpu()
    size = torch.cat(wide).double().abs().amax(dim=1).cpu()
    assert bool((off <= 0.02 * size + 1e-6).all())  # a misplaced row or value would be off by its size


def test_large_calls_repeat_their_bits(device):
    a, b, sa, sb = (t.to(device) for t in _case(_gen("overlap"), 2500, 2510, 640))
    first = shk.mm_fp8(a, b, a_scale=sa, b_scale=sb)
    for _ in range(3):
        assert torch.equal(shk.mm_fp8(a, b, a_scale=sa, b_scale=sb), first)


@pytest.mark.parametrize("a_kind,b_kind", [(E4M3, E5M2), (E5M2, E4M3), (E5M2, E5M2)])
@pytest.mark.parametrize("out_dtype", [BF16, F32])
@pytest.mark.parametrize("m,n,k", [(1000, 3000, 200), (2500, 2700, 300)])
def test_large_types(device, m, n, k, out_dtype, a_kind, b_kind):
    a, b, sa, sb = _case(_gen("large types", m, out_dtype, a_kind, b_kind), m, n, k, 128, a_kind, b_kind)
    got = shk.mm_fp8(a.to(device), b.to(device), a_scale=sa.to(device), b_scale=sb.to(device), out_dtype=out_dtype)
    rows = torch.arange(0, m, 61)
    _check(got[rows.to(device)], a[rows], b, sa[rows], sb)


@pytest.mark.parametrize("out_dtype", [BF16, F16, F32])
@pytest.mark.parametrize("a_kind,b_kind", [(E4M3, E4M3), (E4M3, E5M2), (E5M2, E4M3), (E5M2, E5M2)])
@pytest.mark.parametrize("m", [9, 130])
def test_types(device, out_dtype, a_kind, b_kind, m):
    g = _gen("types", out_dtype, a_kind, b_kind, m)
    a, b, sa, sb = _case(g, m, 200, 333, 1, a_kind, b_kind)
    sa = sa * (1e-3 if E5M2 in (a_kind, b_kind) else 1.0)
    got = shk.mm_fp8(a.to(device), b.to(device), a_scale=sa.to(device), b_scale=sb.to(device), out_dtype=out_dtype)
    _check(got, a, b, sa, sb)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("kind", [E4M3, E5M2])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 129), (128, 128), (130, 300), (257, 1040), (16, 4096)])
def test_quantize(device, rows, cols, kind, dtype):
    g = _gen("quantize", rows, cols, kind, dtype)
    x = (torch.randn((rows, cols), generator=g) * torch.exp2(3 * torch.randn((rows, 1), generator=g))).to(dtype)
    dev = x.to(device)
    for transpose in (False, True):
        for block_rows in (1, 128):
            want, scale = ref.quantized(x.t() if transpose else x, block_rows, kind)
            for given, turn in ((dev, transpose), (dev.t().contiguous().t(), transpose)):
                codes, got = shk.quantize_fp8(given, block_rows=block_rows, transpose=turn, dtype=kind)
                assert codes.dtype == kind and codes.shape == want.shape and got.shape == scale.shape
                assert torch.equal(got.cpu(), scale)
                assert torch.equal(codes.cpu().double(), want)


# ---------------------------------------------------------------------------
# Values that are no numbers, layouts, streams


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,cols", [(131075, 100), (70001, 203)])
def test_quantize_rows_in_pairs(device, rows, cols, dtype):
    """Many blocks are taken two rows at a time: the same codes and scales as those of parts of the rows."""
    x = torch.randn((rows, cols), generator=_gen("pairs", rows, cols, dtype)).to(dtype).to(device)
    codes, scales = shk.quantize_fp8(x)
    for at in range(0, rows, 40000):
        want, want_scales = shk.quantize_fp8(x[at : at + 40000])
        assert torch.equal(codes[at : at + 40000].view(torch.uint8), want.view(torch.uint8))
        assert torch.equal(scales[at : at + 40000], want_scales)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("block_rows,transpose", [(128, False), (128, True), (1, True)])
def test_quantize_many_tiles(device, block_rows, transpose, dtype):
    """Many tiles take another form than few: the same codes and scales as those of parts of the rows, blocks of
    zeros and with infinities and NaN among them."""
    x = torch.randn((3001, 3003), generator=_gen("tiles", block_rows, transpose, dtype)).to(dtype)
    x[256:384] = 0
    x[500, 700], x[2999, 3002], x[700, 128:256] = math.inf, math.nan, -math.inf
    x = x.to(device)
    codes, scales = shk.quantize_fp8(x, block_rows=block_rows, transpose=transpose)
    for at in range(0, 3001, 512):
        want, want_scales = shk.quantize_fp8(x[at : at + 512], block_rows=block_rows, transpose=transpose)
        got, got_scales = codes[at : at + 512], scales[at // 128 : at // 128 + 4]
        if transpose:
            got, got_scales = codes[:, at : at + 512], scales[:, at // 128 : at // 128 + 4]
        assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))
        assert torch.equal(got_scales.contiguous().view(torch.int32), want_scales.contiguous().view(torch.int32))


@pytest.mark.parametrize("kind", [E4M3, E5M2])
def test_quantize_bad_blocks(device, kind):
    """A block with an infinity or a NaN has that as its scale and zero codes; its neighbours do not see it;
    a block of zeros has scale 0; the smallest and largest magnitudes."""
    x = torch.randn((260, 300), generator=_gen("bad", kind))
    x[3, 10], x[140, 200], x[200, 299] = math.inf, math.nan, -math.inf
    x[5], x[7] = 0.0, 1e-42
    x[9, :128], x[9, 128:256] = 3e38, -3e38
    dev = x.to(device)
    for rows in (1, 128):
        for transpose in (False, True):
            want, scale = ref.quantized(x.t() if transpose else x, rows, kind)
            codes, got = shk.quantize_fp8(dev, block_rows=rows, transpose=transpose, dtype=kind)
            got = got.cpu()
            assert torch.equal(torch.isnan(got), torch.isnan(scale))
            assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(scale))
            assert torch.equal(codes.cpu().double(), want)


@pytest.mark.parametrize("m,out_dtype", [(3, BF16), (3, F32), (100, BF16), (100, F32), (2500, F16), (2500, F32)])
def test_nan_stays_in_its_row_and_column(device, m, out_dtype):
    n, k = 2700, 330
    a, b, sa, sb = _case(_gen("nan", m, out_dtype), m, n, k, 1)
    clean = shk.mm_fp8(a.to(device), b.to(device), a_scale=sa.to(device), b_scale=sb.to(device), out_dtype=out_dtype)
    a.view(torch.uint8)[1, 329] = 0x7F  # a NaN code, the last value of K
    sb[5, 1] = math.inf
    b.view(torch.uint8)[5, 128:256] = 0
    sa[2, 2] = math.nan
    got = shk.mm_fp8(a.to(device), b.to(device), a_scale=sa.to(device), b_scale=sb.to(device), out_dtype=out_dtype)
    assert got[1].isnan().all() and got[2].isnan().all() and got[:, 5].isnan().all()
    keep = torch.ones((m, n), dtype=torch.bool, device=device)
    keep[1] = keep[2] = False
    keep[:, 5] = False
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("m", [5, 40, 70, 1100])
@pytest.mark.parametrize("pitch,offset", [(352, 0), (352, 16), (333, 0), (339, 3), (350, 1)])
def test_operands_in_wider_rows(device, m, pitch, offset):
    """Rows with any pitch and start, and NaN codes behind and between them, which no product reads."""
    n, k = 1300, 330
    a, b, sa, sb = _case(_gen("wide rows", m, pitch, offset), m, n, k)

    def inside(t):
        buffer = torch.full((t.shape[0] * pitch + offset,), 0x7F, dtype=torch.uint8, device=device)
        view = buffer.as_strided((t.shape[0], k), (pitch, 1), offset).view(E4M3)
        view.copy_(t)
        return view

    got = shk.mm_fp8(inside(a), inside(b), a_scale=sa.to(device), b_scale=sb.to(device))
    plain = shk.mm_fp8(a.to(device), b.to(device), a_scale=sa.to(device), b_scale=sb.to(device))
    assert torch.equal(got, plain) and bool(torch.isfinite(got).all())


@pytest.mark.parametrize("m", [4, 90, 1500])
def test_scales_of_any_strides_and_out(device, m):
    n, k = 1410, 700
    a, b, sa, sb = (t.to(device) for t in _case(_gen("strides", m), m, n, k, 1))
    want = shk.mm_fp8(a, b, a_scale=sa, b_scale=sb)
    turned = [t.t().contiguous().t() for t in (sa, sb)]
    spaced = [torch.zeros((t.shape[0], 3 * t.shape[1]), device=device)[:, ::3].copy_(t) for t in (sa, sb)]
    for s in (turned, spaced):
        assert torch.equal(shk.mm_fp8(a, b, a_scale=s[0], b_scale=s[1]), want)
    one = torch.full((1, 1), 0.5, device=device)
    same = shk.mm_fp8(a, b, a_scale=one.expand(m, 6), b_scale=one.expand(n, 6))
    full = shk.mm_fp8(a, b, a_scale=one.expand(m, 6).contiguous(), b_scale=one.expand(n, 6).contiguous())
    assert torch.equal(same, full)
    store = torch.full((m, n + 7), 3.0, dtype=BF16, device=device)
    out = store[:, 3:n + 3]
    assert shk.mm_fp8(a, b, a_scale=sa, b_scale=sb, out=out) is out
    assert torch.equal(out, want) and bool((store[:, :3] == 3).all()) and bool((store[:, n + 3:] == 3).all())


def test_no_rows_no_columns_no_k(device):
    f = lambda *s: torch.zeros(s, device=device)  # noqa: E731
    c = lambda *s: f(*s).to(E4M3)  # noqa: E731
    assert shk.mm_fp8(c(0, 128), c(5, 128), a_scale=f(0, 1), b_scale=f(1, 1)).shape == (0, 5)
    assert shk.mm_fp8(c(4, 128), c(0, 128), a_scale=f(4, 1), b_scale=f(0, 1)).shape == (4, 0)
    for m in (4, 100, 2500):
        for dtype in (BF16, F32):
            got = shk.mm_fp8(c(m, 0), c(2600, 0), a_scale=f(m, 0), b_scale=f(21, 0), out_dtype=dtype)
            assert got.shape == (m, 2600) and not got.any()
    for shape in ((0, 5), (5, 0)):
        codes, scales = shk.quantize_fp8(torch.zeros(shape, device=device))
        assert codes.shape == shape and scales.shape == (shape[0], -(-shape[1] // 128))


def test_gradients_of_a_linear_layer(device):
    """y, dx and dw as one kernel's three products, against float64 on the quantized values, and against
    differences of sum(y * g)."""
    g = _gen("linear")
    t, k, n = 300, 264, 200
    x, w, dy = torch.randn((t, k), generator=g), torch.randn((n, k), generator=g), torch.randn((t, n), generator=g)
    q = lambda v, **kw: shk.quantize_fp8(v.to(device), **kw)  # noqa: E731

    def mm(a, b):
        return shk.mm_fp8(a[0], b[0], a_scale=a[1], b_scale=b[1], out_dtype=F32)

    def value(v, rows=1):
        codes, scale = (u.cpu() for u in v)
        return codes.double() * ref.spread(scale, rows, codes.shape)

    pairs = {"y": (q(x), q(w, block_rows=128)),
             "dx": (q(dy, dtype=E5M2), q(w, block_rows=128, transpose=True)),
             "dw": (q(dy, transpose=True, dtype=E5M2), q(x, transpose=True))}
    for name, (a, b) in pairs.items():
        rows = 128 if name != "dw" else 1
        _check(mm(a, b), a[0].cpu(), b[0].cpu(), a[1].cpu(), b[1].cpu())
        want = {"y": x @ w.t(), "dx": dy @ w, "dw": dy.t() @ x}[name].double()
        off = (value(a) @ value(b, rows).t() - want).norm() / want.norm()
        # independent roundings of at most half a step, e5m2's 2^-3 and e4m3's 2^-4 of a value, uniform
        # inside the step: under 2^-3 together
        assert off < 2.0**-3
    # differences: x + step is x with one code moved to its neighbour
    codes, scale = pairs["y"][0]
    moved = codes.clone()
    row, col = 17, 100
    bits = moved.view(torch.uint8)
    bits[row, col] = bits[row, col] + 1 if int(bits[row, col]) % 128 < 120 else bits[row, col] - 1
    step = (moved.float() - codes.float())[row, col].double() * scale[row, col // 128].double()
    weight = pairs["y"][1]
    before, after = mm((codes, scale), weight).double(), mm((moved, scale), weight).double()
    gy = dy.to(device).double()
    rise = ((after - before) * gy).sum() / step
    exact = (gy[row].cpu() * value(weight, 128)[:, col]).sum()
    # f32 products: 132 + 6 roundings of 2^-23 of each row's magnitudes, before and after
    size = (value(pairs["y"][0])[row].abs() @ value(weight, 128).abs().t() * gy[row].abs().cpu()).sum()
    assert abs(float(rise) - float(exact)) <= 2 * 138 * 2.0**-23 * float(size) / abs(float(step))


def test_streams_and_replays(device):
    """Two captured calls share nothing: replayed on two streams at once they give the eager results."""
    g = _gen("replay")
    sizes = [(100, 300, 4200), (70, 1000, 700), (5, 3000, 600), (2500, 2600, 300)]
    cases = [tuple(t.to(device) for t in _case(g, *s)) for s in sizes]

    def step():
        outs = []
        for a, b, sa, sb in cases:
            outs.append(shk.mm_fp8(a, b, a_scale=sa, b_scale=sb))
            codes, scales = shk.quantize_fp8(outs[-1])
            outs.append(shk.mm_fp8(codes, codes, a_scale=scales, b_scale=scales, out_dtype=F32)
                        if codes.shape[0] < 200 else codes.float())
        return outs

    want = step()
    streams, graphs, got = [torch.cuda.Stream(device) for _ in range(2)], [], []
    torch.cuda.synchronize()
    for s in streams:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got.append(step())
        graphs.append(graph)
    for n in range(4):
        for a, b, sa, sb in cases:
            sa.mul_(1.5)
        want = step()
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for outs in got:
            assert all(torch.equal(a, b) for a, b in zip(outs, want))
    side = streams[0]
    a, b, sa, sb = cases[0]
    other = shk.mm_fp8(a, b, a_scale=sa, b_scale=sb, stream=side)
    side.synchronize()
    assert torch.equal(other, want[0])


def test_refusals(device):
    c = torch.zeros((4, 300), device=device).to(E4M3)
    w = torch.zeros((200, 300), device=device).to(E4M3)
    sa, sb = torch.ones((4, 3), device=device), torch.ones((2, 3), device=device)
    ok = {"a_scale": sa, "b_scale": sb}
    for args, kw, match in (((c.float(), w), ok, "a must have dtype"), ((c, w.view(torch.uint8)), ok, "b must have dtype"),
                            ((c[:, :200], w), ok, "must have shapes"), ((c[0], w), ok, "must have shapes"),
                            ((c.t(), w[:, :4]), ok, "rows of a and b"),
                            ((c, w), ok | {"a_scale": sa[:3]}, "a_scale must have shape"),
                            ((c, w), ok | {"b_scale": sb[:1]}, "b_scale must have shape"),
                            ((c, w), ok | {"a_scale": sa.half()}, "a_scale must have dtype"),
                            ((c, w), ok | {"out_dtype": torch.int32}, "the result must have dtype"),
                            ((c, w), ok | {"out": torch.zeros((4, 199), device=device)}, "out must have shape"),
                            ((c, w), ok | {"out": torch.zeros((200, 4), device=device).t()}, "contiguous rows"),
                            ((c, w), ok | {"out": torch.zeros((4, 200), device=device), "out_dtype": BF16}, "out must")):
        with pytest.raises(ValueError, match=match):
            shk.mm_fp8(*args, **kw)
    x = torch.zeros((4, 300), device=device)
    for args, kw, match in (((x.double(),), {}, "x must have dtype"), ((x[0],), {}, "x must have shape"),
                            ((x[:, ::2],), {}, "contiguous along"), ((x,), {"block_rows": 2}, "block_rows"),
                            ((x,), {"dtype": torch.int8}, "float8")):
        with pytest.raises(ValueError, match=match):
            shk.quantize_fp8(*args, **kw)
    with pytest.raises((RuntimeError, ValueError), match="CUDA/HIP|expected"):
        shk.mm_fp8(c, w.cpu(), **ok)


def test_no_gradient_is_said(device):
    x = torch.randn((4, 128), device=device, requires_grad=True)
    codes, scales = shk.quantize_fp8(x)
    out = shk.mm_fp8(codes, codes, a_scale=scales, b_scale=scales, out_dtype=F32)
    with pytest.raises(RuntimeError, match="has no gradient"):
        out.sum().backward()


def test_offsets_past_32_bits(device):
    """Rows of a result and of an operand that start past 4 GiB."""
    m, n, k = 70000, 33000, 128
    g = torch.Generator(device=device).manual_seed(3)
    a = (torch.randn((m, k), generator=g, device=device)).to(E4M3)
    b = (torch.randn((n, k), generator=g, device=device)).to(E4M3)
    sa, sb = torch.rand((m, 1), generator=g, device=device), torch.rand((258, 1), generator=g, device=device)
    out = shk.mm_fp8(a, b, a_scale=sa, b_scale=sb)
    rows = torch.tensor([0, 40000, 65100, m - 1], device=device)
    _check(out[rows], a[rows].cpu(), b.cpu(), sa[rows].cpu(), sb.cpu())
    del out
    wide = torch.zeros((300, 16_000_000), dtype=torch.uint8, device=device)  # rows 16 MB apart
    far = wide[:, :k].view(E4M3)
    far.copy_(a[:300])
    got = shk.mm_fp8(far, b[:500], a_scale=sa[:300], b_scale=sb[:4])
    assert torch.equal(got, shk.mm_fp8(a[:300], b[:500], a_scale=sa[:300], b_scale=sb[:4]))
