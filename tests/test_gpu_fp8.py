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
