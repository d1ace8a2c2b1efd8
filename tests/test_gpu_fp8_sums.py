"""What the sums of fp8 products hold: few rows and f32 results the f32 sums of exact products, 16-bit
results of tiles the products of each eight along K to 2^-13 of the largest one's power of two, cut towards 0."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import amd_strix_halo_kernels as shk  # noqa: E402
from tests import _fp8_ref as ref  # noqa: E402
from tests._util import stable_seed  # noqa: E402

pytestmark = pytest.mark.gpu

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _operands(*parts, m, n, k, large, one_sign, kind=E4M3):
    """One channel of every eight `large` times the others, of both signs or of one."""
    g = torch.Generator().manual_seed(stable_seed(*parts))

    def codes(rows):
        x = torch.randn((rows, k), generator=g)
        x = x.abs() if one_sign else x
        x[:, ::8] *= large
        return (x * (100.0 / large)).clamp(-448.0, 448.0).to(kind)

    b = torch.randn((n, k), generator=g)
    b = ((b.abs() if one_sign else b) * 8.0).to(kind)
    scales = [0.5 + torch.rand((rows, -(-k // 128)), generator=g) for rows in (m, n)]
    return codes(m), b, *scales


def _multiplied(device, a, b, sa, sb, out_dtype):
    return shk.mm_fp8(a.to(device), b.to(device), a_scale=sa.to(device), b_scale=sb.to(device), out_dtype=out_dtype)


def _within(got, want, bound, out_dtype):
    """Whether values lie within their bounds; from 65520 on (half a step above its largest value, 65504) f16
    rounds to an infinity, so a value that may be there may be one."""
    off = (got - want).abs()
    good = off <= bound
    if out_dtype == F16:
        good |= (want.abs() + bound >= 65520.0) & (got == torch.copysign(torch.full_like(want, torch.inf), want))
    assert bool(good.all()), (float((off / bound)[~good].max()), int((~good).sum()))


def _bounds(a, b, sa, sb, out_dtype):
    """The value, and how far f32 sums rounded once to out_dtype may be from it (_fp8_ref.product's terms without
    what the 8-bit unit cuts)."""
    want, wide = ref.product(a, b, sa, sb, F32)
    half = torch.finfo(out_dtype).eps / 2
    return want, wide + half * want.abs() + (2.0**-25 if out_dtype == F16 else 0.0)


SPREADS = [(large, one_sign) for large in (1.0, 100.0, 300.0) for one_sign in (False, True)]


# up to 16, 32 and 64 rows, and 16 to 64 columns a workgroup
@pytest.mark.parametrize("m,n,k", [(1, 300, 1024), (16, 4200, 300), (16, 9000, 256), (16, 13000, 200), (30, 600, 1000),
                                   (30, 5000, 384), (60, 500, 520)])
@pytest.mark.parametrize("out_dtype", [BF16, F16, F32])
@pytest.mark.parametrize("large,one_sign", SPREADS)
@pytest.mark.parametrize("gain", [1.0, 2.0**-9])  # the second keeps all results inside f16's range
def test_few_rows_hold_f32_sums(device, m, n, k, out_dtype, large, one_sign, gain):
    a, b, sa, sb = _operands("few", m, n, k, large, one_sign, m=m, n=n, k=k, large=large, one_sign=one_sign)
    args = (a, b, sa * gain, sb)
    got = _multiplied(device, *args, out_dtype).cpu().double()
    _within(got, *_bounds(*args, out_dtype), out_dtype)


@pytest.mark.parametrize("kind", [E4M3, E5M2])
@pytest.mark.parametrize("out_dtype", [BF16, F16])
def test_few_rows_are_f32_results_rounded(device, kind, out_dtype):
    """The same sums as those of an f32 result, bit for bit."""
    args = _operands("rounded", kind, out_dtype, m=16, n=700, k=1000, large=300.0, one_sign=True, kind=kind)
    assert torch.equal(_multiplied(device, *args, out_dtype), _multiplied(device, *args, F32).to(out_dtype))


# tiles of 64 x 64 by one and two groups of waves, of 64 x 128, 256 x 256, and 128 x 128 for f32 results
@pytest.mark.parametrize("m,n,k", [(100, 500, 1000), (700, 1900, 300), (1000, 3000, 300), (2500, 2700, 300)])
@pytest.mark.parametrize("large,one_sign", SPREADS)
@pytest.mark.parametrize("gain", [1.0, 2.0**-9])
def test_tiles(device, m, n, k, large, one_sign, gain):
    a, b, sa, sb = _operands("tiles", m, n, k, large, one_sign, m=m, n=n, k=k, large=large, one_sign=one_sign)
    sa = sa * gain
    rows = torch.arange(0, m, max(1, m // 50))
    for out_dtype in (BF16, F16, F32):
        got = _multiplied(device, a, b, sa, sb, out_dtype).cpu().double()[rows]
        part = (a[rows], b, sa[rows], sb)
        _within(got, *(_bounds(*part, F32) if out_dtype == F32 else ref.product(*part, out_dtype)), out_dtype)


# few rows, tiles of 64 x 64 whole and with K cut, of 64 x 128 and of 256 x 256
@pytest.mark.parametrize("m,n,k", [(5, 301, 300), (100, 503, 300), (65, 203, 3100), (1000, 3003, 200), (2500, 2703, 300)])
@pytest.mark.parametrize("out_dtype", [BF16, F16])
def test_a_nan_has_the_same_bits_in_every_column(device, m, n, k, out_dtype):
    a, b, sa, sb = _operands("nan", m, n, k, m=m, n=n, k=k, large=1.0, one_sign=False)
    sa.view(torch.int32)[3, 0] = 0x7FD23456
    got = _multiplied(device, a, b, sa * 2.0**-9, sb, out_dtype)
    assert got[3].isnan().all() and torch.isfinite(got[:3]).all() and torch.isfinite(got[4:]).all()
    assert got[3].view(torch.int16).unique().numel() == 1
