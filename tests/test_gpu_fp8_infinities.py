"""Infinities that e5m2 codes can hold, through every product kernel."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import amd_strix_halo_kernels as shk  # noqa: E402
from tests._util import stable_seed  # noqa: E402

pytestmark = pytest.mark.gpu

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2


@pytest.mark.parametrize("m,n,k", [(5, 301, 300), (100, 503, 300), (1000, 3003, 200), (2500, 2703, 300)])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("b_kind", [E4M3, E5M2])
def test_infinite_codes(device, m, n, k, out_dtype, b_kind):
    """An infinity times a number is an infinity, times 0 or against one of the other sign it is no number."""
    g = torch.Generator().manual_seed(stable_seed("infinite", m, n, k))
    a = torch.randn((m, k), generator=g).to(E5M2)
    b = (0.5 + torch.rand((n, k), generator=g)).to(b_kind)
    a[1, 7], a[2, k - 1], a[3, 5], a[3, 150] = torch.inf, -torch.inf, torch.inf, -torch.inf
    b[4, 7] = 0.0
    sa, sb = torch.full((m, -(-k // 128)), 0.25), torch.full((-(-n // 128), -(-k // 128)), 0.5)
    out = shk.mm_fp8(a.to(device), b.to(device), a_scale=sa.to(device), b_scale=sb.to(device), out_dtype=out_dtype).cpu()
    others = torch.arange(n) != 4
    assert bool((out[1, others] == torch.inf).all()) and bool(out[1, 4].isnan())
    assert bool((out[2] == -torch.inf).all()) and bool(out[3].isnan().all())
    assert bool(torch.isfinite(out[0]).all()) and bool(torch.isfinite(out[4:]).all())
