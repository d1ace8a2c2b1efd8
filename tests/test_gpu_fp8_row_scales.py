"""Large fp8 products where every row of b has its own scales, over a K of many blocks: every result against its
definition, and the same bits call after call."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import amd_strix_halo_kernels as shk  # noqa: E402
from tests import _fp8_ref as ref  # noqa: E402
from tests._util import stable_seed  # noqa: E402

pytestmark = pytest.mark.gpu

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
BF16, F16 = torch.bfloat16, torch.float16


# whole blocks, an odd and an even number of them, and an end
@pytest.mark.parametrize("m,n,k", [(2304, 2568, 5120), (2400, 2512, 5248), (2500, 2505, 5200)])
@pytest.mark.parametrize("out_dtype,b_kind", [(BF16, E4M3), (F16, E4M3), (BF16, E5M2)])
def test_every_result(device, m, n, k, out_dtype, b_kind):
    g = torch.Generator(device=device).manual_seed(stable_seed("row scales", m, n, k, out_dtype, b_kind))
    a = torch.randn((m, k), generator=g, device=device).to(E4M3)
    b = torch.randn((n, k), generator=g, device=device).to(b_kind)
    # from block to block far apart: results with another block's scales are far off
    sa, sb = (torch.exp2(2 * torch.randn((rows, -(-k // 128)), generator=g, device=device)) * 1e-3 for rows in (m, n))
    got = shk.mm_fp8(a, b, a_scale=sa, b_scale=sb, out_dtype=out_dtype)
    for at in range(0, m, 256):
        rows = slice(at, min(m, at + 256))
        want, bound = ref.product(a[rows], b, sa[rows], sb, out_dtype)
        off = (got[rows].double() - want).abs()
        assert bool((off <= bound).all()), (at, float((off / bound).max()), int((off > bound).sum()))
    for _ in range(10):
        assert torch.equal(shk.mm_fp8(a, b, a_scale=sa, b_scale=sb, out_dtype=out_dtype), got)
