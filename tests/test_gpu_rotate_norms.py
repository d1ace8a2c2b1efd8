"""Norms of heads whose squares leave the range of 32 bits."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import amd_strix_halo_kernels as shk  # noqa: E402
from tests import _step_ref as ref  # noqa: E402
from tests._util import stable_seed  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


# whole vectors of both pair orders, and heads that are taken value by value
@pytest.mark.parametrize("dim,rotated,interleaved", [(128, 128, False), (64, 32, False), (256, 64, True), (80, 40, False),
                                                     (10, 4, True)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("eps", [0.0, 1e-42, 1e-35, 1e-6])
def test_tiny_and_huge_heads(device, dim, rotated, interleaved, dtype, eps):
    """Heads from 2^-120 to 2^120, among them those whose squares are subnormal, vanish or overflow."""
    g = torch.Generator().manual_seed(stable_seed("tiny", dim, rotated, dtype, eps))
    powers = torch.tensor([-120, -100, -80, -74, -70, -66, -64, -63, -62, -50, -20, 0, 40, 60, 62, 63, 64, 65, 80, 120])
    x = torch.randn((powers.numel(), 3, dim), generator=g) * torch.exp2(powers.float())[:, None, None]
    x = x.to(dtype)
    w = 0.5 + torch.rand((2, dim), generator=g)
    frequencies = ref.half_turns(rotated // 2)
    rotary = shk.new_rotary(frequencies, interleaved=interleaved, device=device)
    positions = torch.arange(powers.numel()) * 7
    dev = x.to(device)
    got = shk.rotate_qk(dev[:, :2], dev[:, 2:], positions.to(device), rotary, eps=eps, q_weight=w[0].to(device),
                        k_weight=w[1].to(device))
    # the given eps is rounded to 32 bits, below 2^-126 in steps of 2^-149
    eps = float(torch.tensor(eps, dtype=F32))
    for out, part, weight in ((got[0], x[:, :2], w[0]), (got[1], x[:, 2:], w[1])):
        want, bound = ref.rotated(part, weight, eps, positions, frequencies, 1.0, interleaved, dtype)
        off = (out.cpu().double() - want).abs()
        assert bool((off <= bound).all()), powers[(off > bound).flatten(1).any(1)].tolist()


@pytest.mark.parametrize("dim", [128, 10])
def test_rows_of_zeros(device, dim):
    """0 / sqrt(0 + eps) is 0 for an eps above 0, and no number for one of 0, here and by the definition."""
    rotary = shk.new_rotary(ref.half_turns(2), device=device)
    x, at, w = (torch.zeros((2, 3, dim), device=device), torch.arange(2, device=device),
                torch.ones(dim, device=device))
    for eps in (1e-6, 1e-35, 1e-42):
        for out in shk.rotate_qk(x[:, :2], x[:, 2:], at, rotary, eps=eps, q_weight=w, k_weight=w):
            assert not out.any()
    for out in shk.rotate_qk(x[:, :2], x[:, 2:], at, rotary, eps=0.0, q_weight=w, k_weight=w):
        assert out.isnan().all()


def test_infinities_and_nan_are_as_before(device):
    """An infinite value makes itself no number and the others 0, a NaN all of them."""
    rotary = shk.new_rotary([], device=device)
    x = torch.ones((2, 2, 64), device=device)
    x[0, 0, 5], x[1, 1, 7] = torch.inf, torch.nan
    w = torch.ones(64, device=device)
    q, k = shk.rotate_qk(x[:, :1], x[:, 1:], torch.arange(2, device=device), rotary, q_weight=w, k_weight=w)
    assert q[0, 0, 5].isnan() and not q[0, 0, :5].any() and not q[0, 0, 6:].any()
    assert k[1].isnan().all() and torch.isfinite(q[1]).all() and torch.isfinite(k[0]).all()
