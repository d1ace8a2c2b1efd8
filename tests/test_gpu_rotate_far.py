"""How exactly a far position turns: cosines and sines against rational arithmetic and 60 digits of pi."""

from __future__ import annotations

import math
from fractions import Fraction

import pytest

torch = pytest.importorskip("torch")

import amd_strix_halo_kernels as shk  # noqa: E402

pytestmark = pytest.mark.gpu

PI = Fraction(3141592653589793238462643383279502884197169399375105820974944, 10**60)


@pytest.mark.parametrize("scaling", ["none", "yarn"])
def test_angles_of_far_positions(device, scaling):
    """The turns' rounding to 64 bits and the product's lose 2^-53 of the whole angle each; what is left of it is
    rounded to 32 bits, and cosine, sine and their product with 1 add at most 9 roundings of 2^-24 more."""
    frequencies, _ = shk.rotary_frequencies(64, scaling=scaling, factor=8.0, trained=4096)
    rotary = shk.new_rotary(frequencies, device=device)
    positions = [0, 1, -1, 12345, 10**6 + 3, 10**8 - 1, -(10**8) + 7, 2**31 - 1, 2**40 + 12345, 2**53 - 1]
    x = torch.zeros((len(positions), 2, 64), device=device)
    x[..., :32] = 1.0
    q, _ = shk.rotate_qk(x[:, :1], x[:, 1:], torch.tensor(positions, device=device), rotary)
    q = q.cpu().double()[:, 0]
    for t, position in enumerate(positions):
        for i, f in enumerate(frequencies):
            angle = Fraction(position) * Fraction(f)
            left = float(angle - 2 * PI * round(angle / (2 * PI)))
            bound = 10 * 2.0**-24 + abs(float(angle)) * 2.0**-52 * 1.001
            assert abs(float(q[t, i]) - math.cos(left)) <= bound, (position, i)
            assert abs(float(q[t, i + 32]) - math.sin(left)) <= bound, (position, i)
