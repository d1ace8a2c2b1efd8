"""Frequencies of a stretched context against the published method's steps, pair by pair, on the host."""

from __future__ import annotations

import math

import pytest

import amd_strix_halo_kernels as shk


def _published(rotated, base, factor, trained, fast, slow):
    """The method by its definition: a ramp over the indices of the pairs, from the one that turns `fast` times over
    the trained positions (rounded down, at least 0) to the one that turns `slow` times (rounded up, at most rotated
    - 1)."""
    def index(turns):
        return rotated * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))

    low, high = max(math.floor(index(fast)), 0), min(math.ceil(index(slow)), rotated - 1)
    high = high + 0.001 if high == low else high
    out = []
    for i in range(rotated // 2):
        extended = 1.0 / base ** (2 * i / rotated)
        stays = 1 - min(1.0, max(0.0, (i - low) / (high - low)))
        out.append(extended / factor * (1 - stays) + extended * stays)
    return out


@pytest.mark.parametrize("rotated", [8, 16, 32, 64, 80, 128, 256])
@pytest.mark.parametrize("trained", [2048, 4096, 8192, 32768, 65536, 131072])
@pytest.mark.parametrize("base", [1e4, 5e5])
def test_yarn_is_the_published_ramp(rotated, trained, base):
    for factor in (2.0, 8.0, 40.0):
        got, _ = shk.rotary_frequencies(rotated, base=base, scaling="yarn", factor=factor, trained=trained)
        want = _published(rotated, base, factor, trained, 32.0, 1.0)
        assert len(got) == len(want)
        for g, w in zip(got, want):
            assert math.isclose(g, w, rel_tol=1e-12)


@pytest.mark.parametrize("rotated,trained", [(16, 32768), (64, 131072), (128, 131072), (128, 65536)])
def test_yarn_slows_no_turning_pair_by_the_whole_factor(rotated, trained):
    """The last pair turns more than once over the trained positions: it is between both ends."""
    plain, _ = shk.rotary_frequencies(rotated)
    got, _ = shk.rotary_frequencies(rotated, scaling="yarn", factor=8.0, trained=trained)
    assert plain[-1] * trained / (2 * math.pi) > 1.0
    assert got[-1] > plain[-1] / 8 * 1.01
    assert all(f / 8 <= g <= f for f, g in zip(plain, got))


def test_yarn_amplitude_of_contexts_that_are_not_longer():
    for factor, want in ((0.5, 1.0), (1.0, 1.0), (4.0, 0.1 * math.log(4.0) + 1.0)):
        assert math.isclose(shk.rotary_frequencies(64, scaling="yarn", factor=factor, trained=4096)[1], want)
