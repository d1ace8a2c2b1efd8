"""Limits of the step's operators and of the fp8 products that the C ABI checks before it touches the device."""

from __future__ import annotations

import pytest

pytest.importorskip("torch")

from amd_strix_halo_kernels import kv_pages, native  # noqa: E402
from tests.test_step_host import PLAN  # noqa: E402


@pytest.fixture(scope="module")
def lib():
    return native.load_dispatch_library()


def test_stacks_of_pages(lib):
    """A sum of pages that saturates at 2^31 - 1 has to be larger than any stack."""
    packed = kv_pages._PLAN.pack(*(PLAN | {"free_total": 2**31 - 1}).values())
    assert lib.amd_strix_halo_kernels_kv_plan(0, 0, packed) == 1
    assert b"2147483646 places" in lib.amd_strix_halo_kernels_last_error()
