"""Limits of the step's operators and of the fp8 products that the C ABI checks before it touches the device."""

from __future__ import annotations

import pytest

pytest.importorskip("torch")

from amd_strix_halo_kernels import fp8, kv_pages, native, rotary  # noqa: E402
from tests.test_step_host import MM, PLAN, ROTATE  # noqa: E402


@pytest.fixture(scope="module")
def lib():
    return native.load_dispatch_library()


def test_stacks_of_pages(lib):
    """A sum of pages that saturates at 2^31 - 1 has to be larger than any stack."""
    packed = kv_pages._PLAN.pack(*(PLAN | {"free_total": 2**31 - 1}).values())
    assert lib.amd_strix_halo_kernels_kv_plan(0, 0, packed) == 1
    assert b"2147483646 places" in lib.amd_strix_halo_kernels_last_error()


@pytest.mark.parametrize("k", [0, 1, 256])
@pytest.mark.parametrize("out_type", [0, 1, 2])
def test_products_hold_their_launch(lib, k, out_type):
    """Fewer than 2^32 work-items of 64 x 64 results where K has no values, of 64 x 128 where it has."""
    tiles = 0xFFFFFF
    columns = 64 if k == 0 else 128
    fits = MM | {"m": 64 * 4095, "n": columns * (tiles // 4095), "k": k, "out_type": out_type}
    for args, good in ((fits, True), (fits | {"n": fits["n"] + columns}, False)):
        args = args | {"out_stride": args["n"], "b_rows": 128, "a_scale_row": 1, "a_scale_block": 0, "b_scale_row": 1,
                       "b_scale_block": 0}
        nbytes = lib.amd_strix_halo_kernels_fp8_mm_workspace(fp8._MM.pack(*args.values()))
        assert (nbytes >= 0) == good, (k, args["n"])
        if not good:
            assert b"too many outputs" in lib.amd_strix_halo_kernels_last_error()


@pytest.mark.parametrize("bad", [{"qot": 0}, {"qoh": 0}, {"kot": 0}, {"koh": 0}, {"qoh": 63}, {"kot": 63}])
def test_rotated_rows_lie_apart(lib, bad):
    """Expanded outputs would be written by several rows at once."""
    assert lib.amd_strix_halo_kernels_rotate(0, 0, None, rotary._ROTATE.pack(*(ROTATE | bad).values())) == 1
    assert b"must not overlap" in lib.amd_strix_halo_kernels_last_error()


def test_strides_of_one_row_may_be_anything(lib):
    """One token's, or one head's: the call fails for its missing q alone."""
    one = ROTATE | {"tokens": 1, "heads": 1, "kv_heads": 1, "qot": 0, "qoh": 0, "kot": 0, "koh": 0, "q": 0}
    assert lib.amd_strix_halo_kernels_rotate(0, 0, None, rotary._ROTATE.pack(*one.values())) == 1
    assert b"non-null" in lib.amd_strix_halo_kernels_last_error()
