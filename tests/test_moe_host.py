"""Refusals of the mixture-of-experts layer's entry points, without a GPU."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import amd_strix_halo_kernels as shk  # noqa: E402
from amd_strix_halo_kernels import kernel_table as kt  # noqa: E402
from amd_strix_halo_kernels import moe, native  # noqa: E402

FAKE = 0x10000  # never dereferenced: every call below fails validation first


def test_needs_the_device():
    with pytest.raises(RuntimeError, match="CUDA/HIP"):
        shk.moe_swiglu_int4(torch.zeros((1, 64), dtype=torch.bfloat16), torch.zeros((2, 32, 128), dtype=torch.uint8),
                            torch.zeros((2, 32, 64), dtype=torch.uint8), torch.zeros((1, 1), dtype=torch.int64),
                            torch.ones((1, 1)), up_gate_scale=torch.ones((2, 128), dtype=torch.bfloat16),
                            down_scale=torch.ones((2, 64), dtype=torch.bfloat16))


@pytest.mark.parametrize("layout", ["tn", "tt"])
def test_refuses_layouts(layout):
    with pytest.raises(ValueError, match="unsupported MoE layout"):
        shk.moe_swiglu_int4(None, None, None, None, None, up_gate_scale=None, down_scale=None,
                            layout=shk.GemmLayout(layout))


@pytest.fixture(scope="module")
def lib():
    return native.load_dispatch_library()


def _args(**kw):
    f = {"x": FAKE, "x_stride": 64, "type": kt.SRC_BF16, "tokens": 2, "hidden": 64, "inner": 32, "experts": 4, "top": 2,
         "up_gate": FAKE, "up_gate_scale": FAKE, "down": FAKE, "down_scale": FAKE, "group": 0, "layout": kt.LAYOUT_NN,
         "ids": FAKE, "id_bytes": 8, "share": FAKE, "out": FAKE, "workspace": FAKE, "workspace_bytes": 1 << 20} | kw
    return moe._MOE.pack(*(v or 0 for v in f.values()))


@pytest.mark.parametrize("kw,match", [
    ({"type": kt.SRC_F32}, "float16 or bfloat16"), ({"layout": kt.LAYOUT_TN}, "NN and NT"),
    ({"group": 48}, "scale group"), ({"group": 512}, "scale group"), ({"tokens": 65}, "64 tokens"), ({"tokens": -1}, "64 tokens"),
    ({"top": 513}, "1024 (token, expert) pairs"), ({"experts": 0}, "1024 experts"), ({"experts": 1025}, "1024 experts"),
    ({"hidden": 1, "inner": 1, "experts": 1}, "at least 4 bytes"), ({"hidden": 0}, "hidden and inner"),
    ({"inner": 2**21}, "hidden and inner"), ({"id_bytes": 2}, "int32 or int64"),
    ({"x": None}, "non-null"), ({"down_scale": None}, "non-null"), ({"ids": None}, "non-null"),
    ({"share": FAKE + 2}, "aligned to their elements"), ({"x": FAKE + 1}, "aligned to their elements"),
    ({"workspace": None}, "workspace must hold"), ({"workspace_bytes": 3075}, "workspace must hold 3076 bytes"),
    ({"workspace": FAKE + 4}, "aligned to 16"),
])
def test_c_abi_refusals(lib, kw, match):
    assert lib.amd_strix_halo_kernels_moe(0, 0, _args(**kw)) == 1
    assert match in lib.amd_strix_halo_kernels_last_error().decode()


def test_c_abi_null_struct_and_no_tokens(lib):
    assert lib.amd_strix_halo_kernels_moe(0, 0, None) == 1
    assert lib.amd_strix_halo_kernels_moe_workspace(None) == -1
    assert lib.amd_strix_halo_kernels_moe(0, 0, _args(tokens=0)) == 0
    assert lib.amd_strix_halo_kernels_moe_workspace(_args()) == 3076
