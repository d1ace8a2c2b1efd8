"""Asking a product for the gradient of any of its operands raises, instead of leaving it out."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import amd_strix_halo_kernels as shk  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["a", "b", "a_scale", "b_scale"])
def test_every_operand(device, which):
    """Codes that torch's own cast made of a leaf ask for its gradient, too."""
    leaves = {"a": torch.randn((4, 256), device=device), "b": torch.randn((300, 256), device=device),
              "a_scale": torch.rand((4, 2), device=device), "b_scale": torch.rand((3, 2), device=device)}
    leaves[which].requires_grad_()
    codes = {n: leaves[n].to(torch.float8_e4m3fn) for n in ("a", "b")}
    out = shk.mm_fp8(codes["a"], codes["b"], a_scale=leaves["a_scale"], b_scale=leaves["b_scale"],
                     out_dtype=torch.float32)
    with pytest.raises(RuntimeError, match="mm_fp8 has no gradient"):
        out.sum().backward()
    with torch.no_grad():
        plain = shk.mm_fp8(codes["a"], codes["b"], a_scale=leaves["a_scale"], b_scale=leaves["b_scale"],
                           out_dtype=torch.float32)
    assert torch.equal(plain, out) and not plain.requires_grad
