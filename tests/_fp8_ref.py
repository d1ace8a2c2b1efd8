"""Plain 64-bit (float64, CPU) definitions of the 8-bit floating-point products
and of the conversion, and the error bounds that their tests use."""

from __future__ import annotations

import torch

LARGEST = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}
# mantissa bits, exponent of the smallest normal value
FORMAT = {torch.float8_e4m3fn: (3, -6), torch.float8_e5m2: (2, -14)}


def rounded(y, kind):
    """float64 y, |y| at most the largest value, to the nearest value of kind, ties to even."""
    bits, least = FORMAT[kind]
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0**-100))).clamp(min=least) - bits)
    return torch.round(y / step) * step


def quantized(x, rows, kind):
    """(code values float64, scales float32) of x in blocks of rows x 128."""
    x = x.double()
    r, c = x.shape
    pad = torch.nn.functional.pad(x, (0, -c % 128, 0, -r % rows))
    pad = pad.view(-1, rows, -(-c // 128), 128)
    top = pad.abs().amax(dim=(1, 3))  # a NaN stays
    scale = (top / LARGEST[kind]).float()
    wide = scale.double()[:, None, :, None].expand(pad.shape)
    fine = (wide > 0) & torch.isfinite(wide)
    q = torch.where(fine, pad / torch.where(fine, wide, 1.0), 0.0).float().double()
    codes = rounded(q.clamp(-LARGEST[kind], LARGEST[kind]), kind)
    return codes.reshape(-1, -(-c // 128) * 128)[:r, :c], scale


def spread(scale, rows, shape):
    """One scale for each value of `shape`."""
    return scale.double().repeat_interleave(rows, 0)[: shape[0]].repeat_interleave(128, 1)[:, : shape[1]]


def largest_of_eights(x, y):
    """For each result, the sum over the eights along K of their largest |product|."""
    k = -x.shape[1] % 8
    x = torch.nn.functional.pad(x.abs(), (0, k)).view(x.shape[0], -1, 8)
    y = torch.nn.functional.pad(y.abs(), (0, k)).view(y.shape[0], -1, 8)
    return torch.stack([(row * y).amax(dim=-1).sum(dim=-1) for row in x])


def product(a, b, a_scale, b_scale, out_dtype):
    """(out, bound) of code tensors a [M, K] and b [N, K] and their scales.

    The products of a block's codes are exact; the matrix unit adds 128 of them
    in f32 (at most 2^-23 of the magnitudes each).  For results of 16 bits it
    first cuts the products of each eight along K at 2^-13 of the largest one's
    power of two, which seven of them can lose.  The scales' product is rounded
    once (2^-24), and each block's term joins the f32 sum with one rounding, as
    the parts of a split K do.  The result is rounded once to its type, f16 also
    below its normal range (2^-25)."""
    a, b = a.double(), b.double()
    blocks = a_scale.shape[1]
    x = a * spread(a_scale, 1, a.shape)
    y = b * spread(b_scale, 1 if b_scale.shape[0] == b.shape[0] else 128, b.shape)
    out = x @ y.t()
    bound = (130 + 2 * blocks) * 2.0**-23 * (x.abs() @ y.abs().t())
    if out_dtype != torch.float32:
        bound = bound + 7 * 2.0**-13 * largest_of_eights(x, y)
    half = torch.finfo(out_dtype).eps / 2
    return out, bound + half * out.abs() + (2.0**-25 if out_dtype == torch.float16 else 2.0**-126)
