"""Plain 64-bit (float64, CPU) definitions of the decode operators, and the
error bounds that their tests use."""

from __future__ import annotations

import math

import torch



def half_ulp(dtype):
    """Unit roundoff: a value rounded once to dtype is off by this much of it."""
    return torch.finfo(dtype).eps / 2


def quantized_rows(x, bits):
    """(codes int64, scales bf16) of rows along the last axis: the scale is
    max|x| / Q rounded to 32 bits and then to bf16, a code the quotient
    rounded to 32 bits and then to a whole number, ties to even."""
    most = 7 if bits == 4 else 127
    x = x.double()
    top = x.abs().amax(dim=-1)
    scale = (top / most).float().bfloat16()
    wide = scale.double()[..., None]
    q = (x / wide).float().double().round().clamp(-most, most)
    fine = (wide > 0) & torch.isfinite(wide)
    return torch.where(fine, q, torch.zeros_like(q)).long(), scale


def pack(codes, bits):
    if bits == 8:
        return codes.to(torch.int8)
    nib = codes.to(torch.int16) & 15
    return (nib[..., 0::2] | (nib[..., 1::2] << 4)).to(torch.uint8)


def unpack(stored):
    if stored.dtype == torch.int8:
        return stored.long()
    u = stored.long()
    both = torch.stack((u & 15, u >> 4), dim=-1).flatten(-2)
    return torch.where(both > 7, both - 16, both)


def rows_of(codes, scales, pages, count):
    """float64 [kv_heads, count, head_dim] of the first `count` tokens of a
    list of pages."""
    page = scales.shape[2]
    at = torch.arange(count)
    idx = torch.as_tensor(pages, dtype=torch.long)[at // page]
    got = unpack(codes[idx, :, at % page]).double() * scales[idx, :, at % page].double()[..., None]
    return got.transpose(0, 1)


def attention(q, cache, table, lengths, prefix_pages=None, prefix_length=0, scale=None):
    """(out, lse, spread, scores, largest): float64 attention over the CPU tensors
    cache = (key_codes, value_codes, key_scales, value_scales); spread is the
    same sum over |v|, scores each row's largest scale * sum |q_i k_i|, and
    largest the largest |v| that a sequence sees."""
    kc, vc, ks, vs = cache
    batch, queries, heads, dim = q.shape
    kv_heads = ks.shape[1]
    ratio = heads // kv_heads
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    q = q.double()
    out = torch.zeros(q.shape, dtype=torch.float64)
    spread, lse = torch.zeros_like(out), torch.full(q.shape[:3], -math.inf, dtype=torch.float64)
    scores = torch.zeros(q.shape[:3], dtype=torch.float64)
    largest = torch.zeros((batch, 1, 1, 1), dtype=torch.float64)
    for b in range(batch):
        n = int(lengths[b])
        keys, values = (rows_of(c, s, table[b], n) for c, s in ((kc, ks), (vc, vs)))
        if prefix_length:
            keys = torch.cat((rows_of(kc, ks, prefix_pages, prefix_length), keys), dim=1)
            values = torch.cat((rows_of(vc, vs, prefix_pages, prefix_length), values), dim=1)
        largest[b] = values.abs().max() if values.numel() else 0.0
        for t in range(queries):
            seen = prefix_length + max(0, n - queries + t + 1)
            if not seen:
                continue
            qt = q[b, t].view(kv_heads, ratio, dim)
            s = qt @ keys[:, :seen].transpose(1, 2) * scale
            p = torch.softmax(s, dim=-1)
            out[b, t] = (p @ values[:, :seen]).flatten(0, 1)
            spread[b, t] = (p @ values[:, :seen].abs()).flatten(0, 1)
            lse[b, t] = torch.logsumexp(s, dim=-1).flatten()
            scores[b, t] = (qt.abs() @ keys[:, :seen].abs().transpose(1, 2) * abs(scale)).amax(dim=-1).flatten()
    return out, lse, spread, scores, largest


def attention_bounds(dtype, dim, tokens, out, lse, spread, scores, largest):
    """How far f32 attention with f16 probabilities may be off, per value.

    A score is a sum of dim exact products in f32, scaled three times:
    |ds| <= (dim + 8) 2^-24 times its sum of magnitudes, and the same again
    for q where its row spans more than f16's normal range.  A probability
    and the sum are off by at most 2 ds relative each, plus the f32 sums over
    the tokens.  Probabilities enter the product rounded once to f16 (2^-11),
    for f16 outputs as two terms (2^-21).  The output is rounded once.  What
    underflows: a probability below f16's normal range is off by up to 2^-25
    in units of 2^-13 of the largest value scale's power of two, so a token's
    term by 2^-37 of the largest |v|; f16 outputs by 2^-25.
    """
    ds = (dim + 8) * 2.0**-23 * scores
    inside = 4 * ds + tokens * 2.0**-23 + (2.0**-11 if dtype == torch.bfloat16 else 2.0**-21)
    under = tokens * 2.0**-37 * largest + 2.0**-25 * (dtype == torch.float16)
    return (half_ulp(dtype) * out.abs() + inside[..., None] * spread + under,
            ds + tokens * 2.0**-23 + 2.0**-22 * (lse.abs() + 1))


def moe(x, up_gate, down, ids, share, up_scale, down_scale, group, layout):
    """(y, bound) of the mixture-of-experts layer in float64 on CPU tensors.

    The bound follows the layer's arithmetic.  A product's terms are exact
    (activations to 2^-17 of themselves where they carry more than bf16's
    bits) and summed in f32 with codes offset by 24: off by at most
    K 2^-24 times the sum of |x| (|v| + 2 * 24 + 1) s.  h inherits that of up
    and gate (silu's slope is at most 1.1) and 2^-20 of its own; y that of h,
    a product's again, the f32 sum over the experts, and one rounding.
    """
    experts, inner = up_gate.shape[0], up_scale.shape[-1] // 2
    xd = x.double()
    y, bound = torch.zeros_like(xd), torch.zeros_like(xd)

    def weight(packed, scale, e, k):
        codes = unpack(packed[e] if layout == "nt" else packed[e].t().contiguous()).t()[:k].double()
        s = scale[e].double()
        s = s.repeat_interleave(group, dim=0)[:k] if group else s.expand(k, -1)
        return codes * s, (codes.abs() + 49.0) * s.abs(), s.abs()

    def product(v, k, e, packed, scale, extra):
        """v @ W, and its bound given that of v."""
        w, wide, s = weight(packed, scale, e, k)
        return v @ w, extra @ w.abs() + k * 2.0**-24 * (v.abs() @ wide) + 2.0**-17 * (v.abs() @ w.abs())

    for e in range(experts):
        for t, j in (ids == e).nonzero().tolist():
            v = xd[t:t + 1]
            ug, off = product(v, v.shape[1], e, up_gate, up_scale, torch.zeros_like(v))
            up, gate = ug[:, :inner], ug[:, inner:]
            sig = torch.sigmoid(gate)
            h = up * gate * sig
            off_h = off[:, :inner] * (gate * sig).abs() + 1.1 * up.abs() * off[:, inner:]
            off_h = off_h + 2 * off[:, :inner] * off[:, inner:]
            z, off_z = product(h, inner, e, down, down_scale, off_h + 2.0**-20 * h.abs())
            f = float(share[t, j])
            y[t] += f * z[0]
            bound[t] += abs(f) * (off_z[0] + ids.shape[1] * 2.0**-23 * z[0].abs())
    return y, bound + half_ulp(x.dtype) * y.abs() + (2.0**-25 if x.dtype == torch.float16 else 0.0)
