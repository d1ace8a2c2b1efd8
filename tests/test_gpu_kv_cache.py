"""The quantized key/value cache and the attention over it, on the GPU.

kv_cache_write and kv_cache_read are compared bit for bit with their 64-bit
definition; kv_cache_attention with float64 attention over the same cached
values, within bounds derived from its arithmetic (_decode_ref).  Everything
that no token has been written to holds NaN scales, so a read of masked
places shows.
"""

from __future__ import annotations

import copy
import math

import pytest

torch = pytest.importorskip("torch")

import amd_strix_halo_kernels as shk  # noqa: E402
from tests import _decode_ref as ref  # noqa: E402
from tests._util import stable_seed  # noqa: E402

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _cpu(cache):
    return tuple(t.cpu() for t in (cache.key_codes, cache.value_codes, cache.key_scales, cache.value_scales))


def _rows(seed, tokens, heads, dim, dtype):
    g = torch.Generator().manual_seed(seed)
    size = torch.exp(3 * torch.randn((2, tokens, heads, 1), generator=g))
    return (torch.randn((2, tokens, heads, dim), generator=g) * size).to(dtype)


def _same_bits(got, want):
    return got.dtype == want.dtype and torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(
        torch.nan_to_num(got), torch.nan_to_num(want))


# ---------------------------------------------------------------------------
# Writing and reading


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("tokens,heads,page", [(1, 1, 16), (7, 3, 16), (130, 2, 64), (1025, 8, 128)])
def test_write_then_read(dtype, bits, dim, tokens, heads, page, device):
    print(f"case write {dtype} int{bits} {tokens}x{heads}x{dim} page {page}", flush=True)
    seed = stable_seed("kv", dtype, bits, dim, tokens, heads, page)
    x = _rows(seed, tokens, heads, dim, DTYPES[dtype])
    x[0, 0, 0] = 0.0  # a row of zeros
    pages = -(-tokens // page) + 2
    cache = shk.new_kv_cache(pages, page, heads, dim, bits=bits, device=device)
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(seed))[:tokens]
    xd = x.to(device)
    shk.kv_cache_write(cache, xd[0], xd[1], slots.to(device))
    for part, rows in (("key", x[0]), ("value", x[1])):
        codes, scales = ref.quantized_rows(rows, bits)
        got_codes = getattr(cache, f"{part}_codes").cpu()
        got_scales = getattr(cache, f"{part}_scales").cpu()
        want_codes, want_scales = torch.zeros_like(got_codes), torch.zeros_like(got_scales)
        want_codes[slots // page, :, slots % page] = ref.pack(codes, bits)
        want_scales[slots // page, :, slots % page] = scales
        assert torch.equal(got_codes, want_codes) and torch.equal(got_scales, want_scales), part
    for out in DTYPES.values():
        got = shk.kv_cache_read(cache, slots.to(device).to(torch.int32), dtype=out)
        for rows, values in zip(x, got):
            codes, scales = ref.quantized_rows(rows, bits)
            want = (codes.double() * scales.double()[..., None]).float().to(out)
            assert values.shape == want.shape and _same_bits(values.cpu(), want)


@pytest.mark.parametrize("bits", [4, 8])
def test_rows_of_extremes(bits, device):
    """Rows whose scale leaves the range the fast quotient is used in, ties,
    infinities and NaN."""
    dim = 64
    rows = torch.zeros((10, 1, dim))
    rows[0] = 3e38
    rows[1, 0, ::2] = 1e-38
    rows[2, 0] = torch.arange(dim) * 2.0**-149  # f32 subnormals: the scale rounds to little or nothing
    rows[3, 0, 5] = math.inf
    rows[4, 0, 6] = math.nan
    rows[5, 0] = (torch.arange(dim) - 32) * 0.5  # ties
    rows[5, 0, 0] = 7.0 if bits == 4 else 127.0
    rows[5, 0, 1:16] = torch.arange(15) * 0.5
    rows[6] = -2.0**-60
    rows[7, 0] = torch.linspace(-(2.0**70), 2.0**70, dim)
    rows[8, 0, 0] = -math.inf
    rows[9, 0] = torch.linspace(-(2.0**-80), 2.0**-81, dim)
    cache = shk.new_kv_cache(1, 16, 1, dim, bits=bits, device=device)
    slots = torch.arange(10, device=device)
    shk.kv_cache_write(cache, rows.to(device), rows.to(device), slots)
    codes, scales = ref.quantized_rows(rows, bits)
    assert torch.equal(cache.key_codes.cpu()[0, :, :10].transpose(0, 1), ref.pack(codes, bits))
    got = shk.kv_cache_read(cache, slots, dtype=torch.float32)[0].cpu()
    want = (codes.double() * scales.double()[..., None]).float()
    assert _same_bits(got, want)
    assert torch.isnan(got[[3, 4, 8]]).all() and torch.isfinite(got[[0, 1, 2, 5, 6, 7, 9]]).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_write_strided_and_misaligned_rows(dtype, device):
    """Slices of a fused projection, a view that starts off 16 bytes, and
    heads in reverse memory order of tokens."""
    tokens, heads, dim = 33, 2, 128
    x = _rows(stable_seed("strided", dtype), tokens, heads, dim, DTYPES[dtype])
    fused = torch.empty((tokens, 3 * heads * dim + 3), dtype=DTYPES[dtype], device=device)
    keys = fused[:, 1:1 + heads * dim].view(tokens, heads, dim)
    values = torch.empty((heads, tokens, dim), dtype=DTYPES[dtype], device=device).transpose(0, 1)
    keys.copy_(x[0])
    values.copy_(x[1])
    cache = shk.new_kv_cache(3, 16, heads, dim, bits=8, device=device)
    slots = torch.arange(tokens, device=device)
    shk.kv_cache_write(cache, keys, values, slots)
    got = shk.kv_cache_read(cache, slots, dtype=torch.float32)
    for rows, have in zip(x, got):
        codes, scales = ref.quantized_rows(rows, 8)
        assert torch.equal(have.cpu(), (codes.double() * scales.double()[..., None]).float())


def test_slots_outside_the_cache(device):
    cache = shk.new_kv_cache(2, 16, 1, 64, bits=4, device=device)
    x = torch.ones((5, 1, 64), device=device, dtype=torch.bfloat16)
    slots = torch.tensor([-1, 3, 32, 31, -(2**40)], device=device)
    shk.kv_cache_write(cache, x, x, slots)
    assert int((cache.key_scales != 0).sum()) == 2 and int((cache.value_codes != 0).any(dim=-1).sum()) == 2
    got = shk.kv_cache_read(cache, slots)[0]
    assert torch.isnan(got[[0, 2, 4]]).all() and torch.equal(got[[1, 3]], x[:2])


def test_a_copy_is_written_alone(device):
    """A prompt's cache is copied, and both go on differently."""
    cache = shk.new_kv_cache(2, 16, 1, 64, bits=8, device=device)
    x = torch.ones((3, 1, 64), device=device, dtype=torch.bfloat16)
    slots = torch.arange(3, device=device)
    shk.kv_cache_write(cache, x, x, slots)
    fork = copy.deepcopy(cache)
    shk.kv_cache_write(fork, 2 * x[:1], 2 * x[:1], slots[:1])
    shk.kv_cache_write(cache, 3 * x[1:2], 3 * x[1:2], slots[1:2])
    for c, want in ((cache, [1, 3, 1]), (fork, [2, 1, 1])):
        keys, _ = shk.kv_cache_read(c, slots)
        assert keys[:, 0].amax(dim=-1).tolist() == keys[:, 0].amin(dim=-1).tolist() == want


def test_no_tokens(device):
    cache = shk.new_kv_cache(1, 16, 2, 64, device=device)
    none = torch.empty((0, 2, 64), device=device)
    shk.kv_cache_write(cache, none, none, torch.empty(0, dtype=torch.int64, device=device))
    keys, values = shk.kv_cache_read(cache, torch.empty(0, dtype=torch.int32, device=device))
    assert keys.shape == values.shape == (0, 2, 64)


# ---------------------------------------------------------------------------
# Attention


def _filled(seed, pages, page, heads, dim, bits, device):
    """A cache of random rows, every scale NaN until _allow allows it."""
    g = torch.Generator().manual_seed(seed)
    most = 7 if bits == 4 else 127
    codes = [ref.pack(torch.randint(-most, most + 1, (pages, heads, page, dim), generator=g), bits) for _ in range(2)]
    scales = [((0.3 + torch.rand((pages, heads, page), generator=g)) * 1.2 / most).bfloat16() for _ in range(2)]
    return codes, scales


def _case(seed, lengths, *, queries=1, ratio=4, kv_heads=2, dim=128, bits=4, page=16, prefix=0, dtype="bf16", spare=1,
          q_gain=2.0, device=None):
    """q, the cache and its tables; tokens that are not held have NaN scales."""
    g = torch.Generator().manual_seed(seed)
    own = [-(-n // page) for n in lengths]
    shared = -(-prefix // page)
    total = sum(own) + shared + 1
    codes, scales = _filled(seed, total, page, kv_heads, dim, bits, device)
    order = torch.randperm(total, generator=g)
    keep = torch.zeros((total, page), dtype=torch.bool)
    # entries past a sequence's tokens are never read
    table = torch.full((len(lengths), max(own + [0]) + spare), 2**31 - 1, dtype=torch.int32)
    at = shared
    for b, n in enumerate(own):
        table[b, :n] = order[at:at + n]
        for i in range(n):
            keep[order[at + i], : min(page, lengths[b] - i * page)] = True
        at += n
    for i in range(shared):
        keep[order[i], : min(page, prefix - i * page)] = True
    for s in scales:
        s.masked_fill_(~keep[:, None].expand_as(s), math.nan)
    q = (q_gain * torch.randn((len(lengths), queries, kv_heads * ratio, dim), generator=g)).to(DTYPES[dtype])
    cache = shk.KVCache(codes[0].to(device), codes[1].to(device), scales[0].to(device), scales[1].to(device))
    return q, cache, table, torch.tensor(lengths, dtype=torch.int32), order[:shared].to(torch.int32)


def _check(got, lse, q, cache, table, lengths, prefix_pages=None, prefix=0, scale=None):
    want = ref.attention(q, _cpu(cache), table, lengths, prefix_pages, prefix, scale)
    tokens = int(lengths.max()) + prefix
    out_bound, lse_bound = ref.attention_bounds(q.dtype, q.shape[-1], tokens, *want)
    got, lse = got.cpu().double().reshape(q.shape), lse.cpu().double().reshape(q.shape[:3])
    assert torch.isfinite(got).all()
    worst = ((got - want[0]).abs() - out_bound).max()
    assert worst <= 0, f"out off by {float((got - want[0]).abs().max())}, {float(worst)} over its bound"
    empty = want[1] == -math.inf
    assert torch.equal(lse == -math.inf, empty) and (got[empty] == 0).all()
    assert ((lse - want[1])[~empty].abs() <= lse_bound[~empty]).all()


def _attend(q, cache, table, lengths, prefix_pages, prefix, device, **kw):
    return shk.kv_cache_attention(q.to(device), cache, table.to(device), lengths.to(device), return_lse=True,
                                  prefix_pages=prefix_pages.to(device) if prefix else None, prefix_length=prefix, **kw)


LENGTHS = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 300]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 64, 1024])
def test_single_tokens(dtype, bits, dim, page, device):
    print(f"case attend {dtype} int{bits} dim {dim} page {page}", flush=True)
    q, cache, table, lengths, _ = _case(stable_seed("one", dtype, bits, dim, page), LENGTHS, dim=dim, bits=bits,
                                        page=page, dtype=dtype, device=device)
    out, lse = _attend(q[:, 0], cache, table, lengths, None, 0, device)
    assert out.shape == q[:, 0].shape and lse.shape == (len(LENGTHS), 8)
    _check(out, lse, q, cache, table, lengths)


@pytest.mark.parametrize("queries,ratio,kv_heads", [(1, 1, 3), (1, 7, 1), (1, 17, 2), (2, 8, 2), (5, 4, 2), (33, 2, 1),
                                                    (70, 1, 1)])
@pytest.mark.parametrize("dtype,bits,dim", [("bf16", 4, 128), ("f16", 8, 64), ("bf16", 8, 256)])
def test_several_queries(queries, ratio, kv_heads, dtype, bits, dim, device):
    """Newest tokens of a sequence see what was written up to themselves;
    sequences shorter than the number of queries leave rows empty."""
    print(f"case attend queries {queries} ratio {ratio} heads {kv_heads} {dtype} int{bits} dim {dim}", flush=True)
    q, cache, table, lengths, _ = _case(stable_seed("several", queries, ratio, kv_heads, dtype, bits, dim),
                                        [0, 1, queries, 64, 150], queries=queries, ratio=ratio, kv_heads=kv_heads,
                                        dtype=dtype, bits=bits, dim=dim, page=32, device=device)
    out, lse = _attend(q, cache, table, lengths, None, 0, device)
    _check(out, lse, q, cache, table, lengths)


@pytest.mark.parametrize("prefix", [1, 16, 63, 200, 1030])
@pytest.mark.parametrize("batch,ratio,queries", [(1, 4, 1), (3, 8, 1), (40, 4, 1), (5, 2, 3)])
@pytest.mark.parametrize("dtype,bits,dim", [("bf16", 4, 128), ("f16", 4, 64), ("bf16", 8, 256), ("f16", 8, 128)])
def test_shared_prefix(prefix, batch, ratio, queries, dtype, bits, dim, device):
    print(f"case prefix {prefix} batch {batch} ratio {ratio} queries {queries} {dtype} int{bits} dim {dim}", flush=True)
    lengths = [(i * 37) % 90 for i in range(batch)]
    q, cache, table, lengths, pages = _case(stable_seed("prefix", prefix, batch, ratio, queries, dtype, bits, dim),
                                            lengths, queries=queries, ratio=ratio, dtype=dtype, bits=bits, dim=dim,
                                            prefix=prefix, device=device)
    out, lse = _attend(q, cache, table, lengths, pages, prefix, device)
    _check(out, lse, q, cache, table, lengths, pages, prefix)


def test_shared_prefix_equals_own_tokens(device):
    """The prefix in front of each sequence's own pages is the same attention."""
    q, cache, table, lengths, pages = _case(11, [20, 0, 47], prefix=64, page=16, device=device)
    out, lse = _attend(q, cache, table, lengths, pages, 64, device)
    joined = torch.cat((pages.expand(3, -1), table), dim=1)
    whole, whole_lse = _attend(q, cache, joined, lengths + 64, None, 0, device)
    assert (out.float() - whole.float()).abs().max() <= 2**-6 and (lse - whole_lse).abs().max() <= 2**-16


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bits", [4, 8])
def test_long_sequences_are_split_and_joined(dtype, bits, device):
    q, cache, table, lengths, pages = _case(stable_seed("long", dtype, bits), [5003, 1, 0], ratio=4, kv_heads=1,
                                            bits=bits, dtype=dtype, page=64, prefix=2049, device=device)
    out, lse = _attend(q, cache, table, lengths, None, 0, device)
    _check(out, lse, q, cache, table, lengths)
    out, lse = _attend(q, cache, table, lengths, pages, 2049, device)
    _check(out, lse, q, cache, table, lengths, pages, 2049)


def _pieces_each(kv_heads, tiles, lengths):
    """The most pieces of 256 tokens that a workgroup of the sequences' own
    tokens takes: they are dealt out over 512 workgroups."""
    total = sum(-(-n // 256) for n in lengths)
    return -(-total // max(1, 512 // (kv_heads * tiles)))


UNEVEN = [3000, 0, 5000, 257, 1, 9000, 256, 3333]


@pytest.mark.parametrize("kv_heads,ratio,queries,lengths,least", [
    (16, 1, 1, UNEVEN, 3),                 # across sequences, an empty and a short one among them
    (64, 1, 3, [3000, 0, 2, 700, 2049], 3),
    (16, 6, 3, [3000, 40, 5000], 2),       # two row tiles
    (64, 1, 1, [5003], 3),                 # one sequence's pieces alone
])
@pytest.mark.parametrize("dtype,bits,dim", [("bf16", 4, 64), ("f16", 4, 128), ("bf16", 8, 128), ("f16", 8, 256)])
def test_workgroups_with_several_pieces(kv_heads, ratio, queries, lengths, least, dtype, bits, dim, device):
    """Several pieces a workgroup, of one sequence and of sequences that follow
    each other."""
    print(f"case pieces {kv_heads} heads ratio {ratio} queries {queries} {dtype} int{bits} dim {dim}", flush=True)
    tiles = -(-queries * ratio // (16 if dim == 256 or queries * ratio <= 16 else 32))
    assert _pieces_each(kv_heads, tiles, lengths) >= least
    q, cache, table, lengths, _ = _case(stable_seed("several pieces", kv_heads, ratio, queries, dtype, bits, dim),
                                        lengths, queries=queries, ratio=ratio, kv_heads=kv_heads, bits=bits, dim=dim,
                                        dtype=dtype, page=64, device=device)
    out, lse = _attend(q, cache, table, lengths, None, 0, device)
    _check(out, lse, q, cache, table, lengths)


@pytest.mark.parametrize("batch", [65, 130])
@pytest.mark.parametrize("kv_heads,dim,prefix", [(2, 128, 0), (32, 64, 0), (2, 128, 300), (32, 64, 300)])
def test_more_sequences_than_a_wave_has_lanes(batch, kv_heads, dim, prefix, device):
    """Empty sequences at either end and past the 64th."""
    lengths = [(i * 97) % 401 * (i % 5 > 0) for i in range(batch)]
    lengths[64:66] = [0, 700]
    lengths = lengths[:batch - 1] + [0] if batch > 65 else lengths[:64] + [700]
    q, cache, table, lengths, pages = _case(stable_seed("many", batch, kv_heads, dim, prefix), lengths, ratio=2,
                                            kv_heads=kv_heads, dim=dim, prefix=prefix, page=32, device=device)
    out, lse = _attend(q, cache, table, lengths, pages, prefix, device)
    _check(out, lse, q, cache, table, lengths, pages if prefix else None, prefix)


@pytest.mark.parametrize("batch,kv_heads,dtype,bits,dim", [
    (3, 64, "bf16", 4, 128), (3, 64, "f16", 8, 64), (3, 64, "bf16", 8, 256),  # the streaming kernel
    (20, 64, "bf16", 4, 128), (20, 64, "f16", 8, 64), (20, 64, "bf16", 8, 256),  # the prefix's own
])
def test_workgroups_with_several_pieces_of_a_prefix(batch, kv_heads, dtype, bits, dim, device):
    prefix = 5003
    assert -(-prefix // 256) >= 2 * -(-512 // kv_heads)  # pieces a workgroup, one row tile
    q, cache, table, lengths, pages = _case(stable_seed("prefix pieces", batch, kv_heads, dtype, bits, dim),
                                            [(i * 37) % 90 for i in range(batch)], kv_heads=kv_heads, bits=bits,
                                            dim=dim, dtype=dtype, prefix=prefix, page=64, device=device)
    out, lse = _attend(q, cache, table, lengths, pages, prefix, device)
    _check(out, lse, q, cache, table, lengths, pages, prefix)


@pytest.mark.parametrize("gain", [0.0, 1e-30, 30.0, 1e4])
def test_flat_and_peaked_scores(gain, device):
    """All probabilities equal; and one that is all but 1, with scores in the
    thousands."""
    q, cache, table, lengths, _ = _case(77, [1, 40, 333], q_gain=gain, device=device)
    out, lse = _attend(q, cache, table, lengths, None, 0, device)
    _check(out, lse, q, cache, table, lengths)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_value_scales_far_apart(dtype, device):
    """Scales of values over many powers of two, the largest at the end."""
    q, cache, table, lengths, _ = _case(stable_seed("apart", dtype), [500], page=64, dtype=dtype, device=device)
    at = torch.arange(cache.value_scales.shape[2], device=device)
    for i in range(8):
        cache.value_scales[int(table[0, i])] *= (2.0 ** ((i + at / 64) * 2 - 20)).bfloat16()
    out, lse = _attend(q, cache, table, lengths, None, 0, device)
    _check(out, lse, q, cache, table, lengths)


@pytest.mark.parametrize("value", [0.0, 2.0**-70, 1.0, 2.0**90])
@pytest.mark.parametrize("prefix", [0, 3])
def test_lse_of_equal_scores(value, prefix, device):
    """The logarithm of the number of tokens, whatever the values' size."""
    q, cache, table, lengths, pages = _case(stable_seed("equal"), list(range(1, 18)), prefix=prefix, q_gain=0.0,
                                            page=64, device=device)
    cache.value_scales[~torch.isnan(cache.value_scales)] = value
    out, lse = _attend(q, cache, table, lengths, pages, prefix, device)
    _check(out, lse, q, cache, table, lengths, pages if prefix else None, prefix)


@pytest.mark.parametrize("dim,bits,ratio,prefix", [(64, 4, 7, 0), (128, 8, 7, 0), (256, 4, 7, 0), (128, 4, 20, 0),
                                                   (64, 8, 7, 10)])
def test_f16_probabilities_keep_both_terms(dim, bits, ratio, prefix, device):
    """The two f16 terms of a probability are of one rounding: with small scores
    the bound is a fraction of what a term off by its last bit does."""
    q, cache, table, lengths, pages = _case(stable_seed("terms", dim, bits, ratio, prefix), [10] * 300, ratio=ratio,
                                            kv_heads=3, dim=dim, bits=bits, dtype="f16", prefix=prefix, q_gain=0.02,
                                            page=64, device=device)
    out, lse = _attend(q, cache, table, lengths, pages, prefix, device)
    _check(out, lse, q, cache, table, lengths, pages if prefix else None, prefix)


@pytest.mark.parametrize("big", [2.0**50, 2.0**90])
@pytest.mark.parametrize("prefix", [0, 600])
@pytest.mark.parametrize("dim,bits", [(128, 4), (256, 8)])
def test_large_values_beside_rows_of_zeros(big, prefix, dim, bits, device):
    """Tokens whose values are zeros keep their share of the sum, whether large
    values come before them, after them or in another piece."""
    q, cache, table, lengths, pages = _case(stable_seed("zeros", prefix, dim, bits), [40, 700, 700, 200], page=64,
                                            q_gain=0.1, dim=dim, bits=bits, prefix=prefix, device=device)
    held = ~torch.isnan(cache.value_scales)
    cache.value_scales[held] = 0.0
    for b, at in ((0, 20), (1, 3), (2, 650), (3, 199)):
        cache.value_scales[int(table[b, at // 64]), :, at % 64] = big
    if prefix:
        cache.value_scales[int(pages[4]), :, 7] = big / 4
    out, lse = _attend(q, cache, table, lengths, pages, prefix, device)
    _check(out, lse, q, cache, table, lengths, pages if prefix else None, prefix)


def test_softmax_scale_and_strides(device):
    q, cache, table, lengths, _ = _case(5, [90, 33], queries=2, device=device)
    wide = torch.zeros((2, 2, 3 * q.shape[2], q.shape[3]), dtype=q.dtype, device=device)
    wide[:, :, 8:16] = q.to(device)
    tables = torch.zeros((2, 20), dtype=torch.int32, device=device)
    tables[:, 5:5 + table.shape[1]] = table.to(device)
    for scale in (0.3, -0.05):
        out, lse = shk.kv_cache_attention(wide[:, :, 8:16], cache, tables[:, 5:5 + table.shape[1]], lengths.to(device),
                                          softmax_scale=scale, return_lse=True)
        _check(out, lse, q, cache, table, lengths, scale=scale)
    flat = torch.zeros(q.numel() + 3, dtype=q.dtype, device=device)  # rows off 16 bytes
    off = flat[3:].view(q.shape)
    off.copy_(q)
    out, lse = shk.kv_cache_attention(off, cache, table.to(device), lengths.to(device), return_lse=True)
    _check(out, lse, q, cache, table, lengths)


@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-60, 1e-44, -1e-30])
@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f16", 256)])
def test_flat_softmax_scales(scale, dtype, dim, device):
    """A scale of zero, or one that a row of zeros leaves no bits of: every
    visible token counts the same."""
    q, cache, table, lengths, pages = _case(stable_seed("flat", dtype, dim), [1, 40, 333, 0], queries=3, dim=dim,
                                            dtype=dtype, prefix=70, device=device)
    q[1] = 0.0
    for prefix in (0, 70):
        out, lse = _attend(q, cache, table, lengths, pages, prefix, device, softmax_scale=scale)
        _check(out, lse, q, cache, table, lengths, pages if prefix else None, prefix, scale=scale)


def test_softmax_scales_that_are_refused(device):
    q, cache, table, lengths, _ = _case(6, [20], device=device)
    for scale in (math.nan, math.inf, -math.inf, 2.0**128 - 2.0**103, 1e300):
        with pytest.raises(ValueError, match="finite in 32 bits"):
            _attend(q, cache, table, lengths, None, 0, device, softmax_scale=scale)


@pytest.mark.parametrize("dtype,bits,dim", [("bf16", 4, 128), ("f16", 8, 64), ("bf16", 8, 256)])
def test_scales_below_zero(dtype, bits, dim, device):
    """Scales of any sign, zeros of either sign among them, count as they
    read back."""
    q, cache, table, lengths, pages = _case(stable_seed("signs", dtype, bits, dim), [1, 40, 600], queries=2, dim=dim,
                                            bits=bits, dtype=dtype, prefix=70, page=32, device=device)
    g = torch.Generator().manual_seed(4)
    for s in (cache.key_scales, cache.value_scales):
        s *= torch.tensor([1.0, -1.0, 0.0, -0.0])[torch.randint(0, 4, s.shape, generator=g)].to(s)
    out, lse = _attend(q, cache, table, lengths, pages, 70, device)
    _check(out, lse, q, cache, table, lengths, pages, 70)
    cache.value_scales.abs_().neg_()
    out, lse = _attend(q, cache, table, lengths, None, 0, device)
    _check(out, lse, q, cache, table, lengths)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_lse_beside_bad_values(dtype, bad, device):
    """The sum of exponentials does not depend on the values."""
    q, cache, table, lengths, _ = _case(stable_seed("lse", dtype), [300, 1500], page=64, q_gain=4.0, dtype=dtype,
                                        device=device)
    for b in range(2):
        cache.value_scales[int(table[b, 0]), :, 9] = bad
    out, lse = _attend(q, cache, table, lengths, None, 0, device)
    assert not torch.isfinite(out).any()
    want = ref.attention(q, _cpu(cache), table, lengths)
    bound = ref.attention_bounds(q.dtype, 128, 1500, *want)[1]
    assert ((lse.cpu().double() - want[1]).abs() <= bound).all()


def test_nan_and_infinity_stay_in_their_sequence(device):
    q, cache, table, lengths, _ = _case(9, [30, 30, 30], kv_heads=1, page=32, device=device)
    cache.value_scales[int(table[1, 0]), 0, 7] = math.inf
    cache.value_codes[int(table[1, 0]), 0, 7] = 0
    cache.key_scales[int(table[2, 0]), 0, 3] = math.nan
    out, lse = _attend(q, cache, table, lengths, None, 0, device)
    assert torch.isnan(out[1]).all() and torch.isnan(out[2]).all() and torch.isnan(lse[2]).all()
    assert torch.isfinite(lse[1]).all()
    _check(out[:1], lse[:1], q[:1], cache, table[:1], lengths[:1])


@pytest.mark.parametrize("queries,ratio", [(2, 1), (5, 2), (6, 4)])
@pytest.mark.parametrize("dtype,bits,dim", [("bf16", 4, 128), ("f16", 8, 64), ("bf16", 8, 256), ("f16", 4, 128)])
def test_values_that_a_query_must_not_see(queries, ratio, dtype, bits, dim, device):
    """The newest token's value is NaN, infinite or larger than all others by
    far: earlier queries give what they give without it."""
    q, cache, table, lengths, _ = _case(stable_seed("unseen", queries, ratio, dtype, bits, dim), [40, 300, 705, 1, 64],
                                        queries=queries, ratio=ratio, bits=bits, dim=dim, dtype=dtype, page=32,
                                        device=device)
    for scale in (math.nan, math.inf, 2.0**60):
        for b, n in enumerate(lengths.tolist()):
            cache.value_scales[int(table[b, (n - 1) // 32]), :, (n - 1) % 32] = scale
        out, lse = _attend(q, cache, table, lengths, None, 0, device)
        _check(out[:, :-1], lse[:, :-1], q[:, :-1], cache, table, lengths - 1)
        if scale != 2.0**60:
            assert not torch.isfinite(out[:, -1]).any() and torch.isfinite(lse[:, -1]).all()
        elif dtype == "bf16":
            _check(out[:, -1:], lse[:, -1:], q[:, -1:], cache, table, lengths)


def _first_page_unused(cache, *tables):
    """Swaps the page that no table names with page 0, which bad page numbers
    are read as."""
    named = torch.cat([t.flatten() for t in tables])
    unused = next(i for i in range(cache.pages) if not (named == i).any())
    for t in tables:
        t[t == 0] = unused
    for part in (cache.key_codes, cache.value_codes, cache.key_scales, cache.value_scales):
        part[[0, unused]] = part[[unused, 0]]


# own tokens alone; after a prefix of few rows and of many
WHERE = {"own": (3, 1, 0), "prefix": (3, 1, 600), "many rows": (3, 6, 600)}


@pytest.mark.parametrize("where", list(WHERE))
@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f16", 64)])
def test_nan_in_one_of_several_pieces(where, dtype, dim, device):
    """A piece in which all visible keys are NaN, one NaN key among the pieces
    that weigh nothing, and queries of NaN: NaN there, and nowhere else."""
    batch, queries, prefix = WHERE[where]
    for gain in (2.0, 1e4):  # at the second, most pieces' weights underflow
        q, cache, table, lengths, pages = _case(stable_seed("pieces", where, dtype, dim), [257, 700, 513],
                                                queries=queries, page=64, dim=dim, dtype=dtype, prefix=prefix,
                                                q_gain=gain, device=device)
        cache.key_scales[int(table[0, 4]), :, 0] = math.nan  # the newest token, alone in its piece
        q[2] = math.nan
        out, lse = _attend(q, cache, table, lengths, pages, prefix, device)
        assert torch.isnan(out[0, -1]).all() and torch.isnan(lse[0, -1]).all()
        assert torch.isnan(out[2]).all() and torch.isnan(lse[2]).all()
        _check(out[1:2], lse[1:2], q[1:2], cache, table[1:2], lengths[1:2], pages, prefix)
        cache.key_scales[int(table[0, 4]), :, 0] = 0.01
        for piece in range(3):
            at = int(table[1, 4 * piece + 1])
            kept = cache.key_scales[at, 1, 5].clone()
            cache.key_scales[at, 1, 5] = math.nan
            out, lse = _attend(q, cache, table, lengths, pages, prefix, device)
            assert torch.isnan(out[1, :, 4:]).all() and torch.isnan(lse[1, :, 4:]).all()
            assert torch.isfinite(out[1, :, :4]).all() and torch.isfinite(lse[1, :, :4]).all()
            cache.key_scales[at, 1, 5] = kept
        _check(out[:1], lse[:1], q[:1], cache, table[:1], lengths[:1], pages, prefix)


@pytest.mark.parametrize("where", list(WHERE))
@pytest.mark.parametrize("gain", [2.0, 1e4])
def test_page_outside_the_cache_in_one_of_several_pieces(where, gain, device):
    """Whichever piece the page is in, whatever the page read instead holds,
    and however little the piece weighs."""
    batch, queries, prefix = WHERE[where]
    q, cache, table, lengths, pages = _case(stable_seed("bad page", where), [700, 0, 90], queries=queries, page=64,
                                            prefix=prefix, q_gain=gain, spare=0, device=device)
    _first_page_unused(cache, table, pages)
    for hold in (math.nan, 1e-3):
        cache.key_scales[0] = cache.value_scales[0] = hold
        for i in range(11):
            bad = table.clone()
            bad[0, i] = -1 if i % 2 else cache.pages
            if i >= 4 and i % 4 == 0:
                bad[0, i:i + 4] = 10**9  # a whole piece
            out, lse = _attend(q, cache, bad, lengths, pages, prefix, device)
            assert torch.isnan(out[0]).all() and torch.isnan(lse[0]).all(), i
            _check(out[1:], lse[1:], q[1:], cache, table[1:], lengths[1:], pages, prefix)
        for i in range(-(-prefix // 64)):
            bad = pages.clone()
            bad[i] = -5
            out, lse = _attend(q, cache, table, lengths, bad, prefix, device)
            assert torch.isnan(out).all() and torch.isnan(lse).all(), i


def test_pages_and_lengths_outside_the_cache(device):
    q, cache, table, lengths, _ = _case(21, [30, 40, 20], page=16, spare=0, device=device)
    table[1, 1] = 10**6
    table[2, 1] = -3
    out, lse = _attend(q, cache, table, lengths, None, 0, device)
    assert torch.isnan(out[1:]).all() and torch.isnan(lse[1:]).all()
    _check(out[:1], lse[:1], q[:1], cache, table[:1], lengths[:1])
    # a length past the table counts as the whole table, a negative one as 0
    odd = torch.tensor([16, 4000, -5], dtype=torch.int32)
    long, _ = _attend(q, cache, table[:1, :1].expand(3, 1), odd, None, 0, device)
    assert torch.isfinite(long).all() and (long[2] == 0).all()


def _refusal(match, call, **kw):
    with pytest.raises((ValueError, RuntimeError), match=match):
        call(**kw)


def test_refusals_of_attention(device):
    q, cache, table, lengths, pages = _case(7, [20, 30], prefix=40, device=device)
    good = {"q": q.to(device), "cache": cache, "page_table": table.to(device), "lengths": lengths.to(device),
            "prefix_pages": pages.to(device), "prefix_length": 40}
    wide = torch.zeros((2, 1, 8, 256), dtype=q.dtype, device=device)
    for name, bad, match in (
        ("q", good["q"].float(), "torch.bfloat16 or torch.float16"), ("q", good["q"][..., :64], "q must have shape"),
        ("q", good["q"][0, 0], "q must have shape"), ("q", good["q"][:, :, :7], "multiple of the cache's 2"),
        ("q", wide[..., ::2], "contiguous along head_dim"), ("q", q, "CUDA/HIP"),
        ("page_table", good["page_table"].long(), "torch.int32"),
        ("page_table", good["page_table"][:1], "page_table must have shape"),
        ("page_table", good["page_table"].t().contiguous().t(), "rows of page_table must be contiguous"),
        ("lengths", good["lengths"].long(), "torch.int32"),
        ("lengths", good["lengths"][:1], "lengths must be contiguous"),
        ("lengths", good["lengths"].expand(2, 2), "lengths must be contiguous"), ("lengths", lengths, "CUDA/HIP"),
        ("prefix_length", 49, "prefix_pages holds 48 tokens"), ("prefix_length", -1, "non-negative"),
        ("prefix_length", True, "non-negative"), ("prefix_pages", None, "needs prefix_pages"),
        ("prefix_pages", good["prefix_pages"].long(), "torch.int32"),
        ("prefix_pages", good["prefix_pages"][::2], "contiguous one-dimensional"),
        ("out", torch.empty_like(good["q"]).float(), "out must be contiguous"),
        ("out", torch.empty((2, 1, 8, 256), dtype=q.dtype, device=device)[..., :128], "out must be contiguous"),
        ("out", torch.empty(2048 + 1, dtype=q.dtype, device=device)[1:].view(q.shape), "out must be aligned to 8"),
    ):
        _refusal(match, shk.kv_cache_attention, **{**good, name: bad})
    shk.kv_cache_attention(**good)


def test_refusals_of_rows(device):
    cache = shk.new_kv_cache(2, 16, 2, 64, device=device)
    x, slots = torch.ones((3, 2, 64), device=device), torch.arange(3, device=device)
    good = {"cache": cache, "keys": x, "values": x, "slots": slots}
    for name, bad, match in (
        ("keys", x.double(), "keys must have dtype"), ("values", x.half(), "values must have the dtype of keys"),
        ("keys", x[:, :1], "keys must have shape"), ("values", x[:2], "values must have shape"),
        ("keys", torch.ones((3, 64, 2), device=device).transpose(1, 2), "contiguous along head_dim"),
        ("slots", slots.float(), "slots must have dtype"), ("slots", slots[:2], "slots must have shape"),
        ("slots", torch.arange(6, device=device)[::2], "slots must be contiguous"), ("keys", x.cpu(), "CUDA/HIP"),
    ):
        _refusal(match, shk.kv_cache_write, **{**good, name: bad})
    for kw, match in (({"dtype": torch.int8}, "the result must have dtype"),
                      ({"slots": slots[None]}, "slots must have shape"), ({"slots": slots.cpu()}, "CUDA/HIP")):
        _refusal(match, shk.kv_cache_read, **{"cache": cache, "slots": slots, **kw})


def test_no_sequences_and_no_pages(device):
    q, cache, table, lengths, _ = _case(3, [4], device=device)
    out = shk.kv_cache_attention(q[:0].to(device), cache, table[:0].to(device), lengths[:0].to(device))
    assert out.shape == (0, 1, 8, 128)
    out, lse = shk.kv_cache_attention(q.to(device), cache, table[:, :0].to(device), lengths.to(device), return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()


def test_no_gradient_is_said(device):
    """Outputs are the same bits; asking them for a gradient raises, and a
    reused buffer keeps no graph."""
    q, cache, table, lengths, _ = _case(51, [30, 9], device=device)
    want = _attend(q, cache, table, lengths, None, 0, device)
    qd = q.to(device).requires_grad_()
    x = torch.ones((1, 2, 128), device=device, requires_grad=True)
    shk.kv_cache_write(cache, x, x, torch.tensor([-1], device=device))
    out = torch.empty_like(qd)
    for kw in ({}, {"out": out}):
        got = _attend(qd, cache, table, lengths, None, 0, device, **kw)
        for g, w in zip(got, want):
            assert torch.equal(g, w)
            with pytest.raises(RuntimeError, match="kv_cache_attention has no gradient"):
                g.sum().backward()
    assert not out.requires_grad and torch.equal(out, want[0])
    with torch.no_grad():
        assert _attend(qd, cache, table, lengths, None, 0, device, out=out)[0] is out


def test_repeated_calls_give_the_same_bits(device):
    q, cache, table, lengths, pages = _case(31, [700, 90], prefix=500, page=64, device=device)
    first = _attend(q, cache, table, lengths, pages, 500, device)
    for _ in range(3):
        again = _attend(q, cache, table, lengths, pages, 500, device)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_other_stream_and_out(device):
    q, cache, table, lengths, _ = _case(41, [700, 90], page=64, device=device)
    qd, td, ld = q.to(device), table.to(device), lengths.to(device)
    want = shk.kv_cache_attention(qd, cache, td, ld)
    stream, out = torch.cuda.Stream(device), torch.zeros_like(qd)
    torch.cuda.synchronize()
    got = shk.kv_cache_attention(qd, cache, td, ld, out=out, stream=stream)
    stream.synchronize()
    assert got is out and torch.equal(out, want)


def _after_a_long_wait(device, sizes, call):
    """Runs `call` on another stream while this one still has to read blocks
    of these sizes that it has given back, and checks what it reads."""
    stream = torch.cuda.Stream(device)
    torch.cuda.synchronize()
    blocks = [torch.full((n,), 7, dtype=torch.uint8, device=device) for n in sizes for _ in range(4)]
    torch.cuda._sleep(20_000_000)
    copies = [b.clone() for b in blocks]
    del blocks
    got = call(stream)
    torch.cuda.synchronize()
    assert all((c == 7).all() for c in copies)
    return got


def test_other_stream_takes_no_block_of_this_one(device):
    q, cache, table, lengths, _ = _case(43, [700, 90], page=64, device=device)
    qd, td, ld = q.to(device), table.to(device), lengths.to(device)
    shifted = torch.empty(qd.numel() + 1, dtype=qd.dtype, device=device)[1:].view(qd.shape).copy_(qd)  # is copied
    slots = torch.arange(90, device=device)
    want, read = shk.kv_cache_attention(qd, cache, td, ld), shk.kv_cache_read(cache, slots)
    sizes = [2 * q.numel(), 2 * read[0].numel()]
    got = _after_a_long_wait(device, sizes, lambda s: (shk.kv_cache_attention(shifted, cache, td, ld, stream=s),
                                                       shk.kv_cache_read(cache, slots, stream=s)))
    assert torch.equal(got[0], want)
    assert torch.equal(got[1][0], read[0]) and torch.equal(got[1][1], read[1])


def test_graph_of_a_step(device):
    """Write and attention captured once; every replay equals the eager step
    on what the buffers hold then."""
    heads, dim, page = 2, 128, 16
    cache = shk.new_kv_cache(8, page, heads, dim, bits=4, device=device)
    table = torch.arange(8, dtype=torch.int32, device=device).view(2, 4)
    lengths = torch.zeros(2, dtype=torch.int32, device=device)
    kv = torch.zeros((2, 2, heads, dim), dtype=torch.bfloat16, device=device)
    q = torch.zeros((2, 8, dim), dtype=torch.bfloat16, device=device)
    slots = torch.zeros(2, dtype=torch.int64, device=device)
    out = torch.zeros_like(q)

    def step():
        shk.kv_cache_write(cache, kv[0], kv[1], slots)
        shk.kv_cache_attention(q, cache, table, lengths, out=out)

    lengths.fill_(1)
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(device).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    g = torch.Generator().manual_seed(1)
    for t in range(5):
        kv.copy_(torch.randn(kv.shape, generator=g))
        q.copy_(torch.randn(q.shape, generator=g))
        lengths.fill_(t + 1)
        slots.copy_(torch.tensor([t, 64 + t]))
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        step()
        assert torch.equal(got, out) and torch.isfinite(got).all()
        _check(out, shk.kv_cache_attention(q, cache, table, lengths, return_lse=True)[1], q.cpu()[:, None], cache,
               table.cpu(), lengths.cpu())


def test_offsets_past_32_bits(device):
    """A pool of more than 4 GiB a part: its last pages are written, read and
    attended over as any others."""
    heads, dim, page = 8, 256, 1024
    pages = 2**32 // (heads * dim * page) + 3
    shape = (pages, heads, page)
    codes = [torch.empty((*shape, dim), dtype=torch.int8, device=device) for _ in range(2)]
    scales = [torch.empty(shape, dtype=torch.bfloat16, device=device) for _ in range(2)]
    cache = shk.KVCache(*codes, *scales)
    tokens = 77
    x = _rows(123, tokens, heads, dim, torch.bfloat16)
    x /= x.float().abs().amax(dim=-1, keepdim=True).bfloat16()
    slots = (pages - 1) * page + torch.arange(tokens)
    xd = x.to(device)
    shk.kv_cache_write(cache, xd[0], xd[1], slots.to(device))
    for rows, got in zip(x, shk.kv_cache_read(cache, slots.to(device), dtype=torch.float32)):
        code, scale = ref.quantized_rows(rows, 8)
        assert torch.equal(got.cpu(), (code.double() * scale.double()[..., None]).float())
    q = torch.randn((1, 1, heads, dim), generator=torch.Generator().manual_seed(2)).bfloat16()
    table, lengths = torch.tensor([[pages - 1]], dtype=torch.int32), torch.tensor([tokens], dtype=torch.int32)
    out, lse = _attend(q, cache, table, lengths, None, 0, device)
    last = tuple(t[-1:].cpu() for t in (*codes, *scales))
    want = ref.attention(q, last, torch.zeros_like(table), lengths)
    bounds = ref.attention_bounds(q.dtype, dim, tokens, *want)
    assert ((out.cpu().double() - want[0]).abs() <= bounds[0]).all()
    assert ((lse.cpu().double() - want[1]).abs() <= bounds[1]).all()
