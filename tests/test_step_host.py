"""Refusals of the step's operators and of the fp8 products, checked without a
GPU: the Python argument checks that come first, and the C ABI's own before it
touches the device.  Also the frequencies of a rotary, which are made on the host."""

from __future__ import annotations

import copy
import ctypes
import math
import pickle

import pytest

torch = pytest.importorskip("torch")

import amd_strix_halo_kernels as shk  # noqa: E402
from amd_strix_halo_kernels import fp8, kv_pages, native, rotary, verify  # noqa: E402
from amd_strix_halo_kernels import kernel_table as kt  # noqa: E402
from amd_strix_halo_kernels import kv_cache  # noqa: E402

FAKE = 0x10000  # never dereferenced: every call below fails validation first


@pytest.fixture(scope="module")
def lib():
    return native.load_dispatch_library()


def test_calls_need_the_device():
    x = torch.zeros((4, 2, 64), dtype=torch.bfloat16)
    turn = shk.new_rotary([1.0], device="cpu")
    pages = shk.new_kv_pages(4, 2, 8, 16, device="cpu")
    codes = torch.zeros((4, 128)).to(torch.float8_e4m3fn)
    for call in (lambda: shk.quantize_fp8(x[:, 0]),
                 lambda: shk.mm_fp8(codes, codes, a_scale=torch.ones((4, 1)), b_scale=torch.ones((1, 1))),
                 lambda: shk.rotate_qk(x, x, torch.arange(4), turn),
                 lambda: shk.kv_pages_step(pages, torch.zeros(4, dtype=torch.int32), 8),
                 lambda: shk.verify_draft(torch.zeros((1, 2, 8)), None, torch.zeros((1, 1), dtype=torch.int64),
                                          torch.zeros((1, 2)))):
        with pytest.raises(RuntimeError, match="CUDA/HIP"):
            call()


# ---------------------------------------------------------------------------
# Frequencies


def test_plain_frequencies():
    got, amplitude = shk.rotary_frequencies(8, base=16.0)
    assert amplitude == 1.0 and got == [1.0, 16.0**-0.25, 16.0**-0.5, 16.0**-0.75]
    assert shk.rotary_frequencies(8, base=16.0, scaling="linear", factor=4.0)[0] == [f / 4 for f in got]


def test_ntk_slows_the_slowest_by_the_factor():
    plain, _ = shk.rotary_frequencies(64)
    got, amplitude = shk.rotary_frequencies(64, scaling="ntk", factor=8.0)
    assert amplitude == 1.0 and got[0] == plain[0] == 1.0
    assert math.isclose(got[-1], plain[-1] / 8, rel_tol=1e-12)
    assert all(a >= b for a, b in zip(plain, got))


def test_yarn_keeps_fast_pairs_and_slows_slow_ones():
    plain, _ = shk.rotary_frequencies(128)
    got, amplitude = shk.rotary_frequencies(128, scaling="yarn", factor=16.0, trained=4096)
    assert math.isclose(amplitude, 0.1 * math.log(16.0) + 1.0)
    turns = [f * 4096 / (2 * math.pi) for f in plain]
    for f, g, t in zip(plain, got, turns):
        assert f / 16 * (1 - 1e-12) <= g <= f * (1 + 1e-12)
        if t > 32 * 1.2:
            assert g == f
        if t < 1 / 1.2:
            assert math.isclose(g, f / 16, rel_tol=1e-12)


@pytest.mark.parametrize("args,match", [({"rotated": 7}, "even"), ({"rotated": 0}, "even"), ({"rotated": True}, "even"),
                                        ({"rotated": 8, "scaling": "more"}, "scaling"),
                                        ({"rotated": 8, "factor": 0.0}, "factor"),
                                        ({"rotated": 8, "base": math.inf}, "base"),
                                        ({"rotated": 8, "scaling": "yarn"}, "trained"),
                                        ({"rotated": 8, "scaling": "yarn", "trained": 64, "slow": 40.0}, "fast > slow")])
def test_frequency_refusals(args, match):
    with pytest.raises(ValueError, match=match):
        shk.rotary_frequencies(**args)


def test_rotary_handle():
    r = shk.new_rotary([2 * math.pi, math.pi], amplitude=2.0, interleaved=True, device="cpu")
    assert r.turns.tolist() == [1.0, 0.5] and r.rotated == 4 and r.amplitude == 2.0 and r.interleaved
    with pytest.raises(ValueError, match="finite"):
        shk.new_rotary([math.nan], device="cpu")
    with pytest.raises(ValueError, match="float64"):
        shk.Rotary(torch.zeros(3), 1.0, False)


# ---------------------------------------------------------------------------
# Pages


def test_new_pages():
    p = shk.new_kv_pages(3, 5, 20, 32, first=4, device="cpu")
    assert p.page_table.shape == (3, 5) and p.free_count.tolist() == [16]
    assert p.free_pages.tolist() == list(range(19, 3, -1))
    for how in (copy.deepcopy, lambda x: pickle.loads(pickle.dumps(x))):
        q = how(p)
        assert q.lengths.data_ptr() != p.lengths.data_ptr() and q._ticket.data_ptr() != p._ticket.data_ptr()
        assert q.free_pages.tolist() == p.free_pages.tolist() and q.page_size == 32


@pytest.mark.parametrize("name,bad,match", [("lengths", torch.zeros(4, dtype=torch.int32), "lengths must"),
                                            ("owned", torch.zeros(3, dtype=torch.int64), "owned must"),
                                            ("page_table", torch.zeros((5, 3), dtype=torch.int32).t(), "page_table must"),
                                            ("page_table", torch.zeros(3, dtype=torch.int32), "page_table must"),
                                            ("free_count", torch.zeros((), dtype=torch.int32), "free_count must"),
                                            ("free_pages", torch.zeros((2, 2), dtype=torch.int32), "free_pages must"),
                                            ("page_size", 24, "power of two"), ("page_size", 8, "power of two")])
def test_pages_refusals(name, bad, match):
    p = shk.new_kv_pages(3, 5, 20, 32, device="cpu")
    parts = {n: getattr(p, n) for n in (*kv_pages._PARTS, "page_size")}
    with pytest.raises(ValueError, match=match):
        shk.KVPages(**{**parts, name: bad})


def test_pages_sizes():
    with pytest.raises(ValueError, match="4096 sequences"):
        shk.new_kv_pages(4097, 1, 8, 16, device="cpu")
    with pytest.raises(ValueError, match="at least one page"):
        shk.new_kv_pages(3, 0, 8, 16, device="cpu")
    with pytest.raises(ValueError, match="first must be"):
        shk.new_kv_pages(3, 2, 8, 16, first=9, device="cpu")


# ---------------------------------------------------------------------------
# The C ABI


def _refuses(lib, fn, packed, match):
    assert fn(0, 0, *packed) == 1
    assert match in lib.amd_strix_halo_kernels_last_error(), lib.amd_strix_halo_kernels_last_error()


QUANTIZE = {"x": FAKE, "type": kt.SRC_BF16, "rows": 4, "cols": 200, "x_stride": 200, "transpose": 0, "block_rows": 1,
            "kind": kt.FP8_E4M3, "codes": FAKE, "code_pitch": 208, "scales": FAKE, "scale_row_stride": 1,
            "scale_block_stride": 4}


@pytest.mark.parametrize("bad,match", [({"type": 3}, b"source type"), ({"kind": 2}, b"e4m3 or e5m2"),
                                       ({"block_rows": 64}, b"1 or 128"), ({"rows": -1}, b"rows and cols"),
                                       ({"x_stride": 199}, b"x must not overlap"),
                                       ({"code_pitch": 199}, b"codes must not overlap"),
                                       ({"x": 0}, b"non-null"), ({"scales": FAKE + 2}, b"aligned"),
                                       ({"x": FAKE + 1}, b"aligned"), ({"rows": 2**31 - 1}, b"too many blocks"),
                                       ({"rows": 2**23, "transpose": 1, "code_pitch": 2**23}, b"too many blocks")])
def test_quantize_refusals(lib, bad, match):
    packed = fp8._QUANTIZE.pack(*(QUANTIZE | bad).values())
    _refuses(lib, lib.amd_strix_halo_kernels_fp8_quantize, (packed,), match)


MM = {"a": FAKE, "a_pitch": 256, "a_kind": 0, "b": FAKE, "b_pitch": 256, "b_kind": 0, "a_scale": FAKE,
      "a_scale_row": 2, "a_scale_block": 1, "b_scale": FAKE, "b_scale_row": 2, "b_scale_block": 1, "b_rows": 128, "m": 64,
      "n": 128, "k": 256, "out": FAKE, "out_stride": 128, "out_type": kt.SRC_BF16, "work": 0, "work_bytes": 0}


@pytest.mark.parametrize("bad,match", [({"a_kind": 2}, b"e4m3 or e5m2"), ({"out_type": 3}, b"output type"),
                                       ({"b_rows": 2}, b"1 or 128"), ({"k": 2**23}, b"8388607"), ({"m": -1}, b"m and n"),
                                       ({"a_pitch": 255}, b"pitches"), ({"b_pitch": 2**24}, b"pitches"),
                                       ({"out_stride": 127}, b"out must not overlap"),
                                       ({"a_scale_row": -1}, b"not negative"), ({"b_scale_block": 2**30}, b"span less"),
                                       ({"out": 0}, b"non-null"), ({"a_scale": 0}, b"non-null"),
                                       ({"out": FAKE + 1}, b"aligned"), ({"a": FAKE + 8, "m": 100}, b"workspace must hold"),
                                       ({"m": 2**28, "n": 2**28, "out_stride": 2**28}, b"too many outputs"),
                                       ({"m": 1, "n": 2**29 - 1, "k": 1, "out_stride": 2**29}, b"too many outputs"),
                                       ({"m": 2**29}, b"m and n")])
def test_product_refusals(lib, bad, match):
    packed = fp8._MM.pack(*(MM | bad).values())
    _refuses(lib, lib.amd_strix_halo_kernels_fp8_mm, (packed,), match)


ROTATE = {"q": FAKE, "qt": 512, "qh": 64, "k": FAKE, "kt": 512, "kh": 64, "type": kt.SRC_BF16, "tokens": 4, "heads": 4,
          "kv_heads": 2, "head_dim": 64, "rotated": 64, "interleaved": 0, "positions": FAKE, "position_bytes": 8,
          "turns": FAKE, "amplitude": 1.0, "q_weight": 0, "k_weight": 0, "weight_type": kt.SRC_BF16, "eps": 1e-6,
          "q_out": FAKE, "qot": 256, "qoh": 64, "k_out": FAKE, "kot": 128, "koh": 64, "values": 0, "vt": 0, "vh": 0,
          "slots": 0, "slot_bytes": 4}
CACHE = {"key_codes": FAKE, "value_codes": FAKE, "key_scales": FAKE, "value_scales": FAKE, "pages": 4, "kv_heads": 2,
         "page_size": 16, "head_dim": 64, "bits": 4}


@pytest.mark.parametrize("bad,match", [({"type": 3}, b"value type"), ({"heads": 0}, b"heads"), ({"head_dim": 65}, b"even"),
                                       ({"head_dim": 258}, b"even"), ({"rotated": 66}, b"rotated"),
                                       ({"rotated": 3}, b"rotated"), ({"position_bytes": 2}, b"int32 or int64"),
                                       ({"amplitude": math.inf}, b"amplitude"), ({"eps": -1.0}, b"eps"),
                                       ({"eps": math.nan}, b"eps"), ({"q_weight": FAKE}, b"both or neither"),
                                       ({"tokens": 2**29}, b"too many rows"), ({"k_out": 0}, b"k_out"),
                                       ({"q": 0}, b"non-null"), ({"positions": FAKE + 4}, b"aligned"),
                                       ({"turns": FAKE + 4}, b"aligned")])
def test_rotate_refusals(lib, bad, match):
    packed = rotary._ROTATE.pack(*(ROTATE | bad).values())
    _refuses(lib, lib.amd_strix_halo_kernels_rotate, (None, packed), match)


@pytest.mark.parametrize("bad,cache,match", [({}, {}, b"values and slots"), ({"values": FAKE}, {}, b"values and slots"),
                                             ({"head_dim": 128}, {}, b"must be the cache's"),
                                             ({"kv_heads": 4}, {}, b"must be the cache's"),
                                             ({"values": FAKE, "slots": FAKE, "slot_bytes": 2}, {}, b"slots are"),
                                             ({"values": FAKE, "slots": FAKE}, {"bits": 5}, b"bits must be"),
                                             ({"values": FAKE, "slots": FAKE + 2}, {}, b"aligned")])
def test_rotate_cache_refusals(lib, bad, cache, match):
    packed = rotary._ROTATE.pack(*(ROTATE | {"k_out": 0} | bad).values())
    _refuses(lib, lib.amd_strix_halo_kernels_rotate, (kv_cache._CACHE.pack(*(CACHE | cache).values()), packed), match)


PLAN = {"page_table": FAKE, "batch": 4, "width": 8, "lengths": FAKE, "owned": FAKE, "free_pages": FAKE, "free_total": 32,
        "free_count": FAKE, "page_size": 16, "new_tokens": FAKE, "capacity": 64, "slots": FAKE, "positions": FAKE,
        "sequences": FAKE, "starts": FAKE, "taken": FAKE, "ticket": FAKE}


@pytest.mark.parametrize("bad,match", [({"batch": 0}, b"1 to 4096"), ({"batch": 4097}, b"1 to 4096"),
                                       ({"page_size": 48}, b"power of two"), ({"width": 0}, b"at least one page"),
                                       ({"width": 2**28}, b"2147483647 tokens"), ({"free_total": -1}, b"free pages"),
                                       ({"capacity": 2**31}, b"capacity"), ({"ticket": 0}, b"non-null"),
                                       ({"slots": FAKE + 4}, b"aligned"), ({"lengths": FAKE + 2}, b"aligned")])
def test_plan_refusals(lib, bad, match):
    packed = kv_pages._PLAN.pack(*(PLAN | bad).values())
    _refuses(lib, lib.amd_strix_halo_kernels_kv_plan, (packed,), match)


VERIFY = {"target": FAKE, "tb": 400, "tr": 100, "draft": FAKE, "db": 300, "dr": 100, "type": kt.SRC_F32, "batch": 2,
          "drafts": 3, "vocab": 100, "tokens": FAKE, "token_bytes": 8, "uniforms": FAKE, "counts": 0, "out": FAKE,
          "kept": FAKE, "lengths": 0, "work": FAKE, "work_bytes": 1 << 20}


@pytest.mark.parametrize("bad,match", [({"type": 3}, b"value type"), ({"batch": 65536}, b"65535 sequences"),
                                       ({"drafts": 64}, b"63 drafts"), ({"vocab": 0}, b"vocabulary"),
                                       ({"token_bytes": 2}, b"int32 or int64"), ({"target": 0}, b"non-null"),
                                       ({"tokens": 0}, b"non-null"), ({"out": FAKE + 4}, b"aligned"),
                                       ({"vocab": 10**6, "work_bytes": 8}, b"workspace must hold"),
                                       ({"vocab": 10**6, "work": 0}, b"workspace must hold")])
def test_verify_refusals(lib, bad, match):
    packed = verify._VERIFY.pack(*(VERIFY | bad).values())
    _refuses(lib, lib.amd_strix_halo_kernels_verify, (packed,), match)


def test_null_structs_and_empty_calls(lib):
    for fn in (lib.amd_strix_halo_kernels_fp8_quantize, lib.amd_strix_halo_kernels_fp8_mm,
               lib.amd_strix_halo_kernels_kv_plan, lib.amd_strix_halo_kernels_verify):
        _refuses(lib, fn, (None,), b"must be non-null")
    _refuses(lib, lib.amd_strix_halo_kernels_rotate, (None, None), b"must be non-null")
    assert lib.amd_strix_halo_kernels_fp8_mm_workspace(None) == -1
    assert lib.amd_strix_halo_kernels_verify_workspace(None) == -1
    none = 0
    assert lib.amd_strix_halo_kernels_fp8_mm(0, none, fp8._MM.pack(*(MM | {"m": 0}).values())) == 0
    assert lib.amd_strix_halo_kernels_fp8_quantize(0, none, fp8._QUANTIZE.pack(*(QUANTIZE | {"rows": 0}).values())) == 0
    assert lib.amd_strix_halo_kernels_rotate(0, none, None, rotary._ROTATE.pack(*(ROTATE | {"tokens": 0}).values())) == 0
    assert lib.amd_strix_halo_kernels_verify(0, none, verify._VERIFY.pack(*(VERIFY | {"batch": 0}).values())) == 0


def test_structs_match_the_header():
    """Every field of the structs is 8 bytes."""
    for packed, fields in ((fp8._QUANTIZE, QUANTIZE), (fp8._MM, MM), (rotary._ROTATE, ROTATE), (kv_pages._PLAN, PLAN),
                           (verify._VERIFY, VERIFY)):
        assert packed.size == 8 * len(fields)
    assert ctypes.sizeof(ctypes.c_double) == 8
