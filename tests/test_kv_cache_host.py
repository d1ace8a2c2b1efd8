"""Refusals of the quantized cache's entry points, checked without a GPU: the
Python argument checks, and the C ABI's own before it touches the device."""

from __future__ import annotations

import copy
import io
import pickle

import pytest

torch = pytest.importorskip("torch")

import amd_strix_halo_kernels as shk  # noqa: E402
from amd_strix_halo_kernels import kernel_table as kt  # noqa: E402
from amd_strix_halo_kernels import kv_cache, native  # noqa: E402

FAKE = 0x10000  # never dereferenced: every call below fails validation first


def _cache(**kw):
    args = {"pages": 4, "page_size": 16, "kv_heads": 2, "head_dim": 64, "device": "cpu"} | kw
    shape = [args.pop(n) for n in ("pages", "page_size", "kv_heads", "head_dim")]
    return shk.new_kv_cache(*shape, **args)


def test_new_cache_layout():
    c = _cache(bits=4)
    assert c.key_codes.shape == (4, 2, 16, 32) and c.key_codes.dtype == torch.uint8
    assert c.key_scales.shape == (4, 2, 16) and c.key_scales.dtype == torch.bfloat16
    assert (c.pages, c.kv_heads, c.page_size, c.head_dim, c.bits) == (4, 2, 16, 64, 4)
    c = _cache(bits=8, head_dim=256)
    assert c.value_codes.shape == (4, 2, 16, 256) and c.value_codes.dtype == torch.int8 and c.bits == 8


@pytest.mark.parametrize("kw,match", [({"bits": 3}, "bits must be 4 or 8"),
                                      ({"head_dim": 96}, "head_dim must be one of"),
                                      ({"page_size": 8}, "power of two"), ({"page_size": 48}, "power of two"),
                                      ({"page_size": 2048}, "power of two"), ({"pages": 0}, "at least one page"),
                                      ({"kv_heads": 0}, "65535 heads")])
def test_cache_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        _cache(**kw)


def test_cache_tensor_refusals():
    c = _cache()
    parts = {n: getattr(c, n) for n in ("key_codes", "value_codes", "key_scales", "value_scales")}
    for name, bad, match in (
        ("key_codes", c.key_codes.float(), "int8 codes or packed int4"),
        ("key_codes", c.key_codes[0], "must have shape"),
        ("value_codes", c.value_codes[:2], "value_codes must have shape"),
        ("value_codes", c.value_codes.to(torch.int8), "value_codes must have shape"),
        ("key_scales", c.key_scales.float(), "key_scales must have shape"),
        ("value_scales", torch.zeros((4, 16, 2), dtype=torch.bfloat16).transpose(1, 2), "must be contiguous"),
    ):
        with pytest.raises(ValueError, match=match):
            shk.KVCache(**{**parts, name: bad})


PARTS = ("key_codes", "value_codes", "key_scales", "value_scales")


def _saved(c):
    f = io.BytesIO()
    torch.save(c, f)
    f.seek(0)
    return torch.load(f, weights_only=False)


@pytest.mark.parametrize("how", [copy.deepcopy, lambda c: pickle.loads(pickle.dumps(c)), _saved, copy.copy])
def test_copies_pass_their_own_memory(how):
    """What reaches the library are the addresses and sizes of the copy's own
    tensors; only a shallow copy shares the original's."""
    c = _cache(bits=8, head_dim=128)
    c._workspaces[(1, 1, 2, 1, 0)] = 64
    d = how(c)
    own = tuple(getattr(d, n).data_ptr() for n in PARTS)
    assert kv_cache._CACHE.unpack(d._native) == (*own, 4, 2, 16, 128, 8)
    assert (own == tuple(getattr(c, n).data_ptr() for n in PARTS)) == (how is copy.copy)
    assert (d.pages, d.kv_heads, d.page_size, d.head_dim, d.bits, d.device) == (4, 2, 16, 128, 8, c.device)
    assert d._workspaces is not c._workspaces


def test_memory_that_a_tensor_was_given_later():
    c = _cache()
    c.key_scales.data = torch.zeros_like(c.key_scales)
    assert kv_cache._CACHE.unpack(c._native)[:4] == tuple(getattr(c, n).data_ptr() for n in PARTS)
    c.value_codes.data = torch.zeros((3, 2, 16, 32), dtype=torch.uint8)
    with pytest.raises(ValueError, match="value_codes must have shape"):
        c._native
    c = _cache()
    for n in PARTS:  # more heads in all of them: the next call checks its arguments against those
        t = getattr(c, n)
        t.data = torch.zeros((4, 5, *t.shape[2:]), dtype=t.dtype)
    with pytest.raises(RuntimeError, match="CUDA/HIP"):
        shk.kv_cache_read(c, torch.arange(3))
    assert c.kv_heads == 5


def test_calls_need_the_device():
    c = _cache()
    x = torch.zeros((3, 2, 64))
    slots = torch.arange(3)
    with pytest.raises(RuntimeError, match="CUDA/HIP"):
        shk.kv_cache_write(c, x, x, slots)
    with pytest.raises(RuntimeError, match="CUDA/HIP"):
        shk.kv_cache_read(c, slots)
    with pytest.raises(RuntimeError, match="CUDA/HIP"):
        shk.kv_cache_attention(x, c, torch.zeros((3, 1), dtype=torch.int32), torch.zeros(3, dtype=torch.int32))


@pytest.fixture(scope="module")
def lib():
    return native.load_dispatch_library()


def _native_cache(**kw):
    f = {"key_codes": FAKE, "value_codes": FAKE, "key_scales": FAKE, "value_scales": FAKE, "pages": 4, "kv_heads": 2,
         "page_size": 16, "head_dim": 64, "bits": 4} | kw
    return kv_cache._CACHE.pack(*(v or 0 for v in f.values()))


def _native_rows(**kw):
    f = {"keys": FAKE, "values": FAKE, "key_token_stride": 128, "key_head_stride": 64, "value_token_stride": 128,
         "value_head_stride": 64, "type": kt.SRC_BF16, "slots": FAKE, "slot_bytes": 8, "tokens": 3} | kw
    return kv_cache._ROWS.pack(*(v or 0 for v in f.values()))


def _native_attention(**kw):
    f = {"q": FAKE, "q_batch_stride": 256, "q_query_stride": 0, "q_head_stride": 64, "type": kt.SRC_BF16, "batch": 2,
         "queries": 1, "heads": 4, "page_table": FAKE, "table_stride": 4, "table_pages": 4, "lengths": FAKE,
         "prefix_pages": None, "prefix_length": 0, "scale": 0.125, "out": FAKE, "lse": None, "workspace": None,
         "workspace_bytes": 0} | kw
    return kv_cache._ATTENTION.pack(*(v or 0 for v in f.values()))


CACHE_FAULTS = [({"bits": 5}, "bits must be 4 or 8"), ({"head_dim": 80}, "head_dim must be"),
                ({"page_size": 24}, "power of two"), ({"pages": 0}, "pages"), ({"pages": 2**31}, "pages"),
                ({"kv_heads": 0}, "heads"), ({"value_scales": None}, "non-null"),
                ({"key_codes": FAKE + 8}, "aligned to 16"), ({"key_scales": FAKE + 4}, "aligned to 8")]


@pytest.mark.parametrize("kw,match", CACHE_FAULTS)
def test_c_abi_refuses_caches(lib, kw, match):
    cache = _native_cache(**kw)
    for call in (lambda: lib.amd_strix_halo_kernels_kv_write(0, 0, cache, _native_rows()),
                 lambda: lib.amd_strix_halo_kernels_kv_read(0, 0, cache, _native_rows()),
                 lambda: lib.amd_strix_halo_kernels_kv_attention(0, 0, cache,
                                                                 _native_attention())):
        assert call() == 1
        assert match in lib.amd_strix_halo_kernels_last_error().decode()
    args = _native_attention()
    assert lib.amd_strix_halo_kernels_kv_attention_workspace(cache, args) == -1


@pytest.mark.parametrize("kw,match", [({"type": kt.SRC_I8}, "row type"), ({"slot_bytes": 2}, "int32 or int64"),
                                      ({"tokens": -1}, "negative"), ({"keys": None}, "non-null"),
                                      ({"slots": None}, "non-null")])
def test_c_abi_refuses_rows(lib, kw, match):
    cache, rows = _native_cache(), _native_rows(**kw)
    assert lib.amd_strix_halo_kernels_kv_write(0, 0, cache, rows) == 1
    assert match in lib.amd_strix_halo_kernels_last_error().decode()


@pytest.mark.parametrize("kw,match", [
    ({"type": kt.SRC_F32}, "float16 or bfloat16"), ({"heads": 3}, "multiple of the cache's kv_heads"),
    ({"heads": 0}, "multiple"), ({"batch": -1}, "negative"), ({"batch": 2**31}, "too many query rows"),
    ({"table_pages": 2**31}, "at most"), ({"prefix_length": -1}, "prefix_length"),
    ({"prefix_length": 5}, "prefix_pages pointer"), ({"q": None}, "non-null"), ({"lengths": None}, "non-null"),
    ({"page_table": None}, "page_table pointer"), ({"q": FAKE + 2}, "aligned to 16"),
    ({"q_head_stride": 65}, "aligned to 16"), ({"out": FAKE + 2}, "out must be aligned"),
    ({"table_pages": 4096}, "workspace must hold"),
    ({"scale": float("nan")}, "finite in 32 bits"), ({"scale": float("-inf")}, "finite in 32 bits"),
    ({"scale": 3.5e38}, "finite in 32 bits"),
])
def test_c_abi_refuses_attention(lib, kw, match):
    args = _native_attention(**kw)
    assert lib.amd_strix_halo_kernels_kv_attention(0, 0, _native_cache(), args) == 1
    assert match in lib.amd_strix_halo_kernels_last_error().decode()


@pytest.mark.parametrize("kw,match", [
    # 32-bit counts of tokens and pieces
    ({"table_pages": (2**31 - 256) // 16}, "at most 2147483391 tokens"),
    ({"prefix_pages": FAKE, "prefix_length": 2**31 - 256}, "prefix_length must be from 0 to 2147483391"),
    ({"batch": 2**12, "table_pages": 2**27 - 256}, "too many tokens in the page table"),
    # a launch of 2^32 work-items or more, of the join and of the first kernel
    ({"batch": 2**21, "heads": 8, "table_pages": 17}, "too many query rows for one launch"),
    ({"batch": 2**23, "heads": 2}, "too many query rows for one launch"),
])
def test_c_abi_refuses_attention_past_its_counts(lib, kw, match):
    args = _native_attention(**kw)
    assert lib.amd_strix_halo_kernels_kv_attention(0, 0, _native_cache(), args) == 1
    assert match in lib.amd_strix_halo_kernels_last_error().decode()
    assert lib.amd_strix_halo_kernels_kv_attention_workspace(_native_cache(), args) == -1
    assert match in lib.amd_strix_halo_kernels_last_error().decode()


@pytest.mark.parametrize("kw", [
    {"table_pages": (2**31 - 257) // 16}, {"prefix_pages": FAKE, "prefix_length": 2**31 - 257},
    {"batch": 2**21 - 1, "heads": 8, "table_pages": 17}, {"batch": 2**21, "heads": 8, "table_pages": 16},
    {"batch": 2**23 - 1, "heads": 2},
    {"batch": 0, "table_pages": 100, "prefix_pages": FAKE, "prefix_length": 100}, {"queries": 0, "table_pages": 100},
])
def test_attention_up_to_its_counts(lib, kw):
    assert lib.amd_strix_halo_kernels_kv_attention_workspace(_native_cache(), _native_attention(**kw)) >= 0


@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_c_abi_refuses_rows_past_a_launch(lib, head_dim):
    """16777215 workgroups of 2048 values written, of 4096 read; rows in 32 bits."""
    cache = _native_cache(head_dim=head_dim, kv_heads=3)
    for call, values in ((lib.amd_strix_halo_kernels_kv_write, 2048), (lib.amd_strix_halo_kernels_kv_read, 4096)):
        most = min(16777215 * (values // head_dim), 2**31 - 1) // 3
        assert call(0, 0, cache, _native_rows(tokens=most + 1)) == 1
        assert "too many tokens for one launch" in lib.amd_strix_halo_kernels_last_error().decode()


def test_c_abi_null_structs_and_empty_calls(lib):
    cache, rows, args = _native_cache(), _native_rows(tokens=0), _native_attention(batch=0)
    assert lib.amd_strix_halo_kernels_kv_write(0, 0, None, rows) == 1
    assert lib.amd_strix_halo_kernels_kv_read(0, 0, cache, None) == 1
    assert lib.amd_strix_halo_kernels_kv_attention(0, 0, cache, None) == 1
    assert lib.amd_strix_halo_kernels_kv_write(0, 0, cache, rows) == 0
    assert lib.amd_strix_halo_kernels_kv_attention(0, 0, cache, args) == 0
    assert lib.amd_strix_halo_kernels_kv_attention_workspace(cache, args) == 0
