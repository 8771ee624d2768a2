"""CPU-side checks of the paged C ABI: every declared symbol is exported and bound, the Rust
block equals the header, and bad arguments are refused on the host before any GPU work."""
import ctypes
import os
import re

import pytest

from unillm_amd import _capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB_RS = os.path.join(ROOT, "unillm_amd", "rust", "src", "lib.rs")

C_TO_RUST = {
    "int": "c_int", "int64_t": "i64", "float": "f32", "void*": "*mut c_void",
    "void**": "*mut *mut c_void", "size_t*": "*mut usize", "const float*": "*const f32",
    "float*": "*mut f32", "const int32_t*": "*const i32", "int32_t**": "*mut *mut i32",
    "const unillm_page_table*": "*const unillm_page_table",
    "unillm_page_table*": "*mut unillm_page_table",
    "unillm_page_table**": "*mut *mut unillm_page_table",
    "const unillm_paged_kv*": "*const unillm_paged_kv", "unillm_paged_kv*": "*mut unillm_paged_kv",
    "unillm_paged_kv**": "*mut *mut unillm_paged_kv",
}


@pytest.fixture(scope="module")
def lib():
    return _capi.lib()


def test_every_paged_symbol_is_exported_and_bound(lib):
    declared = _capi.header_symbols(_capi.PAGED_HEADER)
    assert len(declared) == 13 and sorted(_capi.PAGED_SIGNATURES) == declared
    for name in declared:
        assert hasattr(lib, name), name
    assert '#include "unillm_hip_paged.h"' in open(_capi.HEADER).read()


def test_rust_paged_block_equals_header():
    header = re.sub(r"/\*.*?\*/", " ", open(_capi.PAGED_HEADER).read(), flags=re.S)
    want = {}
    for ret, name, params in re.findall(r"^\s*(\w+)\s+(unillm_hip_\w+)\s*\(([^)]*)\)\s*;", header,
                                        flags=re.M):
        args = []
        for p in " ".join(params.split()).split(","):
            m = re.match(r"^(.*?)(\w+)$", p.strip())
            args.append((m.group(2), C_TO_RUST[re.sub(r"\s*\*", "*", m.group(1).strip())]))
        want[name] = (args, C_TO_RUST[ret])
    blocks = re.findall(r'extern "C" \{(.*?)\n    \}', open(LIB_RS).read(), flags=re.S)
    assert len(blocks) == 2
    got = {}
    for name, params, ret in re.findall(r"pub fn (unillm_hip_\w+)\(([^)]*)\)\s*->\s*([^;]+);",
                                        blocks[1], flags=re.S):
        args = [tuple(s.strip() for s in p.split(":", 1))
                for p in " ".join(params.split()).split(",") if p.strip()]
        got[name] = (args, " ".join(ret.split()))
    assert len(want) == 13 and got == want


GOOD = dict(max_seqs=4, max_pages=8, n_pages=20, page_size=16, max_tokens=64)


@pytest.mark.parametrize("change", [
    dict(max_seqs=0), dict(max_seqs=8193), dict(max_pages=0), dict(max_pages=(1 << 22) + 1),
    dict(n_pages=0), dict(n_pages=1 << 27), dict(page_size=8), dict(page_size=48),
    dict(page_size=512), dict(max_tokens=0), dict(max_tokens=(1 << 22) + 1),
    dict(max_pages=1 << 22, page_size=256 * 4)])
def test_table_shapes_are_checked_on_the_host(lib, change):
    n, h = ctypes.c_size_t(5), ctypes.c_void_p(5)
    args = list({**GOOD, **change}.values())
    assert lib.unillm_hip_page_table_bytes(*args, ctypes.byref(n)) == _capi.ERR_INVALID_ARG
    assert n.value == 0 and "page_size 16 / 32" in _capi.last_error()
    assert lib.unillm_hip_page_table_create(*args, None, ctypes.byref(h)) == _capi.ERR_INVALID_ARG
    assert h.value is None


def test_table_bytes(lib):
    n = ctypes.c_size_t()
    assert lib.unillm_hip_page_table_bytes(*GOOD.values(), ctypes.byref(n)) == _capi.OK
    # nine parts on 256-byte boundaries: 32, 4, 20, 5, 4, 4, 64, 64 and 96 ints
    assert n.value == 256 * (8 * 1 + 2)


def test_null_tables_and_caches_are_refused(lib):
    bad = _capi.ERR_INVALID_ARG
    assert lib.unillm_hip_page_table_bytes(*GOOD.values(), None) == bad
    assert lib.unillm_hip_page_table_create(*GOOD.values(), None, None) == bad
    out = ctypes.c_void_p()
    assert lib.unillm_hip_page_table_create(*GOOD.values(), 128, ctypes.byref(out)) == bad
    assert "256-byte aligned" in _capi.last_error()
    assert lib.unillm_hip_page_table_buffers(None, *[None] * 7) == bad
    assert lib.unillm_hip_page_table_clear(None, None) == bad
    assert lib.unillm_hip_page_table_extend(None, None, None, 0, None) == bad
    assert lib.unillm_hip_page_table_truncate(None, None, None, 0, None) == bad
    assert lib.unillm_hip_page_table_check(None, None) == bad
    assert lib.unillm_hip_page_table_destroy(None) == _capi.OK
    assert lib.unillm_hip_paged_kv_destroy(None) == _capi.OK
    assert lib.unillm_hip_paged_kv_buffers(None, None, None, None) == bad
    assert lib.unillm_hip_paged_attention(None, None, None, 0, 1, 1, 0, 0, None, 0, None) == bad
    assert "cache or table is NULL" in _capi.last_error()
    assert lib.unillm_hip_paged_attention_reserve(None, None, 1, 1, None) == bad


@pytest.mark.parametrize("change,status", [
    (dict(kv_type=_capi.Q8_0), _capi.ERR_UNSUPPORTED), (dict(kv_type=99), _capi.ERR_UNSUPPORTED),
    (dict(heads=0), None), (dict(hd=96), None), (dict(hd=0), None), (dict(n_pages=0), None),
    (dict(page=24), None), (dict(theta=0.0), None), (dict(theta=float("nan")), None),
    (dict(theta=float("inf")), None), (dict(k=16), None), (dict(v=16), None), (dict(k=8, v=16), None),
    (dict(heads=65536), None), (dict(heads=40000, hd=256, page=256), None),
    (dict(heads=60000, n_pages=60000), None), (dict(n_pages=1 << 28), None)])
def test_pool_shapes_are_checked_on_the_host(lib, change, status):
    a = {**dict(kv_type=_capi.F16, heads=2, hd=64, n_pages=4, page=16, theta=1e4, k=None, v=None),
         **change}
    out = ctypes.c_void_p(5)
    rc = lib.unillm_hip_paged_kv_create(*a.values(), ctypes.byref(out))
    assert rc == (status or _capi.ERR_INVALID_ARG) and out.value is None
    assert lib.unillm_hip_paged_kv_create(*a.values(), None) == _capi.ERR_INVALID_ARG
