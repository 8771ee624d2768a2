"""CPU-side checks of the C ABI of rotary positions and 8-bit paged caches: every declared symbol is
exported and bound, the Rust block equals the header, and bad arguments are refused on the host before
any GPU work."""
import ctypes
import os
import re

import pytest

from unillm_amd import _capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
KV8_RS = os.path.join(ROOT, "unillm_amd", "rust", "src", "kv8.rs")

C_TO_RUST = {
    "int": "c_int", "int64_t": "i64", "double": "f64", "const double*": "*const f64",
    "const void*": "*const c_void", "void*": "*mut c_void", "void**": "*mut *mut c_void",
    "size_t*": "*mut usize", "const float*": "*const f32", "float*": "*mut f32",
    "const int32_t*": "*const i32", "const unillm_page_table*": "*const unillm_page_table",
    "const unillm_rope*": "*const unillm_rope", "unillm_rope*": "*mut unillm_rope",
    "unillm_rope**": "*mut *mut unillm_rope", "const unillm_paged_kv8*": "*const unillm_paged_kv8",
    "unillm_paged_kv8*": "*mut unillm_paged_kv8", "unillm_paged_kv8**": "*mut *mut unillm_paged_kv8",
}
BAD = _capi.ERR_INVALID_ARG


@pytest.fixture(scope="module")
def lib():
    return _capi.lib()


def test_every_symbol_is_exported_and_bound(lib):
    declared = _capi.header_symbols(_capi.KV8_HEADER)
    assert len(declared) == 10 and sorted(_capi.KV8_SIGNATURES) == declared
    for name in declared:
        assert hasattr(lib, name), name
    assert '#include "unillm_hip_kv8.h"' in open(_capi.HEADER).read()


def test_rust_block_and_constants_equal_header():
    header = re.sub(r"/\*.*?\*/", " ", open(_capi.KV8_HEADER).read(), flags=re.S)
    rust = open(KV8_RS).read()
    want, got = {}, {}
    for ret, name, params in re.findall(r"^\s*(\w+)\s+(unillm_hip_\w+)\s*\(([^)]*)\)\s*;", header, flags=re.M):
        args = []
        for p in " ".join(params.split()).split(","):
            m = re.match(r"^(.*?)(\w+)$", p.strip())
            args.append((m.group(2), C_TO_RUST[re.sub(r"\s*\*", "*", m.group(1).strip())]))
        want[name] = (args, C_TO_RUST[ret])
    block = re.search(r'extern "C" \{(.*?)\n    \}', rust, flags=re.S).group(1)
    for name, params, ret in re.findall(r"pub fn (unillm_hip_\w+)\(([^)]*)\)\s*->\s*([^;]+);", block, flags=re.S):
        args = [tuple(s.strip() for s in p.split(":", 1)) for p in " ".join(params.split()).split(",") if p.strip()]
        got[name] = (args, " ".join(ret.split()))
    assert len(want) == 10 and got == want
    defines = dict(re.findall(r"#define (UNILLM_(?:ROPE|KV8)_\w+) (\d+)", header))
    assert len(defines) == 8 and defines == dict(re.findall(r"pub const (UNILLM_\w+): c_int = (\d+);", rust))
    assert defines["UNILLM_KV8_INT8"] == str(_capi.KV8_INT8) and defines["UNILLM_KV8_E4M3"] == str(_capi.KV8_E4M3)


ROPE = dict(head_dim=128, rotary_dim=64, layout=0, theta=1e4, scaling=0, factor=0.0, low=0.0, high=0.0,
            original=0, factors=None, magnitude=0.0)
NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("change", [
    dict(head_dim=1), dict(head_dim=513), dict(rotary_dim=0), dict(rotary_dim=3), dict(rotary_dim=130),
    dict(rotary_dim=-2), dict(layout=2), dict(layout=-1), dict(theta=1.0), dict(theta=0.0), dict(theta=NAN),
    dict(theta=INF), dict(scaling=4), dict(scaling=-1), dict(magnitude=NAN), dict(magnitude=INF),
    dict(scaling=1), dict(scaling=1, factor=0.5), dict(scaling=1, factor=NAN), dict(scaling=1, factor=INF),
    dict(scaling=2, factor=8.0), dict(scaling=2, factor=8.0, low=1.0, high=1.0, original=8192),
    dict(scaling=2, factor=8.0, low=1.0, high=4.0), dict(scaling=3, factor=8.0, low=0.0, high=4.0, original=1),
    dict(scaling=3, factor=8.0, low=NAN, high=4.0, original=1), dict(scaling=3, factor=8.0, low=1.0, high=INF, original=1),
    dict(factors=(ctypes.c_double * 32)(*[1.0] * 31 + [0.0])), dict(factors=(ctypes.c_double * 32)(*[NAN] + [1.0] * 31))])
def test_rope_shapes_are_checked_on_the_host(lib, change):
    out = ctypes.c_void_p(5)
    rc = lib.unillm_hip_rope_create(*{**ROPE, **change}.values(), ctypes.byref(out))
    assert rc in (BAD, _capi.ERR_UNSUPPORTED) and out.value is None
    assert _capi.last_error().startswith("rope: ")
    assert lib.unillm_hip_rope_create(*{**ROPE, **change}.values(), None) == BAD


@pytest.mark.parametrize("factor", [1e-7, 1e-310])
def test_frequencies_past_2_to_the_20_are_refused(lib, factor):
    out = ctypes.c_void_p(5)
    factors = (ctypes.c_double * 32)(*[factor] + [1.0] * 31)
    assert lib.unillm_hip_rope_create(*{**ROPE, "factors": factors}.values(), ctypes.byref(out)) == BAD
    assert out.value is None and "frequency" in _capi.last_error()


@pytest.mark.parametrize("change", [
    dict(kv_type=0), dict(kv_type=3), dict(kv_type=24), dict(heads=0), dict(heads=65536), dict(hd=96), dict(hd=0),
    dict(hd=512), dict(n_pages=0), dict(n_pages=1 << 28), dict(page=24), dict(page=8), dict(heads=40000, hd=256, page=256),
    dict(heads=60000, n_pages=60000), dict(k=16), dict(k=16, v=1 << 20, ke=1 << 21), dict(ve=16),
    dict(k=8, v=1 << 20, ke=1 << 21, ve=1 << 22), dict(k=16, v=32, ke=1 << 21, ve=1 << 22),
    dict(k=1 << 16, v=1 << 20, ke=1 << 21, ve=1 << 21)])
def test_pool_shapes_are_checked_on_the_host(lib, change):
    a = {**dict(kv_type=1, heads=2, hd=64, n_pages=4, page=16, rope=None, k=None, v=None, ke=None, ve=None), **change}
    out = ctypes.c_void_p(5)
    rc = lib.unillm_hip_paged_kv8_create(*a.values(), ctypes.byref(out))
    assert rc in (BAD, _capi.ERR_UNSUPPORTED) and out.value is None
    assert lib.unillm_hip_paged_kv8_create(*a.values(), None) == BAD


def test_null_handles_are_refused(lib):
    assert lib.unillm_hip_rope_destroy(None) == _capi.OK
    assert lib.unillm_hip_paged_kv8_destroy(None) == _capi.OK
    assert lib.unillm_hip_rope_apply(None, 0, None, 64, 1, 1, None, None, 64, None) == BAD
    assert lib.unillm_hip_paged_kv8_buffers(None, *[None] * 6) == BAD
    assert lib.unillm_hip_paged_kv8_append(None, None, None, 0, 1, None) == BAD
    assert "cache or table is NULL" in _capi.last_error()
    assert lib.unillm_hip_paged_kv8_attention(None, None, None, 0, 1, 1, 1, 0, 0, None, 0, None) == BAD
    assert lib.unillm_hip_paged_kv8_reserve(None, None, 1, 1, None) == BAD
    assert lib.unillm_hip_paged_kv8_read(None, None, None, None, None, 1, 1, 0, None, None, 64, None) == BAD
