"""Buffers of the paged calls that share memory are refused on the host."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from unillm_amd import HipError, PagedKvCache, PageTable, _capi  # noqa: E402

K = 1 << 20
BYTES = 4 * 2 * 64 * 64 * 2  # 4 pages of 64, 2 heads of 64, f16


@pytest.mark.parametrize("v", [K, K + 16, K + BYTES - 16, K - 16, K - BYTES + 16])
def test_pools_whose_k_and_v_share_memory(v):
    out = ctypes.c_void_p(5)
    rc = _capi.lib().unillm_hip_paged_kv_create(_capi.F16, 2, 64, 4, 64, 1e4, K, v, ctypes.byref(out))
    assert rc == _capi.ERR_INVALID_ARG and out.value is None
    assert "must not share memory" in _capi.last_error()


@pytest.mark.gpu
def test_one_tensor_for_k_and_v():
    both = torch.zeros(8, 2, 64, 64, dtype=torch.float16, device="cuda")
    with pytest.raises(HipError, match="must not share memory"):
        PagedKvCache(2, 64, 8, 64, torch.float16, k=both, v=both)
    PagedKvCache(2, 64, 4, 64, torch.float16, k=both[:4], v=both[4:])  # (beside each other)


@pytest.mark.gpu
def test_rows_in_the_pool_or_the_table():
    table = PageTable(1, 4, 8, 64, 64)
    mem = torch.zeros(2, 8 * 2 * 64 * 64, device="cuda")
    cache = PagedKvCache(2, 64, 8, 64, torch.float32, k=mem[0].view(8, 2, 64, 64), v=mem[1].view(8, 2, 64, 64))
    table.extend(*(torch.tensor([x], dtype=torch.int32, device="cuda") for x in (0, 3)))
    qkv = torch.randn(3, 6 * 64, device="cuda")
    for part in mem:
        with pytest.raises(HipError, match="must not share memory with the pool"):
            cache.attention(table, qkv, 2, out=part[-3 * 128:].view(3, 128))
        with pytest.raises(HipError, match="must not share memory with the pool"):
            cache.attention(table, part[:3 * 6 * 64].view(3, 6 * 64), 2)
    with pytest.raises(HipError, match="must not share memory with the table"):
        cache.attention(table, qkv[:1], 2, out=table._mem[:512].view(torch.float32).view(1, 128))
    assert not mem.any()
    assert torch.isfinite(cache.attention(table, qkv, 2)).all()
    table.check()
