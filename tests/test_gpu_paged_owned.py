"""Page tables and pools whose memory is the library's (the C ABI's NULL storage, which the Rust
crate uses) against those on the caller's tensors."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from unillm_amd import PagedKvCache, PageTable, _capi  # noqa: E402

pytestmark = pytest.mark.gpu

KVH, HD, PAGE = 8, 128, 256
WIDTH = 3 * KVH * HD


def ok(status):
    assert status == _capi.OK, _capi.last_error()


class Owned:
    """A table and a pool of f16 as the C ABI allocates them."""

    def __init__(self, n_pages, kvh=KVH, hd=HD, page=PAGE):
        self.lib, self.t, self.c = _capi.lib(), ctypes.c_void_p(), ctypes.c_void_p()
        ok(self.lib.unillm_hip_page_table_create(4, 4, n_pages, page, 64, None, ctypes.byref(self.t)))
        ok(self.lib.unillm_hip_paged_kv_create(_capi.F16, kvh, hd, n_pages, page, 10000.0, None, None,
                                               ctypes.byref(self.c)))

    def close(self):
        torch.cuda.synchronize()
        ok(self.lib.unillm_hip_paged_kv_destroy(self.c))
        ok(self.lib.unillm_hip_page_table_destroy(self.t))

    def pool(self, elements=None):
        """The first elements (all) of K and of V."""
        k, v, n = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_size_t()
        ok(self.lib.unillm_hip_paged_kv_buffers(self.c, ctypes.byref(k), ctypes.byref(v), ctypes.byref(n)))
        out = []
        for p in (k, v):
            x = np.empty(elements or n.value // 2, np.float16)
            ok(self.lib.unillm_hip_memcpy_dtoh(x.ctypes.data, p, x.nbytes))
            out.append(x)
        return out


def test_a_new_table_and_pool_are_empty():
    o = Owned(9, 2, 64, 16)
    for x in o.pool():
        assert x.size == 9 * 2 * 16 * 64 and not x.any()
    at = [ctypes.c_void_p() for _ in range(7)]
    ok(o.lib.unillm_hip_page_table_buffers(o.t, *[ctypes.byref(p) for p in at]))
    for p, want in zip(at, ([-1] * 16, [0] * 4, list(range(8, -1, -1)), [9], [0] * 5, [-1] * 64, [0] * 64)):
        x = np.empty(len(want), np.int32)
        ok(o.lib.unillm_hip_memcpy_dtoh(x.ctypes.data, p, x.nbytes))
        assert x.tolist() == want
    o.close()


def test_a_new_pool_may_be_used_at_once_on_any_stream():
    # Two pools of 2 GB, whose zeroing takes about a millisecond, and the first step of one issued
    # as soon as the call has returned, on a stream that does not wait for the null stream.
    n_pages, n = 4096, 40
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(n, WIDTH, generator=g).cuda()
    ids, news = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([2, 0], [37, 3]))
    table, cache = PageTable(4, 4, 8, PAGE, 64), PagedKvCache(KVH, HD, 8, PAGE, torch.float16)
    # (the page ids of the large pool, whose stack begins at page 0 as the small one's does)
    table.extend(ids, news)
    want = cache.attention(table, qkv, KVH)
    table.check()
    out = torch.zeros(n, KVH * HD, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    o = Owned(n_pages)
    s = side.cuda_stream
    ok(o.lib.unillm_hip_page_table_extend(o.t, ids.data_ptr(), news.data_ptr(), 2, s))
    ok(o.lib.unillm_hip_paged_attention(o.c, o.t, qkv.data_ptr(), WIDTH, n, KVH, 0, 0, out.data_ptr(),
                                        KVH * HD, s))
    ok(o.lib.unillm_hip_page_table_check(o.t, s))
    torch.cuda.synchronize()
    k, v = o.pool(2 * PAGE * KVH * HD)
    assert (k == cache.k[:2].cpu().numpy().reshape(-1)).all()
    assert (v == cache.v[:2].cpu().numpy().reshape(-1)).all()
    assert torch.equal(out, want)
    o.close()
