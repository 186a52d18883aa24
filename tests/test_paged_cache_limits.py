"""Paged caches that no call would accept are refused where they are made, before any memory is
taken: pages * kv_heads * page_size of at most 2^34 tokens of a head."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from tinyinfer_amd.native_ops import NativeOps, _KvPaged  # noqa: E402


@pytest.mark.parametrize("pages,kv_heads,page_size,head_dim", [
    ((1 << 24) + 1, 1, 1024, 64), ((1 << 29) + 1, 1, 32, 128), (1 << 20, 65535, 1024, 64), (2 ** 31 - 1, 65535, 32, 64)])
def test_more_than_a_call_accepts(pages, kv_heads, page_size, head_dim):
    ops = NativeOps()
    with pytest.raises(ValueError, match="2\\^34"):
        ops.kv_cache_paged(pages, kv_heads, page_size, head_dim)
    native = _KvPaged(4096, pages, kv_heads, page_size, head_dim)
    query = ops.lib.ti_amd_attention_paged_workspace
    assert query(ctypes.addressof(native), 1, 1, kv_heads, 1, 0) == -1
    native.page_count, native.kv_heads, native.page_size = 1 << 24, 1, 1024  # the largest
    assert query(ctypes.addressof(native), 1, 1, 1, 1, 0) == 0
