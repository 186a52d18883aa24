"""Refusals of the int8 cache and sampling entry points that need no GPU: extents of a
new cache, host metadata against a cache that lives in host memory (every check
comes before the first GPU call), and the workspace query of the C ABI."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from tinyinfer_amd.native_ops import Int8KVCache, NativeOps, _KvI8  # noqa: E402


@pytest.fixture(scope="module")
def cpu_ops():
    return NativeOps()


@pytest.fixture(scope="module")
def cache():
    return Int8KVCache(torch, 3, 2, 100, 64, "cpu")


@pytest.mark.parametrize("args", [(0, 2, 64, 64), (1, 0, 64, 64), (1, 65536, 64, 64), (1, 2, 0, 64), (1, 2, 64, 96),
                                  (1, 2, 64, True), (1.0, 2, 64, 64), (True, 2, 64, 64), (1, 2, 2 ** 31 - 1, 64)])
def test_cache_extents(cpu_ops, args):
    with pytest.raises(ValueError):
        cpu_ops.kv_cache_int8(*args, device="cuda")


def test_cache_on_the_cpu_is_refused(cpu_ops):
    with pytest.raises(TypeError):
        cpu_ops.kv_cache_int8(1, 1, 64, 64, device="cpu")


def test_cache_layout(cache):
    """Four regions one after the other, each 16-byte aligned, filling the buffer."""
    tokens = 3 * 2 * 128
    n = cache._native
    assert cache.capacity == 128 and cache.buffer.numel() == tokens * (2 * 64 + 8)
    assert n.v - n.k == tokens * 64 and n.k_scales - n.v == tokens * 64 and n.v_scales - n.k_scales == 4 * tokens
    assert n.v_scales + 4 * tokens == cache.buffer.data_ptr() + cache.buffer.numel()
    assert all(x % 16 == 0 for x in (n.k, n.v, n.k_scales, n.v_scales))


def test_cache_cannot_be_changed_or_copied(cache):
    """Its native descriptor holds the buffer's address."""
    import copy
    for name in ("buffer", "capacity", "slots", "other"):
        with pytest.raises(AttributeError):
            setattr(cache, name, 1)
    with pytest.raises((TypeError, ValueError, AttributeError)):
        copy.deepcopy(cache)


@pytest.mark.parametrize("args", [
    ([0, 3], 0, 4, 4), ([0, -1], 0, 4, 4), (0, 126, 4, 4), ([0, 1], [0, 1, 2], 4, 4), (0, 0, 5, 4), (0, 0, -1, 4), (0, 0, 4, 0),
    (0, 0, 4, 4.0), (None, 0, 4, 4), (0, None, 4, 4), ([0, 1], [0], 4, 4), (0, 128, 0, 4), (0.5, 0, 4, 4)])
def test_read_refuses_host_metadata(cpu_ops, cache, args):
    with pytest.raises((ValueError, TypeError)):
        cpu_ops.kv_read_int8(cache, *args)


def test_host_tensors_are_refused(cpu_ops, cache):
    x = torch.zeros(1, 2, 1, 64, dtype=torch.float16)
    with pytest.raises(TypeError):
        cpu_ops.kv_append_int8(cache, x, x, 0, 0)
    with pytest.raises(TypeError):
        cpu_ops.attention_int8kv(x, cache, 0, 1)
    with pytest.raises(TypeError):
        cpu_ops.attention_shared_prefix(x, cache, 0, 1, 0, 1)
    with pytest.raises(ValueError):
        cpu_ops.attention_shared_prefix(x, cache, 3, 1, 0, 1)
    with pytest.raises(ValueError):
        cpu_ops.attention_shared_prefix(x, cache, 0, 129, 0, 1)
    with pytest.raises(TypeError):
        cpu_ops.sample(torch.zeros(1, 5), torch.zeros(1))


def test_workspace_query(cpu_ops, cache):
    ask = cpu_ops.lib.ti_amd_attention_i8kv_workspace
    assert ask(cache._at, 1, 2, 1, 0, 0) == 0                      # two tiles: nothing to split
    long = _KvI8(16, 16, 16, 16, 1, 2, 1 << 16, 64)
    at = ctypes.addressof(long)
    whole = ask(at, 1, 2, 1, 0, 0)
    assert whole > 0 and whole % (2 * (64 + 2) * 4) == 0
    assert ask(at, 1, 2, 1, 1 << 20, 0) == whole                   # a bound past the capacity is the capacity
    assert 0 <= ask(at, 1, 2, 1, 64, 0) < whole
    assert ask(at, 4, 2, 1, 64, 0) == 0 == ask(at, 4, 2, 1, 64, 64)  # a short prefix is walked with the own keys,
    assert ask(at, 4, 2, 1, 64, 4096) > 0                           # a long one's states join theirs
    for args in ((0, 2, 1, 0, 0), (1, 3, 1, 0, 0), (1, 0, 1, 0, 0), (1, 2, 0, 0, 0), (65536, 2, 1, 0, 0),
                 (1, 2, 1, -1, 0), (1, 2, 1, 0, -1), (1, 2, 1, 0, (1 << 16) + 1), (65535, 65534, 2, 0, 0)):
        assert ask(at, *args) == -1, args
    for field, value in (("head_dim", 96), ("capacity", 100), ("capacity", 0), ("slots", 0), ("kv_heads", 0), ("k", 8),
                         ("v_scales", None)):
        bad = _KvI8(16, 16, 16, 16, 1, 2, 1 << 16, 64)
        setattr(bad, field, value)
        assert ask(ctypes.addressof(bad), 1, 2, 1, 0, 0) == -1, field
    assert ask(None, 1, 2, 1, 0, 0) == -1
