"""Refusals of the rotary, paged cache and log probability entry points that need no GPU: extents of
new caches and rotary positions, and the workspace query of the C ABI (every check comes
before the first GPU call)."""
import math

import pytest

torch = pytest.importorskip("torch")

from tinyinfer_amd.native_ops import NativeOps, PagedKVCache, Rotary  # noqa: E402


@pytest.fixture(scope="module")
def cpu_ops():
    return NativeOps()


@pytest.fixture(scope="module")
def cache():
    return PagedKVCache(torch, 5, 2, 64, 64, "cpu")


@pytest.mark.parametrize("args", [(0, 2, 64, 64), (1, 0, 64, 64), (1, 65536, 64, 64), (1, 2, 16, 64), (1, 2, 48, 64), (1, 2, 2048, 64),
                                  (1, 2, 64, 96), (1, 2, 64, True), (1.0, 2, 64, 64), (1, 2, 64.0, 64), (True, 2, 64, 64)])
def test_cache_extents(cpu_ops, args):
    with pytest.raises(ValueError):
        cpu_ops.kv_cache_paged(*args, device="cuda")


def test_nothing_lives_on_the_cpu(cpu_ops):
    with pytest.raises(TypeError):
        cpu_ops.kv_cache_paged(1, 1, 64, 64, device="cpu")
    with pytest.raises(TypeError):
        cpu_ops.rotary(64, device="cpu")


def test_cache_layout_and_that_it_stays(cache):
    import copy
    assert tuple(cache.buffer.shape) == (5, 2 * 2 * 64 * 64) and cache.buffer.dtype == torch.float16
    assert cache._native.pages == cache.buffer.data_ptr() and cache._native.page_count == 5
    for name in ("buffer", "pages", "other"):
        with pytest.raises(AttributeError):
            setattr(cache, name, 1)
    with pytest.raises((TypeError, ValueError, AttributeError)):
        copy.deepcopy(cache)


@pytest.mark.parametrize("rotated,args", [
    (63, {}), (0, {}), (64.0, {}), (True, {}), (1 << 17, {}), (64, {"base": 0}), (64, {"base": math.inf}), (64, {"base": "10000"}),
    (64, {"interleaved": 1}), (64, {"factor": 2.0}), (64, {"scaling": "linear", "factor": 0}), (64, {"scaling": "other"}),
    (64, {"scaling": "parts", "factor": 2.0}), (64, {"scaling": "parts", "factor": 2.0, "original_length": 0}),
    (64, {"scaling": "parts", "original_length": 10, "fast": 1.0, "slow": 1.0}), (64, {"amplitude": math.nan}),
    (4, {"frequencies": [1.0]}), (4, {"frequencies": [1.0, math.inf]}), (4, {"frequencies": [1.0, 0.5], "base": 500.0}),
    (4, {"frequencies": [1.0, 0.5], "scaling": "linear"})])
def test_rotary_arguments(cpu_ops, rotated, args):
    with pytest.raises(ValueError):
        cpu_ops.rotary(rotated, **args)


def test_frequencies_are_held_to_2_pow_minus_64_of_a_turn():
    f = [0.0, 2 * math.pi, math.pi, -math.pi / 2, 1.0, 1e-15]
    r = Rotary(torch, f, False, 1.0, "cpu")
    whole = [x % 2 ** 64 for x in r.turns.tolist()]
    assert whole[:4] == [0, 0, 2 ** 63, 3 * 2 ** 62]
    assert abs(whole[4] / 2 ** 64 - 1 / (2 * math.pi)) < 2 ** -53 and abs(whole[5] - 1e-15 / (2 * math.pi) * 2 ** 64) <= 1
    assert r.rotated == 12
    with pytest.raises(AttributeError):
        r.rotated = 4


def test_workspace_query(cpu_ops, cache):
    query = cpu_ops.lib.ti_amd_attention_paged_workspace
    assert query(cache._at, 4, 2, 4, 1, 0) == 0                       # short caches are not split
    long = query(cache._at, 1000, 2, 4, 1, 0)
    assert long > 0 and long % ((64 + 2) * 4 * 8) == 0                # states of 8 rows
    assert query(cache._at, 1000, 2, 4, 1, 200) == 0                  # the expected lengths plan
    assert query(cache._at, 2 ** 31 - 1, 2, 4, 1, 0) > 0
    for bad in ((0, 2, 4, 1, 0), (4, 0, 4, 1, 0), (4, 65536, 4, 1, 0), (4, 2, 3, 1, 0), (4, 2, 4, 0, 0), (4, 2, 4, 1, -1),
                (4, 2, 4, 2 ** 30, 0), (4, 2, 131072, 1, 0)):
        assert query(cache._at, *bad) == -1
    for name, value in (("page_size", 48), ("page_size", 16), ("page_size", 2048), ("page_count", 0), ("head_dim", 96),
                        ("kv_heads", 0), ("pages", cache._native.pages + 2)):
        held = getattr(cache._native, name)
        setattr(cache._native, name, value)
        try:
            assert query(cache._at, 4, 2, 4, 1, 0) == -1, name
        finally:
            setattr(cache._native, name, held)


def test_operands_on_the_cpu_are_refused(cpu_ops, cache):
    x = torch.zeros((1, 2, 1, 64), dtype=torch.float16)
    table = torch.zeros((1, 1), dtype=torch.int32)
    rotary = Rotary(torch, [1.0] * 16, False, 1.0, "cpu")
    with pytest.raises(TypeError):
        cpu_ops.rotate(x, rotary, 0)
    with pytest.raises(TypeError):
        cpu_ops.rotate(x, None, 0)
    with pytest.raises(TypeError):
        cpu_ops.kv_append_paged(cache, x, x, table, 0)
    with pytest.raises(TypeError):
        cpu_ops.kv_append_paged(None, x, x, table, 0)
    with pytest.raises(TypeError):
        cpu_ops.kv_read_paged(cache, [[0]], 0, 1, 1)
    with pytest.raises(TypeError):
        cpu_ops.attention_paged(x, cache, table, 1)
    with pytest.raises(TypeError):
        cpu_ops.logprobs(torch.zeros((1, 10)), torch.zeros(1, dtype=torch.int32))
