"""GPU tests of attention over the int8 cache with scores far from 0: finite queries, keys and
values have finite answers, which lie between the values of the keys that count."""
import numpy as np
import pytest

from test_int8_cache_gpu import dev, host, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch,kv_heads,group,dim,q_rows,n", [
    (2, 3, 1, 64, 1, 200), (2, 3, 4, 128, 5, 200), (1, 2, 4, 64, 2, 4000), (16, 25, 1, 64, 200, 333), (16, 16, 1, 128, 300, 310)])
def test_scores_that_are_near_each_other(ops, batch, kv_heads, group, dim, q_rows, n):
    """Two keys in different tiles with scores of 1e7 to 1e9 that differ by a few units, the others far
    below them, and value scales of 1 and more."""
    say("near", batch, kv_heads, group, dim, q_rows, n)
    rng = np.random.default_rng(9)
    heads = kv_heads * group
    cache = ops.kv_cache_int8(batch, kv_heads, n, dim)
    v = rng.integers(-127, 128, (batch, kv_heads, n, dim)).astype(np.float16)
    v[..., 5], v[..., 6] = 127, -127
    first, second = n // 5, n - 1 - n // 7
    q = np.zeros((batch, heads, q_rows, dim), np.float16)
    q[..., 0] = 16384 + 16 * rng.integers(0, 512, q.shape[:3])
    q[..., 1] = rng.integers(1, 64, q.shape[:3]) / 16
    for size in (1, 16):
        low, high = (np.repeat(f(v[:, :, first], v[:, :, second]).astype(float) * size, group, 1)[:, :, None] for f in (np.minimum, np.maximum))
        for big in (1024, 8128, 16256, 32512, 60960):  # 127 times these whole numbers, whose scale is exact
            for at, other in ((first, second), (second, first)):
                k = np.zeros((n, dim), np.float16)
                k[:, 0], k[[at, other], 0], k[other, 1] = -big, big, big / 127
                k = np.broadcast_to(k, v.shape).copy()
                ops.kv_append_int8(cache, dev(k), dev(v * np.float16(size)), list(range(batch)), 0)
                y = host(ops.attention_int8kv(dev(q), cache, list(range(batch)), n, causal=False)).astype(float)
                # (Two roundings to fp16, of a weight and of the answer, of 2^-11 each.)
                slack = 2.0 ** -9 * 127 * size
                assert ((y >= low - slack) & (y <= high + slack)).all(), (size, big, at)
