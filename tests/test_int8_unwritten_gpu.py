"""GPU test: rows of an int8 cache that were never written read as zeros, positive ones."""
import numpy as np
import pytest

from test_int8_cache_gpu import dev, host, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
def test_rows_never_written_read_as_positive_zeros(ops, dim):
    say("never written", dim)
    cache = ops.kv_cache_int8(2, 3, 128, dim)
    x = np.full((1, 3, 2, dim), -1.5, np.float16)
    x[..., 1::2] = 2.0 ** -24                  # (its nearest whole number is 0)
    ops.kv_append_int8(cache, dev(x), dev(x), 1, 70)
    for y in ops.kv_read_int8(cache, [0, 1], 0, 128, 128):
        y = host(y)
        assert np.array_equal(y[1, :, 70:72, ::2], x[0, :, :, ::2]) and not y[1, :, 70:72, 1::2].any()
        y[1, :, 70:72, ::2] = 0
        assert not y.view(np.uint16).any()
