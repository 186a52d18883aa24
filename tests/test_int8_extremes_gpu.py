"""GPU tests of attention over the int8 cache at the ends of what values can be."""
import math

import numpy as np
import pytest

from test_int8_cache_gpu import dev, host, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,nq,kv,token,prefix", [
    (64, 1, 256, 5, 0), (128, 1, 256, 70, 0), (64, 1, 6000, 64 * 40 + 3, 0), (128, 1, 6000, 3, 0),
    (64, 450, 900, 5, 0), (128, 300, 700, 130, 0), (64, 1, 30, 70, 200), (128, 2, 30, 70, 5000)])
def test_a_value_of_nan_that_weighs_nothing(ops, dim, nq, kv, token, prefix):
    """The keys of one tile, a value of which is NaN, are e^-200 as heavy as the others: every
    row that sees it is NaN, whichever wave or workgroup has the tile."""
    say("light NaN", dim, nq, kv, token, prefix)
    rng = np.random.default_rng(dim + nq)
    n, heads = max(kv, prefix), 25 if nq == 450 else 2
    way = rng.standard_normal(dim)
    way *= math.sqrt(dim) / np.linalg.norm(way)
    k = rng.standard_normal((2, heads, n, dim)) * 0.3
    at = token // 64 * 64
    k[:, :, at:at + 64] -= 200 / math.sqrt(dim) * way
    v = rng.standard_normal((2, heads, n, dim))
    v[1 if prefix else 0, :, token, 3] = np.nan
    cache = ops.kv_cache_int8(2, heads, n, dim)
    ops.kv_append_int8(cache, dev(k.astype(np.float16)), dev(v.astype(np.float16)), [0, 1], 0)
    q = (way + 0.1 * rng.standard_normal((1, heads, nq, dim))).astype(np.float16)
    if prefix:
        got = host(ops.attention_shared_prefix(dev(q), cache, 1, prefix, 0, kv))
    else:
        got = host(ops.attention_int8kv(dev(q), cache, 0, kv))
    assert bool(np.isnan(got).all())
