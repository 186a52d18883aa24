"""GPU tests of attention over the int8 cache at the ends of what values can be."""
import math

import numpy as np
import pytest

from test_int8_cache_gpu import dev, host, i32, say

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


@pytest.mark.parametrize("batch,heads,dim,nq,kv", [
    (48, 16, 64, 128, 140), (40, 16, 128, 81, 200), (3, 25, 64, 450, 450), (4, 16, 128, 300, 310), (6, 8, 64, 700, 2100),
    (2, 4, 64, 1, 300), (1, 8, 64, 40, 8300)])
def test_values_at_the_largest_number(ops, batch, heads, dim, nq, kv):
    """Every value is fp16's largest number or its negative: so is every result, to 2^-11, and
    none is infinite though the weights' roundings may sum up to more than theirs."""
    say("largest values", batch, heads, dim, nq, kv)
    rng = np.random.default_rng(batch + nq)
    k = (rng.standard_normal((batch, heads, kv, dim)) * 2).astype(np.float16)
    v = np.empty((batch, heads, kv, dim), np.float16)
    v[...] = np.where(np.arange(dim) % 2, 65504, -65504)
    cache = ops.kv_cache_int8(batch, heads, kv, dim)
    ops.kv_append_int8(cache, dev(k), dev(v), list(range(batch)), 0)
    q = (rng.standard_normal((batch, heads, nq, dim)) * 2).astype(np.float16)
    got = host(ops.attention_int8kv(dev(q), cache, list(range(batch)), i32([kv] * batch))).astype(np.float64)
    want = v[0, 0, 0].astype(np.float64)
    assert bool(np.isfinite(got).all())
    assert bool((np.abs(got - want) <= 1.02 * 2.0 ** -10 * 65504).all())
