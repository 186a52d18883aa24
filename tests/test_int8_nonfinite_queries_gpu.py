"""GPU test: a query row with an infinity or NaN answers NaN wherever it sees a key, as the
definition does (its scores hold an infinity of either sign, or NaN), and 0 where it sees
none; other rows are as without it."""
import numpy as np
import pytest

from test_int8_cache_gpu import bits, dev, ends_of, host, i32, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("batch,heads,kv_heads,dim,nq,kv,prefix", [
    (2, 4, 4, 64, 1, 1, 0), (2, 4, 4, 64, 1, 200, 0), (3, 8, 2, 128, 5, 70, 0), (1, 4, 2, 128, 1, 6000, 0),
    (40, 32, 8, 128, 81, 200, 0), (48, 16, 16, 64, 128, 140, 0), (3, 25, 25, 64, 450, 450, 0), (4, 16, 16, 128, 300, 310, 0),
    (4, 4, 4, 64, 1, 30, 100), (4, 4, 4, 64, 3, 30, 3000), (1, 8, 2, 64, 16, 8300, 0)])
def test_a_query_that_is_not_finite(ops, batch, heads, kv_heads, dim, nq, kv, prefix, value):
    say("query", value, batch, heads, kv_heads, dim, nq, kv, prefix)
    rng = np.random.default_rng(batch + nq)
    n = max(kv, prefix)
    k = rng.standard_normal((batch + 1, kv_heads, n, dim)).astype(np.float16)
    v = rng.standard_normal((batch + 1, kv_heads, n, dim)).astype(np.float16)
    k[..., 5] = np.abs(k[..., 5]) + np.float16(0.5)   # of one sign, and away from 0
    k[..., 6] = -k[..., 5]
    cache = ops.kv_cache_int8(batch + 1, kv_heads, n, dim)
    ops.kv_append_int8(cache, dev(k), dev(v), list(range(batch + 1)), 0)
    q = rng.standard_normal((batch, heads, nq, dim)).astype(np.float16)
    bad = q.copy()
    rows = [(int(rng.integers(batch)), int(rng.integers(heads)), int(rng.integers(nq)), at) for at in (5, 6, 9, dim - 1)]
    for b, h, i, at in rows:
        bad[b, h, i, at] = value
    lengths = [kv] * batch
    lengths[-1] = kv // 2 if batch > 1 else kv        # (in a prompt, queries that see none of their own)

    def run(x):
        if prefix:
            return host(ops.attention_shared_prefix(dev(x), cache, batch, prefix, list(range(batch)), i32(lengths), max_kv_length=kv))
        return host(ops.attention_int8kv(dev(x), cache, list(range(batch)), i32(lengths)))

    want, got, ends = run(q), run(bad), ends_of(lengths, nq)
    assert np.isfinite(want).all()
    for b, h, i in {row[:3] for row in rows}:
        if prefix or ends[b][i] > 0:
            assert bool(np.isnan(got[b, h, i]).all()), (b, h, i)
        else:
            assert not got[b, h, i].any()
        got[b, h, i] = want[b, h, i]
    assert np.array_equal(bits(got), bits(want))
