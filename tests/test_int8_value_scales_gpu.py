"""GPU tests of attention over the int8 KV cache whose values differ in size from token to
token: a row's result is as exact as the values that it weighs, whatever the values of
tokens that it does not see, or weighs next to nothing.

Tolerance: that of test_int8_cache_gpu, but for what weights in fp16's subnormal range
lose.  A row's weights are p_j s_j (s the value's scale) over a power of two that is the
row's own: the heaviest is at least 2^6.  One below 2^-14 is rounded to 2^-25 at most, and
multiplies whole numbers of at most 127, of which the heaviest key's row holds one:
  |got - want| <= 1.02 ((2^-11 + d) A + N 2^-31 max_j(p_j max|V_j|) / sum p + 2^-11 |want|) + 2^-25
with A and d as there: no term has the value of a key without its weight."""
import math

import numpy as np
import pytest

from test_int8_cache_gpu import dev, ends_of, held, host, i32, random_rows, say

pytestmark = pytest.mark.gpu

PLANS = [  # batch, heads, kv_heads, dim, queries, keys: every way the rows are walked
    (3, 4, 4, 64, 1, 200),          # single tokens
    (2, 8, 2, 128, 5, 300),         # a few
    (1, 4, 2, 128, 1, 6000),        # split
    (48, 16, 16, 64, 128, 140),     # shared tiles
    (40, 32, 8, 128, 81, 200),      # shared tiles, 128 dims
    (3, 25, 25, 64, 450, 450),      # two waves to a block of 32 rows
    (6, 8, 8, 64, 700, 2100),       # four waves, long
    (4, 16, 16, 128, 300, 310),     # four waves, 128 dims
    (1, 8, 2, 64, 16, 8300),        # few rows, many keys: two blocks, split
]


def reference(q, keys, values, end):
    """One row: float64 output and tolerance over keys [0, end)."""
    dim = len(q)
    if end <= 0:
        return np.zeros(dim), np.zeros(dim)
    kk, vv = keys[:end], np.abs(values[:end])
    s = kk @ q / math.sqrt(dim)
    p = np.exp(s - s.max())
    total = p.sum()
    want, a = p @ values[:end] / total, p @ vv / total
    d = 2 * (dim + 8) * 2.0 ** -24 * ((np.abs(kk) @ np.abs(q)).max() / math.sqrt(dim) + 32)
    heavy = (p * vv.max(-1)).max() / total
    return want, 1.02 * ((2.0 ** -11 + d) * a + end * 2.0 ** -31 * heavy + 2.0 ** -11 * np.abs(want)) + 2.0 ** -25


class Filled:
    def __init__(self, ops, k, v):
        slots, self.kv_heads, n, dim = k.shape
        self.cache = ops.kv_cache_int8(slots, self.kv_heads, n, dim)
        ops.kv_append_int8(self.cache, dev(k), dev(v), list(range(slots)), 0)
        self.hk, self.hv = held(k)[0], held(v)[0]


def check(got, q, filled, slots, ends, rng, rows, prefix=None):
    """`rows` rows of got [B,H,Q,D]; all are finite."""
    got = host(got).astype(np.float64)
    batch, heads, nq, _ = q.shape
    assert np.isfinite(got).all()
    worst = 0.0
    for n in range(rows):
        b, h, i = int(rng.integers(batch)), int(rng.integers(heads)), int(rng.integers(nq))
        g, end = h * filled.kv_heads // heads, int(ends[b][i])
        keys, values = filled.hk[slots[b], g], filled.hv[slots[b], g]
        if prefix:
            slot, length = prefix
            keys = np.concatenate([filled.hk[slot, g, :length], keys[:max(end, 0)]])
            values = np.concatenate([filled.hv[slot, g, :length], values[:max(end, 0)]])
            end = length + end if end >= 0 else 0
        want, tol = reference(q[b, h, i].astype(np.float64), keys, values, end)
        err = np.abs(got[b, h, i] - want)
        worst = max(worst, float((err / np.maximum(tol, 1e-30)).max()))
        right = bool((err <= tol).all())
        assert right, f"b {b} h {h} q {i} of {end} keys: {(err / tol).max():.3g} of the tolerance"
    say("  worst share of the tolerance", round(worst, 3))


@pytest.mark.parametrize("batch,heads,kv_heads,dim,nq,kv", PLANS)
def test_values_that_a_row_does_not_see(ops, batch, heads, kv_heads, dim, nq, kv):
    """Causal prompts whose later tokens have values 2^23 times as large, in every part of a
    tile; and large values behind the last token that any query sees."""
    say("masked values", batch, heads, kv_heads, dim, nq, kv)
    rng = np.random.default_rng(batch + nq + dim)
    k = random_rows(rng, batch, kv_heads, kv, dim)
    v = (rng.standard_normal((batch, kv_heads, kv, dim)) * 2.0 ** -10).astype(np.float16)
    at = kv - 1 if nq == 1 else kv - 1 - nq // 3  # the first large one: most queries come before it
    v[:, :, at::7] *= np.float16(2.0 ** 12)
    v[:, :, at::7] *= np.float16(2.0 ** 11)
    filled = Filled(ops, k, v)
    q = rng.standard_normal((batch, heads, nq, dim)).astype(np.float16)
    slots = rng.permutation(batch)
    lengths = [kv - 1 if nq == 1 else kv] * batch
    got = ops.attention_int8kv(dev(q), filled.cache, i32(slots), i32(lengths))
    check(got, q, filled, slots, ends_of(lengths, nq), rng, 60)


@pytest.mark.parametrize("batch,heads,kv_heads,dim,nq,kv", PLANS)
def test_values_that_a_row_weighs_next_to_nothing(ops, batch, heads, kv_heads, dim, nq, kv):
    """Every third key is 2^-40 times as heavy as the others, its value up to 2^23 times as large."""
    say("light values", batch, heads, kv_heads, dim, nq, kv)
    rng = np.random.default_rng(batch + nq + dim + 1)
    way = rng.standard_normal(dim)
    way *= math.sqrt(dim) / np.linalg.norm(way)
    k = rng.standard_normal((batch, kv_heads, kv, dim)) * 0.3
    v = rng.standard_normal((batch, kv_heads, kv, dim)) * 2.0 ** -10
    k[:, :, 1::3] -= 28 / math.sqrt(dim) * way         # scores of about -28
    v[:, :, 1::3] *= 2.0 ** rng.integers(10, 24, v[:, :, 1::3].shape[:-1])[..., None]
    filled = Filled(ops, k.astype(np.float16), v.astype(np.float16))
    q = (way + 0.1 * rng.standard_normal((batch, heads, nq, dim))).astype(np.float16)
    slots = rng.permutation(batch)
    got = ops.attention_int8kv(dev(q), filled.cache, i32(slots), [kv] * batch, causal=nq % 2 == 0)
    check(got, q, filled, slots, ends_of([kv] * batch, nq, causal=nq % 2 == 0), rng, 60)


@pytest.mark.parametrize("batch,heads,kv_heads,dim,nq,prefix,kv", [
    (5, 4, 4, 64, 1, 100, 20), (5, 8, 2, 128, 3, 500, 70),   # walked in front of the own keys
    (30, 24, 8, 128, 1, 3000, 100), (3, 24, 24, 128, 300, 2000, 310), (64, 16, 2, 64, 1, 8200, 40)])
def test_values_of_a_prefix_and_of_own_tokens(ops, batch, heads, kv_heads, dim, nq, prefix, kv):
    """Own values 2^23 times the prefix's, for requests that weigh them less and less, and the
    other way round; the last own ones are seen by nobody, or by the last queries alone."""
    say("prefix values", batch, heads, kv_heads, dim, nq, prefix, kv)
    for turn in range(2):
        rng = np.random.default_rng(prefix + turn)
        n = max(prefix, kv)
        way = rng.standard_normal(dim)
        way *= math.sqrt(dim) / np.linalg.norm(way)
        k = rng.standard_normal((batch + 1, kv_heads, n, dim)) * 0.3
        v = rng.standard_normal((batch + 1, kv_heads, n, dim)) * 2.0 ** -10
        large = slice(0, batch) if turn == 0 else slice(batch, batch + 1)
        v[large] *= 2.0 ** 23
        k[large] -= (np.linspace(0, 28, batch) if turn == 0 else np.array([20.0]))[:, None, None, None] / math.sqrt(dim) * way
        filled = Filled(ops, k.astype(np.float16), v.astype(np.float16))
        q = (way + 0.1 * rng.standard_normal((batch, heads, nq, dim))).astype(np.float16)
        lengths = [int(x) for x in rng.integers(0, kv, batch)]
        got = ops.attention_shared_prefix(dev(q), filled.cache, batch, prefix, list(range(batch)), i32(lengths), max_kv_length=kv)
        check(got, q, filled, range(batch), ends_of(lengths, nq), rng, 60, prefix=(batch, prefix))


@pytest.mark.parametrize("batch,heads,kv_heads,dim,nq,kv", PLANS)
@pytest.mark.parametrize("score", [8, 60])
def test_value_rows_of_zeros(ops, score, batch, heads, kv_heads, dim, nq, kv):
    """Heavy tokens whose values are all 0 beside light ones of small values."""
    say("zero values", score, batch, heads, kv_heads, dim, nq, kv)
    rng = np.random.default_rng(batch + nq + dim + score)
    way = rng.standard_normal(dim)
    way *= math.sqrt(dim) / np.linalg.norm(way)
    k = rng.standard_normal((batch, kv_heads, kv, dim)) * 0.3
    v = rng.choice([-1, 1], (batch, kv_heads, kv, dim)) * 2.0 ** -10
    zero = [3, kv // 2, kv - 2] if score == 8 else list(range(64, 128)) + [kv - 1]
    k[:, :, zero] += score / math.sqrt(dim) * way
    v[:, :, zero] = 0
    filled = Filled(ops, k.astype(np.float16), v.astype(np.float16))
    q = (way + 0.1 * rng.standard_normal((batch, heads, nq, dim))).astype(np.float16)
    slots = rng.permutation(batch)
    got = ops.attention_int8kv(dev(q), filled.cache, i32(slots), [kv] * batch, causal=nq > 1)
    check(got, q, filled, slots, ends_of([kv] * batch, nq, causal=nq > 1), rng, 60)
    k[...], v[...] = 1, 0                   # nothing but zeros
    filled = Filled(ops, k.astype(np.float16), v.astype(np.float16))
    assert not host(ops.attention_int8kv(dev(q), filled.cache, i32(slots), [kv] * batch)).any()


@pytest.mark.parametrize("prefix,own", [(200, 50), (4000, 50)])
def test_a_prefix_of_zeros(ops, prefix, own):
    """Zero values, and rows never written, in front of own tokens of small values."""
    say("zero prefix", prefix, own)
    rng = np.random.default_rng(prefix)
    batch, heads, dim = 4, 4, 64
    k = rng.standard_normal((batch + 2, heads, prefix, dim)) * 0.3
    v = rng.choice([-1, 1], (batch + 2, heads, prefix, dim)) * 2.0 ** -10
    v[batch] = 0
    k[batch + 1], v[batch + 1] = 0, 0       # what a slot that was never written stands for
    k, v = k.astype(np.float16), v.astype(np.float16)
    filled = Filled(ops, k, v)
    filled.cache = ops.kv_cache_int8(batch + 2, heads, prefix, dim)
    ops.kv_append_int8(filled.cache, dev(k[:-1]), dev(v[:-1]), list(range(batch + 1)), 0)
    q = rng.standard_normal((batch, heads, 1, dim)).astype(np.float16)
    for slot in (batch, batch + 1):
        got = ops.attention_shared_prefix(dev(q), filled.cache, slot, prefix, [0, 1, 2, 3], own, max_kv_length=own)
        check(got, q, filled, range(batch), ends_of([own] * batch, 1), rng, 16, prefix=(slot, prefix))
        assert not host(ops.attention_shared_prefix(dev(q), filled.cache, slot, prefix, [batch] * 4, own)).any()


@pytest.mark.parametrize("rows", [3, 40])
def test_a_row_of_zeros_has_the_scale_0(ops, rows):
    """fp32_rn(max|x| / 127) as for every other row, negative zeros too; it reads as 0."""
    say("zero scale", rows)
    cache = ops.kv_cache_int8(1, 2, 64, 64)
    x = np.ones((1, 2, rows, 64), np.float16)
    x[0, 0, 1], x[0, 1, 2] = 0.0, -0.0
    ops.kv_append_int8(cache, dev(x), dev(x), 0, 7)
    size = 2 * 64 * 64
    scales = host(cache.buffer)[2 * size:].view(np.float32).reshape(2, 2, 64)[:, :, 7:7 + rows]
    want = np.where(x[0].any(-1), np.float32(1) / np.float32(127), np.float32(0))
    assert np.array_equal(scales[0], want) and np.array_equal(scales[1], want)
    for y in ops.kv_read_int8(cache, 0, 7, rows, rows):
        assert np.array_equal(host(y), np.abs(x)) and not np.signbit(host(y)).any()
