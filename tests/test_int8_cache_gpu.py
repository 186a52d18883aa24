"""GPU tests of the int8 KV cache (kv_append_int8, kv_read_int8) and the attention
over it (attention_int8kv, attention_shared_prefix) against plain 64-bit
implementations in numpy.

Cache contents are compared bit for bit: the definition fixes every byte.

Attention tolerance, from the operator's roundings: a key's weight is rounded to
fp16 once (relative 2^-11, or 2^-25 absolute below fp16's normal range, on weights
of which the heaviest is at least 2^6 and which carry at most the largest value
scale times two), scores are fp32 sums of D products scaled three times (D + 8
roundings of 2^-24 of their absolute terms, in a power of e), and the result is
rounded to fp16 once (2^-11, or 2^-25 absolute):
  |got - want| <= (2^-11 + d) A + N 2^-25 2^-6 2 max|V| + 2^-11 |want| + 2^-25,
  A = sum p |V| / sum p,  d = 2 (D + 8) 2^-24 (max_j sum_d |q_d K_jd| / sqrt(D) + 32)
with 1.02 for the products of these terms and the fp32 sums of p."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def torch():
    import torch as t
    return t


def dev(a):
    return torch().from_numpy(np.ascontiguousarray(a)).cuda()


def i32(values):
    return dev(np.asarray(values, np.int32))


def host(x):
    torch().cuda.synchronize()
    return x.cpu().numpy()


def say(*args):
    print("[case]", *args, flush=True)


def quantise(x):
    """(whole numbers, fp32 scales) of fp16 rows, from the definition."""
    a = np.abs(x.astype(np.float64))
    bad = ~np.isfinite(x).all(-1)
    top = np.where(bad, 0.0, a.max(-1, initial=0.0, where=np.isfinite(a)))
    s = (top / 127.0).astype(np.float32)
    s[top == 0] = 1.0
    with np.errstate(invalid="ignore"):
        c = np.rint(np.where(bad[..., None], 0.0, x.astype(np.float64)) / s.astype(np.float64)[..., None])
    s[bad] = np.nan
    return c, s


def held(x):
    """The values a cache stands for: fp32 products (exact value, and as kv_read gives them)."""
    c, s = quantise(x)
    return c * s.astype(np.float64)[..., None], (c.astype(np.float32) * s[..., None]).astype(np.float16)


def random_rows(rng, *shape):
    x = rng.standard_normal(shape).astype(np.float32)
    x *= np.exp(rng.uniform(-3, 3, shape[:-1]))[..., None]
    return x.astype(np.float16)


def bits(x):
    return np.ascontiguousarray(x).view(np.uint16)


def same(got, want):
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan)
    bad = (got != want) & ~nan  # (-0 equals 0)
    assert not bad.any(), f"{bad.sum()} differ, first at {np.argwhere(bad)[0]}: {got[bad][0]} against {want[bad][0]}"


# ---------------------------------------------------------------- cache
@pytest.mark.parametrize("dim,heads,batch,rows,capacity", [
    (64, 12, 3, 1, 100), (128, 2, 5, 1, 64), (64, 3, 2, 8, 70), (64, 3, 2, 9, 70), (128, 5, 2, 8, 130),
    (64, 2, 2, 64, 200), (64, 1, 3, 65, 300), (128, 3, 2, 130, 333), (64, 25, 1, 200, 257), (128, 1, 1, 1, 1)])
def test_append_then_read(ops, dim, heads, batch, rows, capacity):
    say("append/read", dim, heads, batch, rows, capacity)
    t = torch()
    rng = np.random.default_rng(dim + 7 * heads + rows)
    cache = ops.kv_cache_int8(batch + 2, heads, capacity, dim)
    assert cache.capacity == -(-capacity // 64) * 64
    full = np.zeros((batch + 2, heads, cache.capacity, dim), np.float16)
    full_v = full.copy()
    for turn in range(3):
        k, v = random_rows(rng, batch, heads, rows, dim), random_rows(rng, batch, heads, rows, dim)
        k[0, 0, 0] = 0                              # a row of zeros
        v[-1, -1, -1] = 2.0 ** -24                  # the smallest numbers
        k[-1, 0, -1, :] = 127.0 / 64                # steps of 2^-6: ties at odd multiples of 2^-7
        k[-1, 0, -1, 1:8] = np.array([1, 3, 5, 7, -1, -3, 253], np.float16) / 128
        v[0, 0, 0, :3] = [65504, -65504, 32752]     # the largest, and half of it
        slots = rng.permutation(batch + 2)[:batch].astype(np.int32)
        pos = rng.integers(0, cache.capacity - rows + 1, batch).astype(np.int32)
        lens = rng.integers(0, rows + 1, batch).astype(np.int32) if turn else np.full(batch, rows, np.int32)
        ops.kv_append_int8(cache, dev(k), dev(v), dev(slots), dev(pos), lengths=dev(lens) if turn else None)
        for b in range(batch):
            at = slice(pos[b], pos[b] + lens[b])
            full[slots[b], :, at] = held(k)[1][b, :, :lens[b]]
            full_v[slots[b], :, at] = held(v)[1][b, :, :lens[b]]
        # Every row of the cache, written now, earlier or never.
        gk, gv = ops.kv_read_int8(cache, list(range(batch + 2)), 0, cache.capacity, cache.capacity)
        same(host(gk), full)
        same(host(gv), full_v)
        # A ragged window.
        gk, gv = ops.kv_read_int8(cache, dev(slots), dev(pos), dev(lens), rows)
        for b in range(batch):
            want = full[slots[b], :, pos[b]:pos[b] + rows].copy()
            want_v = full_v[slots[b], :, pos[b]:pos[b] + rows].copy()
            want[:, lens[b]:] = want_v[:, lens[b]:] = 0
            same(host(gk)[b], want)
            same(host(gv)[b], want_v)
    assert t.cuda.current_stream() is not None


def test_every_fp16_value_is_quantised_as_defined(ops):
    """Every finite fp16 number once as a row's value, against maxima of every binade and odd ones."""
    say("quantiser sweep")
    values = np.arange(0x7c00, dtype=np.uint16).view(np.float16)
    rng = np.random.default_rng(3)
    tops = np.concatenate([np.float16(2.0) ** np.arange(-14, 16), rng.choice(values[1024:], 34)]).astype(np.float16)
    rows = np.zeros((64, 1, 512, 64), np.float16)
    for i, top in enumerate(tops):
        # 63 * 512 values at or below the maximum, alternately negative, and the maximum.
        below = values[values <= top]
        pick = below[np.linspace(0, len(below) - 1, 63 * 512).astype(int)].reshape(512, 63)
        rows[i, 0, :, :63] = pick * np.where(np.arange(63) % 2, 1, -1).astype(np.float16)
        rows[i, 0, :, 63] = top
    cache = ops.kv_cache_int8(64, 1, 512, 64)
    order = list(range(64))
    ops.kv_append_int8(cache, dev(rows), dev(rows[:, :, ::-1]), order, 0)
    gk, gv = ops.kv_read_int8(cache, order, 0, 512, 512)
    want = held(rows)[1]
    same(host(gk), want)
    same(host(gv), want[:, :, ::-1])


@pytest.mark.parametrize("rows", [3, 40])
def test_rows_with_infinities_or_nan_read_as_nan(ops, rows):
    say("non-finite rows", rows)
    rng = np.random.default_rng(rows)
    k, v = random_rows(rng, 1, 2, rows, 64), random_rows(rng, 1, 2, rows, 64)
    k[0, 0, 1, 5], k[0, 1, 2, 63], v[0, 1, 0, 0] = np.nan, np.inf, -np.inf
    cache = ops.kv_cache_int8(1, 2, 64, 64)
    ops.kv_append_int8(cache, dev(k), dev(v), 0, 5)
    gk, gv = ops.kv_read_int8(cache, 0, 5, rows, rows)
    same(host(gk), held(k)[1])
    same(host(gv), held(v)[1])
    assert np.isnan(host(gk)[0, 0, 1]).all() and not np.isnan(host(gk)[0, 0, 0]).any()


@pytest.mark.parametrize("rows", [2, 70])
def test_rows_outside_the_cache_are_not_written(ops, rows):
    say("outside", rows)
    rng = np.random.default_rng(rows)
    cache = ops.kv_cache_int8(4, 2, 128, 64)
    base = random_rows(rng, 4, 2, 128, 64)
    ops.kv_append_int8(cache, dev(base), dev(base), [0, 1, 2, 3], 0)
    want = held(base)[1]
    x = random_rows(rng, 7, 2, rows, 64)
    slots = [-1, 4, 2 ** 31 - 1, 0, 1, 2, 3]
    pos = [0, 0, 0, 128, 128 - rows + 1, -1, 2 ** 31 - 1]
    ops.kv_append_int8(cache, dev(x), dev(x), i32(slots), i32(pos))
    got = held(x)[1]
    want[1, :, 128 - rows + 1:] = got[4, :, :rows - 1]
    want[2, :, :rows - 1] = got[5, :, 1:]
    gk, gv = ops.kv_read_int8(cache, [0, 1, 2, 3], 0, 128, 128)
    same(host(gk), want)
    same(host(gv), want)
    gk, gv = ops.kv_read_int8(cache, i32(slots), i32(pos), None, rows)
    expect = np.zeros_like(x)
    expect[4, :, :rows - 1] = want[1, :, 128 - rows + 1:]
    expect[5, :, 1:] = want[2, :, :rows - 1]
    same(host(gk), expect)
    same(host(gv), expect)
    gk, _ = ops.kv_read_int8(cache, i32([0, 1]), i32([0, 0]), i32([-5, 2 ** 31 - 1]), rows)
    assert not host(gk)[0].any()
    same(host(gk)[1], want[1, :, :rows])


@pytest.mark.parametrize("rows", [1, 8, 30])
def test_the_later_of_two_requests_stays(ops, rows):
    say("same token twice", rows)
    rng = np.random.default_rng(rows)
    batch = 70
    cache = ops.kv_cache_int8(3, 2, 128, 64)
    x = random_rows(rng, batch, 2, rows, 64)
    slots = rng.integers(0, 3, batch).astype(np.int32)
    pos = rng.integers(0, 100, batch).astype(np.int32)
    lens = rng.integers(0, rows + 1, batch).astype(np.int32)
    ops.kv_append_int8(cache, dev(x), dev(x), dev(slots), dev(pos), lengths=dev(lens))
    want = np.zeros((3, 2, 128, 64), np.float16)
    for b in range(batch):
        want[slots[b], :, pos[b]:pos[b] + lens[b]] = held(x)[1][b, :, :lens[b]]
    gk, gv = ops.kv_read_int8(cache, [0, 1, 2], 0, 128, 128)
    same(host(gk), want)
    same(host(gv), want)


@pytest.mark.parametrize("dim,heads", [(64, 3), (128, 2)])
@pytest.mark.parametrize("rows", [9, 31, 32, 33, 65, 128])
def test_rows_on_both_sides_of_the_append_rule(ops, dim, heads, rows):
    """Ragged requests that share slots and cross blocks of 64 tokens, in an order that says
    which row stays; what no request writes stays as it was."""
    say("append rule", dim, heads, rows)
    rng = np.random.default_rng(dim + rows)
    cache = ops.kv_cache_int8(4, heads, 192, dim)
    base = random_rows(rng, 4, heads, 192, dim)
    ops.kv_append_int8(cache, dev(base), dev(base[..., ::-1]), [0, 1, 2, 3], 0)
    want_k, want_v = held(base)[1], held(base[..., ::-1])[1]
    slots = np.array([0, 1, 1, 3, 1, 0], np.int32)
    pos = np.array([0, 5, 33, 192 - rows, 63, 64], np.int32)
    lens = np.array([rows, rows, max(rows - 7, 1), rows, 1, 0], np.int32)
    k, v = random_rows(rng, 6, heads, rows, dim), random_rows(rng, 6, heads, rows, dim)
    ops.kv_append_int8(cache, dev(k), dev(v), dev(slots), dev(pos), lengths=dev(lens))
    for b in range(6):
        n = min(lens[b], 192 - pos[b])
        want_k[slots[b], :, pos[b]:pos[b] + n] = held(k)[1][b, :, :n]
        want_v[slots[b], :, pos[b]:pos[b] + n] = held(v)[1][b, :, :n]
    gk, gv = ops.kv_read_int8(cache, [0, 1, 2, 3], 0, 192, 192)
    same(host(gk), want_k)
    same(host(gv), want_v)


# ---------------------------------------------------------------- attention
def reference(q, keys, values, ends):
    """float64 outputs and their tolerance: rows q [R, D] over keys, values [N, D]
    (exact cached values), row r seeing keys [0, ends[r])."""
    n, dim = keys.shape[0], q.shape[1]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for r, end in enumerate(ends):
        if end <= 0:
            continue
        kk, vv = keys[:end], values[:end]
        s = kk @ q[r] / math.sqrt(dim)
        p = np.exp(s - s.max())
        out[r] = p @ vv / p.sum()
        a = p @ np.abs(vv) / p.sum()
        d = 2 * (dim + 8) * 2.0 ** -24 * ((np.abs(kk) @ np.abs(q[r])).max() / math.sqrt(dim) + 32)
        tol[r] = 1.02 * ((2.0 ** -11 + d) * a + end * 2.0 ** -30 * np.abs(vv).max() + 2.0 ** -11 * np.abs(out[r])) + 2.0 ** -25
    return out, tol


class Case:
    """A filled cache and its 64-bit contents."""

    def __init__(self, ops, rng, slots, kv_heads, dim, lengths, capacity=None):
        self.kv_heads, self.dim = kv_heads, dim
        n = capacity or max(max(lengths), 1)
        self.cache = ops.kv_cache_int8(slots, kv_heads, n, dim)
        self.k, self.v = random_rows(rng, slots, kv_heads, n, dim), random_rows(rng, slots, kv_heads, n, dim)
        ops.kv_append_int8(self.cache, dev(self.k), dev(self.v), list(range(slots)), 0)
        self.hk, self.hv = held(self.k)[0], held(self.v)[0]


def check(got, q, case, slots, ends, prefix=None):
    """got, q [B,H,Q,D]; ends[b][i]: keys of the request's own that query i sees."""
    got = host(got).astype(np.float64)
    batch, heads, nq, _ = q.shape
    group = heads // case.kv_heads
    worst = 0.0
    for b in range(batch):
        for h in range(heads):
            g = h // group
            keys, values = case.hk[slots[b], g], case.hv[slots[b], g]
            e = np.asarray(ends[b])
            if prefix:
                slot, n = prefix
                longest = max(int(e.max()), 0)
                keys = np.concatenate([case.hk[slot, g, :n], keys[:longest]])
                values = np.concatenate([case.hv[slot, g, :n], values[:longest]])
                e = np.where(e < 0, 0, n + e)
            want, tol = reference(q[b, h].astype(np.float64), keys, values, e)
            err = np.abs(got[b, h] - want)
            assert np.isfinite(got[b, h]).all()
            assert (err <= tol).all(), f"b {b} h {h}: {np.argwhere(err > tol)[0]} off {err.max():.3g}, {(err / np.maximum(tol, 1e-30)).max():.3g} of the tolerance"
            worst = max(worst, float((err / np.maximum(tol, 1e-30)).max()))
            assert not got[b, h][np.asarray(e) <= 0].any()
    say("  worst share of the tolerance", round(worst, 3))


def ends_of(kv, nq, q_lengths=None, offsets=None, causal=True):
    out = []
    for b, n in enumerate(kv):
        ql = nq if q_lengths is None else q_lengths[b]
        off = n - ql if offsets is None else offsets[b]
        out.append([(max(0, min(n, off + i + 1)) if causal else n) if i < ql else -1 for i in range(nq)])
    return out


@pytest.mark.parametrize("heads,kv_heads,dim,nq,lengths,causal", [
    (12, 12, 64, 1, [1], True), (12, 12, 64, 1, [300], True), (4, 4, 64, 1, [64, 63, 65, 0, 2], True),
    (8, 2, 128, 1, [700, 1, 129], True), (25, 25, 64, 1, [100, 37], False), (6, 1, 128, 1, [515], True),
    (32, 2, 64, 1, [200, 90], True), (34, 2, 64, 1, [200, 90], True), (40, 1, 128, 1, [130], False),
    (96, 1, 64, 1, [70, 300], True), (4, 4, 64, 2, [50, 2, 1], True), (8, 2, 128, 5, [260, 5], True),
    (4, 4, 64, 17, [17, 100], True), (2, 2, 64, 64, [64, 200], False), (2, 2, 128, 33, [33, 100], True),
    (4, 2, 64, 130, [130, 140], True), (3, 3, 64, 257, [257], True), (7, 1, 128, 75, [75, 160], True)])
def test_attention_lengths_and_heads(ops, heads, kv_heads, dim, nq, lengths, causal):
    say("attention", heads, kv_heads, dim, nq, lengths, causal)
    rng = np.random.default_rng(heads * 31 + nq + dim)
    batch = len(lengths)
    case = Case(ops, rng, batch + 1, kv_heads, dim, lengths)
    q = (rng.standard_normal((batch, heads, nq, dim)) * 2).astype(np.float16)
    slots = rng.permutation(batch + 1)[:batch]
    got = ops.attention_int8kv(dev(q), case.cache, i32(slots), i32(lengths), causal=causal)
    check(got, q, case, slots, ends_of(lengths, nq, causal=causal))
    # Host metadata gives the same bits, and so does a second call.
    again = ops.attention_int8kv(dev(q), case.cache, [int(s) for s in slots], lengths, causal=causal)
    assert np.array_equal(bits(host(got)), bits(host(again)))


@pytest.mark.parametrize("batch,heads,kv_heads,dim,length", [(1, 4, 1, 64, 9001), (1, 2, 2, 128, 20000), (3, 8, 4, 64, 4097)])
def test_attention_long_caches(ops, batch, heads, kv_heads, dim, length):
    say("long", batch, heads, kv_heads, dim, length)
    rng = np.random.default_rng(length)
    lengths = [length] + [int(x) for x in rng.integers(1, length, batch - 1)]
    case = Case(ops, rng, batch, kv_heads, dim, lengths)
    q = (rng.standard_normal((batch, heads, 1, dim)) * 3).astype(np.float16)
    got = ops.attention_int8kv(dev(q), case.cache, list(range(batch)), i32(lengths))
    check(got, q, case, range(batch), ends_of(lengths, 1))
    # A bound on the lengths that is too small plans fewer splits; the answer is whole.
    short = ops.attention_int8kv(dev(q), case.cache, list(range(batch)), i32(lengths), max_kv_length=100)
    check(short, q, case, range(batch), ends_of(lengths, 1))


@pytest.mark.parametrize("heads,kv_heads,dim,nq", [(4, 2, 64, 7), (4, 4, 128, 40), (2, 2, 64, 100), (6, 1, 64, 1)])
def test_attention_masks_that_leave_rows_empty(ops, heads, kv_heads, dim, nq):
    say("masks", heads, kv_heads, dim, nq)
    rng = np.random.default_rng(nq + dim)
    lengths = [90, 0, 64, 3, 200, 90]
    q_lengths = [nq, nq, nq // 2, 1, 0, nq]
    offsets = [-3, 0, 63, 500, 0, -10 ** 9]  # negative: the first queries, or all, see nothing
    case = Case(ops, rng, 6, kv_heads, dim, lengths)
    q = (rng.standard_normal((6, heads, nq, dim)) * 2).astype(np.float16)
    for causal in (True, False):
        got = ops.attention_int8kv(dev(q), case.cache, list(range(6)), i32(lengths), q_lengths=i32(q_lengths),
                                   query_offsets=i32(offsets), causal=causal)
        check(got, q, case, range(6), ends_of(lengths, nq, q_lengths, offsets, causal))
    # More queries than keys: the first have none.
    got = ops.attention_int8kv(dev(q), case.cache, list(range(6)), 2)
    check(got, q, case, range(6), ends_of([2] * 6, nq))


def some_of(got, q, case, slots, ends, rng, count, prefix=None):
    """check() for `count` of the (request, head) pairs; all are finite."""
    batch, heads = q.shape[:2]
    assert np.isfinite(host(got)).all()
    group = heads // case.kv_heads
    for _ in range(count):
        b, h = int(rng.integers(batch)), int(rng.integers(heads))
        one = Case.__new__(Case)
        one.kv_heads, one.dim, g = 1, case.dim, h // group
        one.hk, one.hv = case.hk[:, g:g + 1], case.hv[:, g:g + 1]
        check(got[b:b + 1, h:h + 1], q[b:b + 1, h:h + 1], one, [slots[b]], [ends[b]], prefix)


@pytest.mark.parametrize("batch,heads,kv_heads,dim,nq,kv", [
    (48, 16, 16, 64, 128, 140),     # shared tiles
    (40, 32, 8, 128, 81, 200),      # shared tiles, groups of rows that end inside one, 128 dims
    (3, 25, 25, 64, 450, 450),      # two waves to a block of 32 rows
    (6, 8, 8, 64, 700, 2100),       # four waves, long
    (4, 16, 16, 128, 300, 310),     # four waves, 128 dims
    (1, 8, 2, 64, 16, 8300),        # few rows, many keys: two blocks, split
])
def test_attention_plans(ops, batch, heads, kv_heads, dim, nq, kv):
    """Shapes of every way the rows are walked, with ragged lengths, queries and offsets."""
    say("plan", batch, heads, kv_heads, dim, nq, kv)
    rng = np.random.default_rng(batch + nq)
    lengths = [int(x) for x in rng.integers(0, kv + 1, batch)]
    lengths[0], lengths[-1] = kv, kv - 1
    case = Case(ops, rng, batch, kv_heads, dim, [kv])
    q = (rng.standard_normal((batch, heads, nq, dim)) * 2).astype(np.float16)
    slots = rng.permutation(batch)
    got = ops.attention_int8kv(dev(q), case.cache, i32(slots), i32(lengths))
    some_of(got, q, case, slots, ends_of(lengths, nq), rng, 12)
    q_lengths = [int(x) for x in rng.integers(0, nq + 1, batch)]
    offsets = [int(x) for x in rng.integers(-nq // 2, kv, batch)]
    for causal in (True, False):
        got = ops.attention_int8kv(dev(q), case.cache, i32(slots), i32(lengths), q_lengths=i32(q_lengths),
                                   query_offsets=i32(offsets), causal=causal)
        some_of(got, q, case, slots, ends_of(lengths, nq, q_lengths, offsets, causal), rng, 8)
    # A row whose token is not finite reaches only those who see it.
    bad = np.full((1, kv_heads, 1, dim), np.nan, np.float16)
    ops.kv_append_int8(case.cache, dev(bad), dev(bad), int(slots[0]), kv - 2)
    got = host(ops.attention_int8kv(dev(q), case.cache, i32(slots), i32(lengths)))
    sees = np.asarray(ends_of(lengths, nq)[0]) > kv - 2
    assert sees.any() and np.isnan(got[0, :, sees]).all() and np.isfinite(got[0, :, ~sees]).all() and np.isfinite(got[1:]).all()


@pytest.mark.parametrize("batch,heads,kv_heads,dim,nq,prefix,kv", [
    (64, 16, 2, 64, 1, 8200, 40), (30, 24, 8, 128, 1, 700, 100), (2, 8, 8, 64, 40, 300, 8300), (3, 40, 40, 64, 300, 8200, 310)])
def test_shared_prefix_plans(ops, batch, heads, kv_heads, dim, nq, prefix, kv):
    say("prefix plan", batch, heads, kv_heads, dim, nq, prefix, kv)
    rng = np.random.default_rng(batch + prefix)
    lengths = [int(x) for x in rng.integers(0, kv + 1, batch)]
    case = Case(ops, rng, batch + 1, kv_heads, dim, [kv], capacity=max(prefix, kv))
    q = (rng.standard_normal((batch, heads, nq, dim)) * 2).astype(np.float16)
    order = rng.permutation(batch + 1)
    got = ops.attention_shared_prefix(dev(q), case.cache, int(order[-1]), prefix, i32(order[:-1]), i32(lengths),
                                      max_kv_length=kv)
    some_of(got, q, case, order[:-1], ends_of(lengths, nq), rng, 10, prefix=(int(order[-1]), prefix))


@pytest.mark.parametrize("batch,heads,kv_heads,dim,nq,prefix,kv", [
    (64, 32, 8, 128, 1, 4000, 40),      # single tokens, two blocks of rows over the prefix
    (2, 8, 8, 128, 40, 300, 8300),      # two blocks over the own keys alone
    (3, 24, 24, 128, 300, 2000, 310),   # over both
    (5, 6, 2, 64, 33, 2000, 70),
])
def test_shared_prefix_plans_of_more_shapes(ops, batch, heads, kv_heads, dim, nq, prefix, kv):
    test_shared_prefix_plans(ops, batch, heads, kv_heads, dim, nq, prefix, kv)


@pytest.mark.parametrize("prefix", [1, 63, 64, 65, 500])
@pytest.mark.parametrize("heads,kv_heads,dim,nq", [(4, 4, 64, 1), (8, 2, 128, 1), (3, 3, 64, 5), (6, 2, 128, 5), (4, 4, 64, 17)])
def test_short_prefixes(ops, heads, kv_heads, dim, nq, prefix):
    """A prefix that ends inside a tile, own keys from none on, queries that see none of their
    own, requests of slots outside the cache, and a row that is not finite in each."""
    say("short prefix", heads, kv_heads, dim, nq, prefix)
    rng = np.random.default_rng(heads + nq + prefix)
    lengths, kv = [0, 1, 64, 70, 129, 3], 130
    batch = len(lengths)
    case = Case(ops, rng, batch + 1, kv_heads, dim, [kv], capacity=640)
    order = [4, 0, 6, 2, 1, 5]
    q = (rng.standard_normal((batch, heads, nq, dim)) * 2).astype(np.float16)

    def run(**more):
        return ops.attention_shared_prefix(dev(q), case.cache, 3, prefix, i32(order), i32(lengths), max_kv_length=kv, **more)

    check(run(), q, case, order, ends_of(lengths, nq), prefix=(3, prefix))
    q_lengths = [nq, nq - 1, 0, nq, 1, nq]
    offsets = [0, -nq, 5, 200, 60, -1]
    for causal in (True, False):
        got = run(q_lengths=i32(q_lengths), query_offsets=i32(offsets), causal=causal)
        check(got, q, case, order, ends_of(lengths, nq, q_lengths, offsets, causal), prefix=(3, prefix))
    got = host(ops.attention_shared_prefix(dev(q), case.cache, 3, prefix, i32([-1, 7, 99, 2, 2, 2]), i32(lengths), max_kv_length=kv))
    none = host(ops.attention_shared_prefix(dev(q), case.cache, 3, prefix, i32([2] * 6), i32([0, 0, 0] + lengths[3:]), max_kv_length=kv,
                                            causal=False))
    if nq == 1:
        assert np.array_equal(got[:3], none[:3]) and got[:3].any()
    bad = np.full((1, kv_heads, 1, dim), np.nan, np.float16)
    ops.kv_append_int8(case.cache, dev(bad), dev(bad), 2, 69)         # request 3's last key
    got = host(run())
    assert np.isnan(got[3, :, -1]).all() and np.isfinite(np.delete(got, 3, 0)).all() and np.isfinite(got[3, :, :-1]).all()
    ops.kv_append_int8(case.cache, dev(bad), dev(bad), 3, prefix - 1)  # every row's
    assert np.isnan(host(run())).all()
    if prefix < 500:
        ops.kv_append_int8(case.cache, dev(case.k[3:4, :, prefix - 1:prefix]), dev(case.v[3:4, :, prefix - 1:prefix]), 3, prefix - 1)
        ops.kv_append_int8(case.cache, dev(bad), dev(bad), 3, prefix)  # nobody's
        assert np.isfinite(np.delete(host(run()), 3, 0)).all()


@pytest.mark.parametrize("batch,heads,kv_heads,dim,nq,kv", [
    (8, 16, 16, 128, 64, 2000),         # rows for two blocks by their keys
    (2, 25, 25, 64, 90, 3000),
    (1, 8, 1, 128, 1, 40000),           # one pair, as many splits as there may be
    (160, 2, 1, 64, 1, 5000),           # pairs on more than half of the units
])
def test_attention_plans_of_more_shapes(ops, batch, heads, kv_heads, dim, nq, kv):
    say("more plans", batch, heads, kv_heads, dim, nq, kv)
    rng = np.random.default_rng(batch + kv)
    lengths = [int(x) for x in rng.integers(0, kv + 1, batch)]
    lengths[0] = kv
    case = Case(ops, rng, batch, kv_heads, dim, [kv])
    q = (rng.standard_normal((batch, heads, nq, dim)) * 2).astype(np.float16)
    got = ops.attention_int8kv(dev(q), case.cache, list(range(batch)), i32(lengths))
    some_of(got, q, case, range(batch), ends_of(lengths, nq), rng, 10)


@pytest.mark.parametrize("batch,heads,kv_heads,dim,nq,kv,mean", [
    (3, 25, 25, 64, 440, 440, 30.0),    # two waves to a block of 32 rows
    (4, 16, 16, 128, 520, 530, 30.0),   # the same, 128 dims
    (1, 4, 2, 128, 9, 8300, 30.0),      # four waves, split
    (40, 16, 16, 64, 120, 130, 30.0),   # shared tiles
    (2, 3, 3, 128, 1, 200, 30.0),       # single tokens
])
def test_attention_queries_of_one_sign(ops, batch, heads, kv_heads, dim, nq, kv, mean):
    """Queries whose dims share a sign, where sums that start at -1152 sum q run furthest from
    q . c: one rounding per 8 dims of terms up to 1280 sum |q| adds to d of the tolerance
      2 (D / 8) 2^-24 1280 / 127 max|K| sum |q| / sqrt(D)."""
    say("one sign", batch, heads, kv_heads, dim, nq, kv)
    rng = np.random.default_rng(batch + kv)
    case = Case(ops, rng, batch, kv_heads, dim, [kv])
    q = ((rng.standard_normal((batch, heads, nq, dim)) + mean) / (8 * mean)).astype(np.float16)
    got = host(ops.attention_int8kv(dev(q), case.cache, list(range(batch)), [kv] * batch)).astype(np.float64)
    ends = np.asarray(ends_of([kv], nq)[0])
    for _ in range(10):
        b, h = int(rng.integers(batch)), int(rng.integers(heads))
        rows = rng.choice(nq, min(nq, 20), replace=False)
        keys, values = case.hk[b, h * kv_heads // heads], case.hv[b, h * kv_heads // heads]
        x = q[b, h, rows].astype(np.float64)
        want, tol = reference(x, keys, values, ends[rows])
        more = 2 * dim / 8 * 2.0 ** -24 * 1280 / 127 * np.abs(keys).max() * np.abs(x).sum(-1, keepdims=True) / math.sqrt(dim)
        for i, end in enumerate(ends[rows]):
            s = keys[:end] @ x[i] / math.sqrt(dim)
            p = np.exp(s - s.max())
            tol[i] += 1.02 * more[i] * (p @ np.abs(values[:end]) / p.sum())
        err = np.abs(got[b, h, rows] - want)
        assert (err <= tol).all(), f"b {b} h {h}: {(err / tol).max():.3g} of the tolerance"


def test_split_calls_on_two_streams_at_once(ops):
    """Each call has its own workspace."""
    say("two streams")
    t = torch()
    rng = np.random.default_rng(21)
    case = Case(ops, rng, 2, 2, 128, [6000])
    qs = [dev(rng.standard_normal((2, 8, 1, 128)).astype(np.float16)) for _ in range(2)]
    lens, slots = i32([6000, 4321]), i32([0, 1])
    want = [host(ops.attention_int8kv(q, case.cache, slots, lens)) for q in qs]
    t.cuda.synchronize()
    streams = [t.cuda.Stream(), t.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i in (0, 1):
            with t.cuda.stream(streams[i]):
                got[i].append(ops.attention_int8kv(qs[i], case.cache, slots, lens))
    t.cuda.synchronize()
    for i in (0, 1):
        for y in got[i]:
            assert np.array_equal(bits(host(y)), bits(want[i]))


def test_first_calls_of_a_process_can_be_captured():
    """In a fresh process: the first calls ever, among them kernels with more than 64 KiB of
    LDS, inside a capture."""
    import subprocess
    import sys
    say("first calls captured")
    script = """
import torch
from tinyinfer_amd.native_ops import NativeOps
ops = NativeOps()
cache = ops.kv_cache_int8(2, 2, 256, 128)
i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
torch.manual_seed(0)
k, v = torch.randn(2, 2, 200, 128, device="cuda").half(), torch.randn(2, 2, 200, 128, device="cuda").half()
q, x = torch.randn(2, 4, 200, 128, device="cuda").half(), torch.randn(2, 5000, device="cuda")
u, slots, zero, n = torch.rand(2, device="cuda"), i(0, 1), i(0, 0), i(200, 150)
def step():
    ops.kv_append_int8(cache, k, v, slots, zero, lengths=n)
    return (ops.attention_int8kv(q, cache, slots, n), ops.attention_shared_prefix(q, cache, 0, 180, slots, n),
            *ops.kv_read_int8(cache, slots, zero, n, 200), *ops.sample(x, u, top_p=0.9), *ops.sample(x, u, top_k=50))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = step()
for turn in range(3):
    k.normal_(); q.normal_(); u.uniform_()
    graph.replay()
    torch.cuda.synchronize()
    got = [y.clone() for y in out]
    for a, b in zip(got, step()):
        assert torch.equal(a, b)
print("captured")
"""
    from tests.conftest import ROOT
    done = subprocess.run([sys.executable, "-c", script], cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert done.returncode == 0 and "captured" in done.stdout, done.stderr[-2000:]


def test_attention_metadata_outside_the_cache(ops):
    """A slot outside the cache has no keys, lengths are clamped to the capacity and to zero."""
    say("metadata outside")
    rng = np.random.default_rng(8)
    case = Case(ops, rng, 2, 2, 64, [128])
    q = rng.standard_normal((6, 4, 2, 64)).astype(np.float16)
    slots, lengths = [-1, 2, 1, 0, 2 ** 31 - 1, 1], [50, 50, 2 ** 31 - 1, -7, 50, 128]
    got = host(ops.attention_int8kv(dev(q), case.cache, i32(slots), i32(lengths)))
    for b in (0, 1, 3, 4):
        assert not got[b].any()
    check(ops.attention_int8kv(dev(q), case.cache, i32([1] * 6), i32([128] * 6)), q, case, [1] * 6, ends_of([128] * 6, 2))
    want = host(ops.attention_int8kv(dev(q[2:3]), case.cache, i32([1]), i32([128])))
    assert np.array_equal(bits(want[0]), bits(got[2]))
    got = host(ops.attention_int8kv(dev(q), case.cache, i32([1] * 6), i32([128] * 6), q_lengths=i32([-4, 9, 2, 1, 0, 2])))
    assert not got[0].any() and not got[4].any() and not got[3][:, 1:].any()


@pytest.mark.parametrize("nq", [1, 3, 70])
def test_attention_nonfinite_rows_reach_only_those_who_see_them(ops, nq):
    say("non-finite", nq)
    rng = np.random.default_rng(nq)
    case = Case(ops, rng, 2, 2, 64, [150])
    bad = np.full((2, 2, 1, 64), np.inf, np.float16)
    bad[1] = np.nan
    # Token 100 of both slots is not finite: visible to no query of length 100, to the later ones of 101 and more.
    ops.kv_append_int8(case.cache, dev(bad), dev(bad), [0, 1], 100)
    q = rng.standard_normal((2, 4, nq, 64)).astype(np.float16)
    got = ops.attention_int8kv(dev(q), case.cache, [0, 1], 100)
    check(got, q, case, range(2), ends_of([100, 100], nq))
    got = host(ops.attention_int8kv(dev(q), case.cache, [0, 1], 101))
    assert np.isnan(got[:, :, -1]).all()
    if nq > 1:
        check(dev(got[:, :, :-1]), q[:, :, :-1], case, range(2), [e[:-1] for e in ends_of([101, 101], nq)])
    if nq > 1:  # The same tile holds the bad row and the end of what a row sees.
        got = host(ops.attention_int8kv(dev(q), case.cache, [0, 1], 101 + nq - 2))
        assert np.isnan(got[:, :, 1:]).all()
        check(dev(got[:, :, :1]), q[:, :, :1], case, range(2), [[100], [100]])


def test_attention_values_of_every_size(ops):
    """Value scales from fp16's smallest numbers to its largest, rising and falling along the keys."""
    say("value sizes")
    rng = np.random.default_rng(4)
    n = 400
    case = Case(ops, rng, 4, 1, 64, [n])
    size = np.stack([np.geomspace(1e-6, 1e3, n), np.geomspace(1e3, 1e-6, n), np.full(n, 2e-7), np.full(n, 4e4)])
    v = (np.clip(rng.standard_normal((4, 1, n, 64)), -1.6, 1.6) * size[:, None, :, None]).astype(np.float16)
    case.v, case.hv = v, held(v)[0]
    ops.kv_append_int8(case.cache, dev(case.k), dev(v), [0, 1, 2, 3], 0)
    q = (rng.standard_normal((4, 2, 9, 64)) * 0.5).astype(np.float16)
    got = ops.attention_int8kv(dev(q), case.cache, [0, 1, 2, 3], n, causal=False)
    check(got, q, case, range(4), ends_of([n] * 4, 9, causal=False))


def test_attention_scores_of_every_size(ops):
    """Queries from zero to ones whose scores leave a single key, of either sign."""
    say("score sizes")
    rng = np.random.default_rng(5)
    case = Case(ops, rng, 1, 2, 128, [333])
    q = (rng.standard_normal((1, 4, 6, 128)) * np.array([0, 1e-3, 1, 10, 100, 1000])[:, None]).astype(np.float16)
    got = ops.attention_int8kv(dev(q), case.cache, 0, 333, causal=False)
    check(got, q, case, [0], ends_of([333], 6, causal=False))


def test_attention_operands_at_odd_addresses(ops):
    """Contiguous tensors that start at any fp16 element."""
    say("odd addresses")
    t = torch()
    rng = np.random.default_rng(6)
    case = Case(ops, rng, 2, 2, 64, [100])
    flat = t.zeros(2 * 4 * 20 * 64 + 3, dtype=t.float16, device="cuda")
    q = rng.standard_normal((2, 4, 20, 64)).astype(np.float16)
    odd = flat[3:].view(2, 4, 20, 64)
    odd.copy_(dev(q))
    got = ops.attention_int8kv(odd, case.cache, [0, 1], 100)
    check(got, q, case, range(2), ends_of([100, 100], 20))
    x = random_rows(rng, 2, 2, 20, 64)
    src = t.zeros(x.size + 1, dtype=t.float16, device="cuda")[1:].view(x.shape)
    src.copy_(dev(x))
    ops.kv_append_int8(case.cache, src, src, [0, 1], 30)
    gk, _ = ops.kv_read_int8(case.cache, [0, 1], 30, 20, 20)
    same(host(gk), held(x)[1])


def test_cache_beyond_32_bit_offsets(ops):
    """A cache of more than 2^32 bytes of keys, used at its far end."""
    say("far end")
    t = torch()
    rng = np.random.default_rng(7)
    slots, heads, capacity, dim = 9, 8, 1 << 19, 128
    cache = ops.kv_cache_int8(slots, heads, capacity, dim)
    assert slots * heads * capacity * dim > 1 << 32
    n = 200
    k, v = random_rows(rng, 1, heads, n, dim), random_rows(rng, 1, heads, n, dim)
    for at in (0, capacity - n):
        ops.kv_append_int8(cache, dev(k), dev(v), slots - 1, at)
        gk, gv = ops.kv_read_int8(cache, slots - 1, at, n, n)
        same(host(gk), held(k)[1])
        same(host(gv), held(v)[1])
    ops.kv_append_int8(cache, dev(k[:, :, :1]), dev(v[:, :, :1]), slots - 1, capacity - 1)
    # Keys nobody wrote have value 0 and score 0; the written ones at both ends are seen.
    q = (rng.standard_normal((1, heads, 1, dim)) * 2).astype(np.float16)
    got = host(ops.attention_int8kv(dev(q), cache, slots - 1, capacity)).astype(np.float64)
    far_k, far_v = k.copy(), v.copy()
    far_k[:, :, -1], far_v[:, :, -1] = k[:, :, 0], v[:, :, 0]
    for h in range(heads):
        kk = np.concatenate([held(k)[0][0, h], held(far_k)[0][0, h]])
        vv = np.concatenate([held(v)[0][0, h], held(far_v)[0][0, h]])
        s = kk @ q[0, h, 0].astype(np.float64) / math.sqrt(dim)
        top = max(s.max(), 0.0)
        p = np.exp(s - top)
        total = p.sum() + (capacity - 2 * n) * math.exp(-top)
        want, a = p @ vv / total, p @ np.abs(vv) / total
        d = 2 * (dim + 8) * 2.0 ** -24 * ((np.abs(kk) @ np.abs(q[0, h, 0].astype(np.float64))).max() / math.sqrt(dim) + 32)
        # l is an fp32 sum of 2^19 terms, 2^13 to a wave's lane at most: 2^13 roundings.
        tol = 1.02 * ((2.0 ** -11 + d + 2.0 ** -11) * a + 2 * n * 2.0 ** -30 * np.abs(vv).max() + 2.0 ** -11 * np.abs(want)) + 2.0 ** -25
        assert (np.abs(got[0, h, 0] - want) <= tol).all()
    del cache
    t.cuda.empty_cache()


# ---------------------------------------------------------------- shared prefix
@pytest.mark.parametrize("heads,kv_heads,dim,nq,prefix,lengths", [
    (12, 12, 64, 1, 100, [1, 20, 64, 65, 7]), (8, 2, 128, 1, 700, [300, 1, 2]), (4, 4, 64, 1, 1, [5, 1]),
    (4, 4, 64, 1, 63, [0, 1, 0]), (4, 2, 128, 3, 64, [3, 50, 4, 9]), (2, 1, 64, 5, 65, [5, 10] * 8),
    (25, 25, 64, 1, 500, [10] * 40), (2, 2, 64, 1, 4000, [1, 2]), (16, 1, 128, 2, 300, [2, 77]), (3, 3, 64, 1, 0, [4, 0, 90])])
def test_shared_prefix(ops, heads, kv_heads, dim, nq, prefix, lengths):
    say("prefix", heads, kv_heads, dim, nq, prefix, len(lengths))
    rng = np.random.default_rng(prefix + heads)
    batch = len(lengths)
    case = Case(ops, rng, batch + 1, kv_heads, dim, lengths, capacity=max(prefix, max(lengths)))
    order = rng.permutation(batch + 1)
    slots, at = order[:batch], int(order[batch])
    q = (rng.standard_normal((batch, heads, nq, dim)) * 2).astype(np.float16)
    got = ops.attention_shared_prefix(dev(q), case.cache, at, prefix, i32(slots), i32(lengths), max_kv_length=max(lengths))
    ends = ends_of(lengths, nq)
    check(got, q, case, slots, ends, prefix=(at, prefix))
    # Ragged queries: those past q_lengths are 0 although the prefix is there for all.
    q_lengths = [int(x) for x in rng.integers(0, nq + 1, batch)]
    got = ops.attention_shared_prefix(dev(q), case.cache, at, prefix, i32(slots), i32(lengths), q_lengths=i32(q_lengths))
    check(got, q, case, slots, ends_of(lengths, nq, q_lengths), prefix=(at, prefix))


# ---------------------------------------------------------------- streams and graphs
def step_of(ops, cache, q, k, v, slots, pos, lens):
    ops.kv_append_int8(cache, k, v, slots, pos)
    return ops.attention_int8kv(q, cache, slots, lens)


def test_calls_on_another_stream(ops):
    say("side stream")
    t = torch()
    rng = np.random.default_rng(11)
    case = Case(ops, rng, 3, 4, 64, [700])
    q = rng.standard_normal((3, 4, 1, 64)).astype(np.float16)
    want = host(ops.attention_int8kv(dev(q), case.cache, [0, 1, 2], 700))
    side = t.cuda.Stream()
    with t.cuda.stream(side):
        for _ in range(3):
            dq = dev(q)
            got = ops.attention_int8kv(dq, case.cache, [0, 1, 2], 700)
            del dq
            t.zeros(3 * 4 * 64, dtype=t.float16, device="cuda")
    side.synchronize()
    assert np.array_equal(bits(host(got)), bits(want))


def test_two_captured_decode_steps_replayed_in_turn(ops):
    """Append and attention captured with device metadata, twice over two caches; replays
    alternate, with new tokens, lengths and eager work between them."""
    say("graphs")
    t = torch()
    rng = np.random.default_rng(12)
    batch, heads, kv_heads, dim, start = 2, 8, 2, 64, 900
    sets = []
    for _ in range(2):
        case = Case(ops, rng, batch, kv_heads, dim, [1024])
        mirror = Case(ops, rng, batch, kv_heads, dim, [1024])
        mirror.cache.buffer.copy_(case.cache.buffer)
        made = dict(q=t.zeros(batch, heads, 1, dim, dtype=t.float16, device="cuda"),
                    k=t.zeros(batch, kv_heads, 1, dim, dtype=t.float16, device="cuda"),
                    v=t.zeros(batch, kv_heads, 1, dim, dtype=t.float16, device="cuda"),
                    slots=i32([1, 0]), pos=i32([start] * batch), lens=i32([start + 1] * batch))
        step_of(ops, case.cache, **made)
        t.cuda.synchronize()
        graph = t.cuda.CUDAGraph()
        with t.cuda.graph(graph):
            out = step_of(ops, case.cache, **made)
        sets.append((case, mirror, made, graph, out))
    for turn in range(4):
        for case, mirror, made, graph, out in sets:
            for name in ("q", "k", "v"):
                made[name].copy_(dev(rng.standard_normal(made[name].shape).astype(np.float16)))
            made["pos"].fill_(start + 5 * turn)
            made["lens"].copy_(i32([start + 5 * turn + 1, 100 + turn]))
        for _, _, _, graph, _ in sets:
            graph.replay()
        t.cuda.synchronize()
        for case, mirror, made, graph, out in sets:
            want = step_of(ops, mirror.cache, **made)
            assert np.array_equal(bits(host(out)), bits(host(want))), turn
            assert t.equal(case.cache.buffer, mirror.cache.buffer)


def test_host_metadata_is_refused_under_capture(ops):
    say("capture refusal")
    t = torch()
    rng = np.random.default_rng(13)
    case = Case(ops, rng, 1, 2, 64, [100])
    q = dev(rng.standard_normal((1, 2, 1, 64)).astype(np.float16))
    lens = i32([100])
    ops.attention_int8kv(q, case.cache, i32([0]), lens)
    t.cuda.synchronize()
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="captured"):
            ops.attention_int8kv(q, case.cache, 0, lens)
        y = q + 1
    graph.replay()
    t.cuda.synchronize()
    assert t.equal(y, q + 1)


# ---------------------------------------------------------------- as they are used
def test_prompt_then_decode_steps(ops):
    """A prompt is appended and attended to, then single tokens join; every step equals the
    64-bit result over the tokens written so far, with and without a shared prefix."""
    say("prompt and steps")
    rng = np.random.default_rng(14)
    batch, heads, kv_heads, dim, capacity = 3, 6, 3, 64, 160
    lengths = np.array([70, 1, 33])
    case = Case(ops, rng, batch + 1, kv_heads, dim, [capacity])
    k, v = random_rows(rng, batch, kv_heads, 70, dim), random_rows(rng, batch, kv_heads, 70, dim)
    ops.kv_append_int8(case.cache, dev(k), dev(v), [0, 1, 2], 0, lengths=[int(n) for n in lengths])
    for b in range(batch):
        case.hk[b, :, :lengths[b]], case.hv[b, :, :lengths[b]] = held(k)[0][b, :, :lengths[b]], held(v)[0][b, :, :lengths[b]]
    q = rng.standard_normal((batch, heads, 70, dim)).astype(np.float16)
    got = ops.attention_int8kv(dev(q), case.cache, [0, 1, 2], i32(lengths), q_lengths=i32(lengths))
    check(got, q, case, range(batch), ends_of(lengths, 70, lengths))
    for _ in range(5):
        k, v = random_rows(rng, batch, kv_heads, 1, dim), random_rows(rng, batch, kv_heads, 1, dim)
        ops.kv_append_int8(case.cache, dev(k), dev(v), [0, 1, 2], i32(lengths))
        for b in range(batch):
            case.hk[b, :, lengths[b]], case.hv[b, :, lengths[b]] = held(k)[0][b, :, 0], held(v)[0][b, :, 0]
        lengths = lengths + 1
        q = rng.standard_normal((batch, heads, 1, dim)).astype(np.float16)
        check(ops.attention_int8kv(dev(q), case.cache, [0, 1, 2], i32(lengths)), q, case, range(batch), ends_of(lengths, 1))
        got = ops.attention_shared_prefix(dev(q), case.cache, 3, 150, [0, 1, 2], i32(lengths))
        check(got, q, case, range(batch), ends_of(lengths, 1), prefix=(3, 150))


# ---------------------------------------------------------------- refusals
def test_refusals(ops):
    say("refusals")
    t = torch()
    cache = ops.kv_cache_int8(2, 2, 100, 64)
    before = cache.buffer.clone()
    k = t.ones(2, 2, 3, 64, dtype=t.float16, device="cuda")
    q = t.ones(2, 4, 3, 64, dtype=t.float16, device="cuda")
    slots, lens = i32([0, 1]), i32([3, 3])
    bad = [
        (TypeError, lambda: ops.kv_append_int8(None, k, k, slots, 0)),
        (TypeError, lambda: ops.kv_append_int8(cache, k.float(), k, slots, 0)),
        (TypeError, lambda: ops.kv_append_int8(cache, k.transpose(1, 2), k, slots, 0)),
        (TypeError, lambda: ops.kv_append_int8(cache, k, k, slots.long(), 0)),
        (TypeError, lambda: ops.kv_append_int8(cache, k, k, slots.cpu(), 0)),
        (ValueError, lambda: ops.kv_append_int8(cache, k, k[:1], slots, 0)),
        (ValueError, lambda: ops.kv_append_int8(cache, k[:, :1].contiguous(), k, slots, 0)),
        (ValueError, lambda: ops.kv_append_int8(cache, k, k, slots[:1], 0)),
        (ValueError, lambda: ops.kv_append_int8(cache, k, k, None, 0)),
        (ValueError, lambda: ops.kv_append_int8(cache, k, k, slots, None)),
        (ValueError, lambda: ops.kv_append_int8(cache, k, k, [0, 2], 0)),
        (ValueError, lambda: ops.kv_append_int8(cache, k, k, [0, 1], -1)),
        (ValueError, lambda: ops.kv_append_int8(cache, k, k, [0, 1], [0, 126])),
        (ValueError, lambda: ops.kv_append_int8(cache, k, k, [0, 1], 0, lengths=4)),
        (ValueError, lambda: ops.kv_read_int8(cache, [0, 1], 0, 3, 0)),
        (ValueError, lambda: ops.kv_read_int8(cache, [0, 1], [0, 127], [1, 2], 2)),
        (ValueError, lambda: ops.kv_read_int8(cache, None, 0, 3, 3)),
        (ValueError, lambda: ops.attention_int8kv(q[:, :3].contiguous(), cache, slots, lens)),
        (ValueError, lambda: ops.attention_int8kv(q[0], cache, slots, lens)),
        (ValueError, lambda: ops.attention_int8kv(q, cache, None, lens)),
        (ValueError, lambda: ops.attention_int8kv(q, cache, slots, None)),
        (ValueError, lambda: ops.attention_int8kv(q, cache, slots, [129, 1])),
        (ValueError, lambda: ops.attention_int8kv(q, cache, slots, lens, causal=1)),
        (ValueError, lambda: ops.attention_int8kv(q, cache, slots, lens, max_kv_length=-1)),
        (ValueError, lambda: ops.attention_int8kv(q, cache, slots, lens, q_lengths=[4, 0])),
        (ValueError, lambda: ops.attention_int8kv(t.ones(2, 4, 3, 128, dtype=t.float16, device="cuda"), cache, slots, lens)),
        (ValueError, lambda: ops.attention_int8kv(q.clone().requires_grad_(), cache, slots, lens)),
        (ValueError, lambda: ops.attention_shared_prefix(q, cache, 2, 10, slots, lens)),
        (ValueError, lambda: ops.attention_shared_prefix(q, cache, 0, 129, slots, lens)),
        (TypeError, lambda: ops.attention_shared_prefix(q, cache.buffer, 0, 1, slots, lens)),
    ]
    for i, (error, call) in enumerate(bad):
        with pytest.raises(error):
            call()
            pytest.fail(f"call {i} was accepted")
    t.cuda.synchronize()
    assert t.equal(cache.buffer, before)


def test_c_entry_refuses_a_missing_or_small_workspace(ops):
    say("workspace refusal")
    t = torch()
    cache = ops.kv_cache_int8(1, 1, 4096, 64)
    q = t.zeros(1, 1, 1, 64, dtype=t.float16, device="cuda")
    y, meta = t.full_like(q, 7), i32([0])
    lib, at = ops.lib, cache._at
    needed = lib.ti_amd_attention_i8kv_workspace(at, 1, 1, 1, 0, 0)
    assert needed > 0
    stream = t.cuda.current_stream().cuda_stream
    ws = t.empty(needed, dtype=t.uint8, device="cuda")

    def call(pointer, size):
        return lib.ti_amd_attention_i8kv(at, q.data_ptr(), y.data_ptr(), meta.data_ptr(), meta.data_ptr(), None, None,
                                         pointer, size, 1, 1, 1, 0, 1, 0, 0, stream, 0)
    assert call(None, 0) == 1 and call(ws.data_ptr(), needed - 1) == 1 and call(ws.data_ptr() + 4, needed) == 1
    t.cuda.synchronize()
    assert (y == 7).all()
    assert call(ws.data_ptr(), needed) == 0
    t.cuda.synchronize()
    assert not y.any()


def test_a_cache_dropped_while_another_stream_still_reads_it(ops):
    """The allocator waits for every stream that a call used the cache on."""
    say("dropped cache")
    t = torch()
    rng = np.random.default_rng(15)
    n = 4096
    k, v = random_rows(rng, 4, 8, n, 128), random_rows(rng, 4, 8, n, 128)
    q = dev(rng.standard_normal((4, 8, 1, 128)).astype(np.float16))
    slots, lengths = i32([0, 1, 2, 3]), i32([n] * 4)
    dk, dv = dev(k), dev(v)

    def filled():
        cache = ops.kv_cache_int8(4, 8, n, 128)
        ops.kv_append_int8(cache, dk, dv, slots, 0)
        return cache

    cache = filled()
    want = host(ops.attention_int8kv(q, cache, slots, lengths))
    size = cache.buffer.numel()
    del cache
    side = t.cuda.Stream()
    for _ in range(4):
        cache = filled()
        side.wait_stream(t.cuda.current_stream())
        with t.cuda.stream(side):
            for _ in range(20):                # (work in front of the call that counts)
                ops.attention_int8kv(q, cache, slots, lengths)
            got = ops.attention_int8kv(q, cache, slots, lengths)
        del cache
        t.zeros(size, dtype=t.uint8, device="cuda").fill_(255)   # takes the freed block, if it was
        side.synchronize()
        assert np.array_equal(got.cpu().numpy(), want)
