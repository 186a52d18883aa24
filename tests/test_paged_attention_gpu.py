"""GPU tests of attention over the paged fp16 KV cache against a plain 64-bit implementation.

Tolerance, from the operator's roundings: a key's weight is rounded to fp16 once (relative
2^-11, or 2^-25 absolute below fp16's normal range, of weights the heaviest of which is at
least 2^6; single tokens round what is left over once more, which is less), scores are fp32
sums of D products scaled once (D + 8 roundings of 2^-24 of their absolute terms, in a power of
e), and the result is rounded to fp16 once (2^-11, or 2^-25 absolute):
  |got - want| <= (2^-11 + d) A + N 2^-31 max|V| + 2^-11 |want| + 2^-25,
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


def seen_by(q_rows, kv, ql, offset, causal):
    """Number of keys each query sees."""
    ends = []
    for i in range(q_rows):
        if i >= ql:
            ends.append(0)
        elif causal:
            ends.append(max(0, min(kv, (kv - ql if offset is None else offset) + i + 1)))
        else:
            ends.append(kv)
    return ends


def attend(q, k, v, sees):
    """q [Q, D], k, v [N, D], sees [Q, N]: (values, tolerances) in 64 bits; 0 where nothing is seen."""
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    root = math.sqrt(q.shape[1])
    for i in range(len(q)):
        at = np.flatnonzero(sees[i])
        if not len(at):
            continue
        kk, vv = k[at], v[at]
        s = kk @ q[i] / root
        p = np.exp(s - s.max())
        p /= p.sum()
        out[i] = p @ vv
        d = 2 * (q.shape[1] + 8) * 2.0 ** -24 * ((np.abs(kk) @ np.abs(q[i])).max() / root + 32)
        tol[i] = 1.02 * ((2.0 ** -11 + d) * (p @ np.abs(vv)) + len(at) * 2.0 ** -31 * np.abs(vv).max()
                         + 2.0 ** -11 * np.abs(out[i]) + 2.0 ** -25)
    return out, tol


def filled(ops, rng, batch, kv_heads, dim, page, n, scale=1.0):
    """A cache with n tokens of every request, its table and the contents [B, G, n, D]."""
    width = -(-n // page)
    pages = batch * width + 2
    table = rng.permutation(pages)[:batch * width].reshape(batch, width).astype(np.int32)
    cache = ops.kv_cache_paged(pages, kv_heads, page, dim)
    k, v = ((rng.standard_normal((batch, kv_heads, n, dim)) * scale).astype(np.float16) for _ in range(2))
    ops.kv_append_paged(cache, dev(k), dev(v), dev(table), 0)
    return cache, table, k, v


def check(got, q, k, v, kv, ql, offsets, causal):
    group = q.shape[1] // k.shape[1]
    for b in range(q.shape[0]):
        ends = seen_by(q.shape[2], kv[b], ql[b], None if offsets is None else offsets[b], causal)
        sees = np.arange(k.shape[2])[None] < np.array(ends)[:, None]
        for h in range(q.shape[1]):
            want, tol = attend(q[b, h], k[b, h // group], v[b, h // group], sees)
            bad = ~(np.abs(got[b, h] - want) <= tol)
            assert not bad.any(), (b, h, np.argwhere(bad)[0].tolist(), got[b, h][bad][0], want[bad][0], tol[bad][0])


@pytest.mark.parametrize("batch,kv_heads,group,dim,page,q_rows,n", [
    (1, 12, 1, 64, 64, 1, 300), (3, 2, 1, 64, 32, 1, 1), (2, 3, 4, 128, 32, 1, 33), (3, 2, 7, 128, 64, 1, 64),
    (2, 2, 8, 64, 128, 1, 65), (1, 1, 12, 128, 256, 1, 500), (2, 4, 1, 64, 32, 2, 95), (2, 2, 4, 128, 64, 5, 129),
    (1, 2, 5, 64, 32, 7, 161), (2, 3, 1, 128, 32, 40, 100), (1, 2, 2, 64, 1024, 33, 200), (40, 1, 1, 64, 32, 1, 70),
    (1, 1, 16, 64, 64, 1, 2000), (2, 2, 4, 128, 32, 1, 1500), (1, 1, 17, 128, 64, 1, 90), (1, 1, 1, 64, 32, 1, 5000),
    (2, 1, 28, 128, 128, 1, 9000), (1, 1, 1, 128, 64, 1, 17000)])
@pytest.mark.parametrize("causal", [True, False])
def test_against_the_formula(ops, batch, kv_heads, group, dim, page, q_rows, n, causal):
    say("attention", batch, kv_heads, group, dim, page, q_rows, n, causal)
    rng = np.random.default_rng(n + dim)
    cache, table, k, v = filled(ops, rng, batch, kv_heads, dim, page, n)
    q = (rng.standard_normal((batch, kv_heads * group, q_rows, dim)) * 1.5).astype(np.float16)
    kv = rng.integers(max(1, n // 2), n + 1, batch)
    kv[0] = n
    ql = rng.integers(0, q_rows + 1, batch)
    ql[0] = q_rows
    y = ops.attention_paged(dev(q), cache, dev(table), i32(kv), q_lengths=i32(ql), causal=causal)
    check(host(y), q, k, v, kv, ql, None, causal)
    y = ops.attention_paged(dev(q), cache, dev(table), kv.tolist(), causal=causal, max_kv_length=n)
    check(host(y), q, k, v, kv, [q_rows] * batch, None, causal)


@pytest.mark.parametrize("batch,kv_heads,group,dim,page,q_rows,n", [
    (8, 25, 1, 64, 32, 200, 333), (32, 12, 1, 64, 64, 96, 96), (3, 8, 4, 128, 64, 250, 300), (70, 8, 1, 128, 32, 130, 190),
    (1, 2, 3, 64, 256, 900, 1000), (2, 1, 4, 128, 32, 300, 9000)])
def test_prompts(ops, batch, kv_heads, group, dim, page, q_rows, n):
    """Several row blocks, shared tiles; some heads of every request are checked."""
    say("prompts", batch, kv_heads, group, dim, page, q_rows, n)
    rng = np.random.default_rng(n)
    cache, table, k, v = filled(ops, rng, batch, kv_heads, dim, page, n)
    q = (rng.standard_normal((batch, kv_heads * group, q_rows, dim)) * 1.5).astype(np.float16)
    kv, ql = rng.integers(q_rows, n + 1, batch), rng.integers(q_rows // 2, q_rows + 1, batch)
    kv[-1], ql[-1] = n, q_rows
    y = host(ops.attention_paged(dev(q), cache, dev(table), i32(kv), q_lengths=i32(ql)))
    for b in sorted({0, batch // 2, batch - 1}):
        for h in sorted({0, kv_heads * group - 1}):
            sees = np.arange(n)[None] < np.array(seen_by(q_rows, kv[b], ql[b], None, True))[:, None]
            want, tol = attend(q[b, h], k[b, h // group], v[b, h // group], sees)
            bad = ~(np.abs(y[b, h] - want) <= tol)
            assert not bad.any(), (b, h, np.argwhere(bad)[0].tolist())
    # Batches of one walk their rows in other ways: the same values within both roundings.
    alone = host(ops.attention_paged(dev(q[-1:]), cache, dev(table[-1:]), int(kv[-1])))
    assert np.allclose(alone[0].astype(float), y[-1].astype(float), rtol=2e-3, atol=2e-3)


@pytest.mark.parametrize("q_rows", [1, 70])
def test_masks_that_leave_nothing(ops, q_rows):
    """Lengths of zero, offsets before the first key and far behind the last, lengths past the table."""
    say("empty", q_rows)
    rng = np.random.default_rng(1)
    batch, n, page = 6, 150, 32
    cache, table, k, v = filled(ops, rng, batch, 3, 64, page, n)
    q = rng.standard_normal((batch, 6, q_rows, 64)).astype(np.float16)
    kv, ql = [0, 150, 150, 1, -5, 100], [q_rows, q_rows, 0, q_rows, q_rows, q_rows + 9]
    offsets = [0, -30, 0, 2 ** 31 - 100, 5, 40]
    y = host(ops.attention_paged(dev(q), cache, dev(table), i32(kv), q_lengths=i32(ql), query_offsets=i32(offsets)))
    check(y, q, k, v, np.maximum(kv, 0), np.minimum(ql, q_rows), offsets, True)
    assert (y[0] == 0).all() and (y[2] == 0).all() and (y[4] == 0).all()
    # A length past the table: what the table holds (its last page is full of zeros behind n).
    y = host(ops.attention_paged(dev(q), cache, dev(table), i32([2 ** 31 - 1] * batch), causal=False))
    full = [np.concatenate([x, np.zeros((batch, 3, table.shape[1] * page - n, 64), np.float16)], 2) for x in (k, v)]
    check(y, q, *full, [table.shape[1] * page] * batch, [q_rows] * batch, None, False)
    # Causal, with the last 20 tokens past it: queries stay where their lengths put them.
    held = table.shape[1] * page
    y = host(ops.attention_paged(dev(q), cache, dev(table), i32([held + 20] * batch)))
    check(y, q, *full, [held] * batch, [q_rows] * batch, [held + 20 - q_rows] * batch, True)


@pytest.mark.parametrize("dim,q_rows,heads", [(64, 1, 3), (128, 1, 4), (64, 40, 2), (128, 300, 40)])
def test_keys_of_no_weight(ops, dim, q_rows, heads):
    """Scores of -inf: such keys are as if masked, and a row with no others is 0."""
    say("no weight", dim, q_rows, heads)
    rng = np.random.default_rng(dim)
    n = 130
    cache, table, k, v = filled(ops, rng, 1, heads, dim, 32, n)
    q = rng.standard_normal((1, heads, q_rows, dim)).astype(np.float16)
    q[..., 3] = -1
    k[:, :, :70, 3] = np.inf
    ops.kv_append_paged(cache, dev(k), dev(v), dev(table), 0)
    y = host(ops.attention_paged(dev(q), cache, dev(table), n, causal=False))
    sees = np.tile(np.arange(n) >= 70, (q_rows, 1))
    for h in sorted({0, heads - 1}):
        want, tol = attend(q[0, h], k[0, h], v[0, h], sees)
        assert (np.abs(y[0, h] - want) <= tol).all(), h
    assert (host(ops.attention_paged(dev(q), cache, dev(table), 70, causal=False)) == 0).all()


@pytest.mark.parametrize("dim,q_rows,heads", [(64, 1, 12), (128, 1, 4), (64, 40, 2), (128, 300, 40)])
def test_pages_that_are_not_there(ops, dim, q_rows, heads):
    """Tokens on pages outside the cache are not seen: a window that has left its first pages."""
    say("missing pages", dim, q_rows, heads)
    rng = np.random.default_rng(2)
    batch, n, page = 3, 400, 32
    cache, table, k, v = filled(ops, rng, batch, heads, dim, page, n)
    q = rng.standard_normal((batch, heads, q_rows, dim)).astype(np.float16)
    gone = table.copy()
    gone[0, :5] = -1
    gone[1, [1, 3, 12]] = [cache.pages, 2 ** 31 - 1, -2 ** 31]
    gone[2] = -1
    y = host(ops.attention_paged(dev(q), cache, dev(gone), n))
    assert (y[2] == 0).all()
    for b in (0, 1):
        held = np.repeat((gone[b] >= 0) & (gone[b] < cache.pages), page)[:n]
        sees = (np.arange(n)[None] < np.array(seen_by(q_rows, n, q_rows, None, True))[:, None]) & held
        for h in (0, heads - 1):
            want, tol = attend(q[b, h], k[b, h], v[b, h], sees)
            assert (np.abs(y[b, h] - want) <= tol).all(), (b, h)


@pytest.mark.parametrize("dim,q_rows,heads,batch", [(64, 1, 12, 3), (128, 1, 4, 3), (64, 24, 2, 3), (128, 24, 2, 3), (64, 200, 25, 12),
                                                    (128, 200, 10, 12), (128, 200, 12, 12)])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_what_a_row_does_not_see_does_not_count(ops, dim, q_rows, heads, batch, value):
    """Infinities and NaN behind a request's keys, in pages of other requests, and in keys and
    values that only later rows see; those rows are not finite in the dims concerned."""
    say("garbage", dim, q_rows, heads, batch, value)
    rng = np.random.default_rng(dim + q_rows)
    n, page = 260, 32
    cache, table, k, v = filled(ops, rng, batch, heads, dim, page, n + 50)
    kv = rng.integers(q_rows, n, batch)
    q = rng.standard_normal((batch, heads, q_rows, dim)).astype(np.float16)
    spoilt_k, spoilt_v = k.copy(), v.copy()
    for b in range(batch):
        spoilt_k[b, :, kv[b]:], spoilt_v[b, :, kv[b]:] = value, value
    ops.kv_append_paged(cache, dev(spoilt_k), dev(spoilt_v), dev(table), 0)
    cache.buffer[[p for p in range(cache.pages) if p not in table]] = value
    y = host(ops.attention_paged(dev(q), cache, dev(table), i32(kv)))
    some = [(b, h) for b in (0, batch - 1) for h in (0, heads - 1)]
    for b, h in some:
        sees = np.arange(n)[None] < np.array(seen_by(q_rows, kv[b], q_rows, None, True))[:, None]
        want, tol = attend(q[b, h], k[b, h, :n], v[b, h, :n], sees)
        assert (np.abs(y[b, h] - want) <= tol).all(), (b, h)
    if q_rows == 1:
        return
    # The keys of the last 8 rows, one value each, in two dims of the values.
    for b in range(batch):
        spoilt_v[b, :, kv[b] - 8:kv[b], [3, dim - 1]] = value
    ops.kv_append_paged(cache, dev(spoilt_k), dev(spoilt_v), dev(table), 0)
    y = host(ops.attention_paged(dev(q), cache, dev(table), i32(kv)))
    for b, h in some:
        sees = np.arange(n)[None] < np.array(seen_by(q_rows, kv[b], q_rows, None, True))[:, None]
        want, tol = attend(q[b, h], k[b, h, :n], v[b, h, :n], sees)
        hit = np.zeros((q_rows, dim), bool)
        hit[-8:, [3, dim - 1]] = True
        assert not np.isfinite(y[b, h][hit]).any()
        assert (np.abs(y[b, h] - want) <= tol)[~hit].all(), (b, h)
    # A NaN in a key: the rows that see it are NaN, the others as they were.
    ops.kv_append_paged(cache, dev(k), dev(v), dev(table), 0)
    spoilt_k = k.copy()
    for b in range(batch):
        spoilt_k[b, :, kv[b] - 8, 5] = math.nan
    ops.kv_append_paged(cache, dev(spoilt_k), dev(v), dev(table), 0)
    y = host(ops.attention_paged(dev(q), cache, dev(table), i32(kv)))
    for b, h in some:
        sees = np.arange(n)[None] < np.array(seen_by(q_rows, kv[b], q_rows, None, True))[:, None]
        want, tol = attend(q[b, h], k[b, h, :n], v[b, h, :n], sees)
        assert np.isnan(y[b, h, -8:]).all()
        assert (np.abs(y[b, h] - want) <= tol)[:-8].all(), (b, h)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("value", [0.0, math.nan])
def test_a_few_more_row_blocks_than_a_round(ops, dim, causal, value):
    """260 blocks of 128 rows: the last workgroups walk their rows in another way; the tokens of a
    page that is gone and what lies behind the keys do not count for either."""
    say("more than a round", dim, causal, value)
    rng = np.random.default_rng(dim + causal)
    batch, kv_heads, group, q_rows, n, page = 4, 4, 8, 257, 600, 32
    cache, table, k, v = filled(ops, rng, batch, kv_heads, dim, page, n)
    if value:
        behind = np.full((batch, kv_heads, table.shape[1] * page - n, dim), value, np.float16)
        ops.kv_append_paged(cache, dev(behind), dev(behind), dev(table), n)
        cache.buffer[[p for p in range(cache.pages) if p not in table]] = value
    gone = table.copy()
    gone[3, 7] = -1
    q = (rng.standard_normal((batch, kv_heads * group, q_rows, dim)) * 1.5).astype(np.float16)
    ql = [q_rows, 3, 250, q_rows]
    y = host(ops.attention_paged(dev(q), cache, dev(gone), n, q_lengths=i32(ql), causal=causal))
    for b in range(batch):
        held = np.repeat(gone[b] >= 0, page)[:n]
        sees = (np.arange(n)[None] < np.array(seen_by(q_rows, n, ql[b], None, causal))[:, None]) & held
        for h in (0, kv_heads * group - 1):
            want, tol = attend(q[b, h], k[b, h // group], v[b, h // group], sees)
            assert (np.abs(y[b, h] - want) <= tol).all(), (b, h)


@pytest.mark.parametrize("dim,q_rows,n,heads", [(64, 1, 700, 4), (128, 1, 4000, 1), (64, 30, 700, 4), (128, 200, 300, 40)])
def test_not_finite_values_that_rows_see(ops, dim, q_rows, n, heads):
    """In the middle of the keys, however little they weigh; in a query."""
    say("not finite", dim, q_rows, n, heads)
    rng = np.random.default_rng(5)
    cache, table, k, v = filled(ops, rng, 2, heads, dim, 64, n)
    q = rng.standard_normal((2, heads, q_rows, dim)).astype(np.float16)
    v[0, :, 65, 2], v[1, :, 10, dim - 2] = math.inf, math.nan
    k[0, :, 65] = -30 * np.sign(q[0, :, 0])  # next to no weight for the first query
    ops.kv_append_paged(cache, dev(k), dev(v), dev(table), 0)
    q[1, 0, 0, 7] = math.inf
    y = host(ops.attention_paged(dev(q), cache, dev(table), n, causal=False))
    assert not np.isfinite(y[0, :, :, 2]).any() and not np.isfinite(y[1, :, :, dim - 2]).any()
    assert np.isnan(y[1, 0, 0]).all()
    rest = np.delete(y[0], 2, -1)
    assert np.isfinite(rest).all() and np.isfinite(np.delete(y[1, 1:], dim - 2, -1)).all()


@pytest.mark.parametrize("dim,q_rows", [(64, 1), (128, 1), (64, 40), (128, 40)])
def test_extreme_values(ops, dim, q_rows):
    """The largest values have a finite result; scores far apart pick one key; the smallest survive."""
    say("extremes", dim, q_rows)
    rng = np.random.default_rng(6)
    n = 200
    cache, table, k, v = filled(ops, rng, 3, 2, dim, 64, n)
    v[0] = 65504 * rng.choice([-1, 1], (2, 1, dim))
    k[1] *= 40
    v[2] *= 2.0 ** -14
    ops.kv_append_paged(cache, dev(k), dev(v), dev(table), 0)
    q = (rng.standard_normal((3, 2, q_rows, dim)) * np.array([1, 40, 1])[:, None, None, None]).astype(np.float16)
    y = host(ops.attention_paged(dev(q), cache, dev(table), n))
    assert np.isfinite(y).all()
    check(y, q, k, v, [n] * 3, [q_rows] * 3, None, True)


def test_scores_that_rise_all_along(ops):
    """The running reference is raised tile by tile."""
    say("rising")
    rng = np.random.default_rng(7)
    for dim, q_rows in ((64, 1), (128, 1), (64, 20), (128, 20)):
        n = 1000
        cache, table, k, v = filled(ops, rng, 1, 2, dim, 32, n)
        q = np.abs(rng.standard_normal((1, 2, q_rows, dim))).astype(np.float16)
        k = (np.abs(k) * np.linspace(-3, 3, n)[None, None, :, None]).astype(np.float16)
        for kk in (k, k[:, :, ::-1].copy()):
            ops.kv_append_paged(cache, dev(kk), dev(v), dev(table), 0)
            check(host(ops.attention_paged(dev(q), cache, dev(table), n)), q, kk, v, [n], [q_rows], None, True)


def test_equal_calls_give_equal_bits_on_two_streams_and_in_graphs(ops):
    say("graphs")
    t = torch()
    rng = np.random.default_rng(8)
    batch, n = 2, 3000
    cache, table, _, _ = filled(ops, rng, batch, 4, 128, 64, n)
    q = dev(rng.standard_normal((batch, 8, 1, 128)).astype(np.float16))
    table, kv = dev(table), i32([n, 1700])
    want = ops.attention_paged(q, cache, table, kv)
    streams = [t.cuda.Stream(), t.cuda.Stream()]
    graphs, outs = [], []
    for s in streams:
        s.wait_stream(t.cuda.current_stream())
        g = t.cuda.CUDAGraph()
        with t.cuda.graph(g, stream=s):
            outs.append(ops.attention_paged(q, cache, table, kv))
        graphs.append(g)
    t.cuda.synchronize()
    for turn in range(3):
        kv.sub_(100)
        want = ops.attention_paged(q, cache, table, kv)
        t.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with t.cuda.stream(s):
                g.replay()
        t.cuda.synchronize()
        for y in outs:
            assert t.equal(y, want), turn
