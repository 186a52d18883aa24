"""GPU tests of attention over the paged fp16 KV cache at extents that reach every way its rows
and keys are walked, with scores that stress the running reference of the exponents.

The formula and its tolerance are those of test_paged_attention_gpu.py.  Where scores are so far
apart that a row's weights are 1 or 0, its answer is one key's values, or the mean of a few: a
weight w cancels but for the fp32 roundings of its sum, its reciprocal and their product (2^-22 of
the values' sizes at most), less than half a step of fp16, so one key's values come back as they
are and the mean of two is off by half a step, 2^-11, and 2^-21 of the sizes."""
import numpy as np
import pytest

from test_paged_attention_gpu import attend, dev, host, i32, say, seen_by, torch

pytestmark = pytest.mark.gpu

# (batch, kv_heads, group, dim, page, q_rows, keys): blocks of 16 rows whole, cut in parts and in three;
# two blocks whole, cut in parts and in three; tiles shared by 128 rows, of more blocks than CUs and of fewer;
# and with the first row blocks of a pair, one or two of them, by waves of two.
WALKS = {
    "one 64": (2, 3, 1, 64, 32, 1, 200), "one 128": (2, 3, 1, 128, 32, 5, 200),
    "one cut 64": (1, 2, 4, 64, 64, 1, 4000), "one cut 128": (1, 2, 4, 128, 64, 2, 2100),
    "one in three 128": (12, 11, 1, 128, 64, 1, 4100), "one in three 64": (12, 11, 2, 64, 64, 1, 4100),
    "two 64": (13, 10, 1, 64, 64, 32, 1300), "two 128": (13, 10, 4, 128, 32, 8, 300),
    "two cut 64": (1, 2, 16, 64, 128, 19, 9100), "two cut 128": (2, 1, 16, 128, 128, 19, 13500),
    "two in three 64": (9, 4, 4, 64, 64, 25, 4200), "two in three 128": (9, 4, 4, 128, 64, 25, 4200),
    "shared 64": (8, 16, 1, 64, 64, 512, 640), "shared 128": (8, 16, 1, 128, 64, 512, 640),
    "mixed 64": (4, 4, 8, 64, 32, 257, 600), "mixed 128": (4, 4, 8, 128, 32, 257, 600),
    "two mixed 64": (4, 4, 8, 64, 64, 288, 1100), "two mixed 128": (4, 4, 8, 128, 64, 288, 1100),
    "ragged mixed 64": (5, 8, 1, 64, 64, 900, 1100), "ragged mixed 128": (5, 8, 1, 128, 64, 900, 1100),
    "few shared 64": (3, 16, 1, 64, 64, 450, 640), "few shared 128": (3, 16, 1, 128, 64, 450, 640)}
walks = pytest.mark.parametrize("walk", WALKS)


def filled(ops, rng, batch, kv_heads, dim, page, n):
    """A cache with n tokens of every request, its table and the contents [B, G, n, D]: of one row of
    tokens a head, those from another place on for every request."""
    width = -(-n // page)
    table = rng.permutation(batch * width + 2)[:batch * width].reshape(batch, width).astype(np.int32)
    cache = ops.kv_cache_paged(batch * width + 2, kv_heads, page, dim)
    k, v = (np.stack([x[:, b:b + n] for b in range(batch)])
            for x in rng.standard_normal((2, kv_heads, n + batch, dim), np.float32).astype(np.float16))
    ops.kv_append_paged(cache, dev(k), dev(v), dev(table), 0)
    return cache, table, k, v


def check_some(y, q, k, v, kv, ql, causal, batches=None):
    """Some heads of some requests against the formula."""
    batch, heads, q_rows, _ = q.shape
    group, n = heads // k.shape[1], k.shape[2]
    for b in batches or sorted({0, batch - 1}):
        for h in sorted({0, heads - 1}):
            sees = np.arange(n)[None] < np.array(seen_by(q_rows, kv[b], ql[b], None, causal))[:, None]
            want, tol = attend(q[b, h], k[b, h // group], v[b, h // group], sees)
            bad = ~(np.abs(y[b, h] - want) <= tol)
            assert not bad.any(), (b, h, np.argwhere(bad)[0].tolist(), y[b, h][bad][0], want[bad][0], tol[bad][0])


@walks
def test_ragged_lengths(ops, walk):
    """Full and short requests and one without a key, causal and not; equal calls give equal bits."""
    batch, kv_heads, group, dim, page, q_rows, n = WALKS[walk]
    say("ragged", walk)
    rng = np.random.default_rng(n + dim)
    cache, table, k, v = filled(ops, rng, batch, kv_heads, dim, page, n)
    q = (rng.standard_normal((batch, kv_heads * group, q_rows, dim)) * 1.5).astype(np.float16)
    kv = rng.integers(1, n + 1, batch)
    kv[-1], kv[batch // 3], ql = 65, 0, np.maximum(rng.integers(q_rows // 2, q_rows + 1, batch), 1)
    kv[0], ql[0] = n, q_rows
    for causal in (False, True):
        x = dev(q), cache, dev(table), i32(kv)
        y = ops.attention_paged(*x, q_lengths=i32(ql), causal=causal)
        for _ in range(3):
            assert torch().equal(ops.attention_paged(*x, q_lengths=i32(ql), causal=causal), y)
        check_some(host(y), q, k, v, kv, ql, causal, sorted({0, batch // 3, batch - 1}))


@walks
def test_scores_that_rise_and_fall(ops, walk):
    """The running reference is raised tile by tile, or never again."""
    batch, kv_heads, group, dim, page, q_rows, n = WALKS[walk]
    say("rising", walk)
    rng = np.random.default_rng(7)
    cache, table, k, v = filled(ops, rng, batch, kv_heads, dim, page, n)
    q = np.abs(rng.standard_normal((batch, kv_heads * group, q_rows, dim))).astype(np.float16)
    k = (np.abs(k) * np.linspace(-3, 3, n)[None, None, :, None]).astype(np.float16)
    for kk in (k, k[:, :, ::-1].copy()):
        ops.kv_append_paged(cache, dev(kk), dev(v), dev(table), 0)
        y = host(ops.attention_paged(dev(q), cache, dev(table), n, causal=False))
        check_some(y, q, kk, v, [n] * batch, [q_rows] * batch, False)


@walks
def test_values_of_any_size(ops, walk):
    """The largest values have a finite result; scores far apart pick one key; the smallest survive."""
    batch, kv_heads, group, dim, page, q_rows, n = WALKS[walk]
    say("sizes", walk)
    rng = np.random.default_rng(6)
    cache, table, k, v = filled(ops, rng, batch, kv_heads, dim, page, n)
    q = rng.standard_normal((batch, kv_heads * group, q_rows, dim)).astype(np.float16)
    for size, far in ((65504.0, 1), (1.0, 40), (2.0 ** -14, 1)):
        vv = v * np.float16(size) if size < 2 else (size * rng.choice([-1, 1], (batch, kv_heads, 1, dim))).astype(np.float16)
        vv = np.broadcast_to(vv, v.shape).copy()
        kk, qq = k * np.float16(far), q * np.float16(far)
        ops.kv_append_paged(cache, dev(kk), dev(vv), dev(table), 0)
        y = host(ops.attention_paged(dev(qq), cache, dev(table), n, causal=False))
        assert np.isfinite(y).all(), size
        check_some(y, qq, kk, vv, [n] * batch, [q_rows] * batch, False)


@walks
def test_scores_of_any_size(ops, walk):
    """Scores from thousands to 5e10: one key, two equal ones, rising ones, two that are near."""
    t = torch()
    batch, kv_heads, group, dim, page, q_rows, n = WALKS[walk]
    say("scores", walk)
    rng = np.random.default_rng(8)
    cache, table, _, v = filled(ops, rng, batch, kv_heads, dim, page, n)
    table, v = dev(table), dev(v)
    signs = rng.choice([-1.0, 1.0], dim)
    # Whole numbers of at most 7 bits times a power of two: products and sums of these are exact in fp32.
    rows = rng.integers(64, 128, (batch, kv_heads * group, q_rows, 1)) * signs

    def answers(keys, scale):
        """keys [n]: signs * keys, times scale, as queries are."""
        k = t.from_numpy((keys[:, None] * signs * scale).astype(np.float16)).cuda().expand(batch, kv_heads, n, dim)
        ops.kv_append_paged(cache, k, v, table, 0)
        return ops.attention_paged(dev((rows * scale).astype(np.float16)), cache, table, n, causal=False)

    def values(at):
        return v[:, :, at].repeat_interleave(group, 1)[:, :, None]

    first, second = n // 5, n - 1 - n // 7
    for power in range(-2, 10):  # scores x = sqrt(dim) log2(e) 2^(12 + 2 power) and up
        scale, below = 2.0 ** power, np.full(n, -64.0)
        keys = below.copy()
        keys[first] = 100
        assert t.equal(answers(keys, scale), values(first).expand(-1, -1, q_rows, -1)), (power, "one")
        keys[second] = 100
        y, a, b = answers(keys, scale).double(), values(first).double(), values(second).double()
        off, tol = (y - (a + b) / 2).abs(), 2.0 ** -11 * ((a + b) / 2).abs() + 2.0 ** -21 * (a.abs() + b.abs()) + 2.0 ** -25
        assert (off <= tol).all(), (power, "two", off.max().item())
        rising = np.floor(np.linspace(-127, 126, n))
        rising[-1] = 127
        for keys, at in ((rising, n - 1), (rising[::-1], 0)):
            assert t.equal(answers(keys, scale), values(at).expand(-1, -1, q_rows, -1)), (power, "rising")


@walks
def test_far_scores_that_are_near_each_other(ops, walk):
    """Two keys in different tiles with scores of 1e7 to 1e9 that differ by a few units: weights are what
    fp32 scores make of them, and answers lie between the two keys' values."""
    t = torch()
    batch, kv_heads, group, dim, page, q_rows, n = WALKS[walk]
    say("near", walk)
    rng = np.random.default_rng(9)
    cache, table, _, v = filled(ops, rng, batch, kv_heads, dim, page, n)
    table, v = dev(table), dev(v)
    first, second = n // 5, n - 1 - n // 7
    low, high = (f(v[:, :, first], v[:, :, second]).float().repeat_interleave(group, 1)[:, :, None]
                 for f in (t.minimum, t.maximum))
    slack = 2.0 ** -10 * t.maximum(low.abs(), high.abs()) + 2.0 ** -24
    q = np.zeros((batch, kv_heads * group, q_rows, dim), np.float16)
    q[..., 0] = 16384 + 16 * rng.integers(0, 512, q.shape[:3])
    q[..., 1] = rng.integers(1, 9, q.shape[:3])
    for big in (4096, 16384, 50000):
        for step in (1, 4, 16, 64):
            for at, other in ((first, second), (second, first)):
                k = np.zeros((n, dim), np.float16)
                k[:, 0], k[[at, other], 0], k[other, 1] = -big, big, step
                ops.kv_append_paged(cache, dev(k).expand(batch, kv_heads, n, dim), v, table, 0)
                y = ops.attention_paged(dev(q), cache, table, n, causal=False).float()
                assert ((y >= low - slack) & (y <= high + slack)).all(), (big, step, at)


@pytest.mark.parametrize("batch,kv_heads,group,dim,q_rows,n", [
    (2, 3, 16, 64, 1, 300), (2, 3, 4, 128, 4, 300), (1, 2, 16, 128, 1, 4000), (1, 1, 8, 64, 2, 9000), (24, 6, 16, 64, 1, 4100),
    (140, 2, 16, 128, 1, 700), (33, 4, 2, 128, 8, 700)])
def test_few_rows_keep_the_weights_digits(ops, batch, kv_heads, group, dim, q_rows, n):
    """16 rows of a key head and fewer: what a weight's rounding leaves out is added, whatever the batch.
    Two sorts of keys, of weights 1 and e^(r / sqrt(D)) and values of -8 and 8 that nearly cancel.  Scores
    are exact; a weight is off by two roundings of an exponent of at most 14 and the hardware's 2^x (2^-20
    and 2^-22), twice rounded (2^-22), and n of them are summed up, at least 16 sums side by side in fp32
    (n / 16 roundings, of the weights and of the products); rounded once they are off by up to 2^-11."""
    say("few rows", batch, kv_heads, group, dim, q_rows, n)
    rng = np.random.default_rng(n + batch)
    cache, table, _, _ = filled(ops, rng, batch, kv_heads, dim, 64, n)
    sort = rng.random((batch, 1, n, 1)) < 0.25
    k, v = np.zeros((batch, kv_heads, n, dim), np.float16), np.where(sort, 8, -8) * rng.choice([-1, 1], dim)
    k[..., :1] = sort
    v = np.broadcast_to(v.astype(np.float16), k.shape).copy()
    ops.kv_append_paged(cache, dev(k), dev(v), dev(table), 0)
    q = rng.standard_normal((batch, kv_heads * group, q_rows, dim)).astype(np.float16)
    q[..., 0] = rng.integers(4, 21, q.shape[:3])
    y = host(ops.attention_paged(dev(q), cache, dev(table), n, causal=False))
    many = sort.sum(2, keepdims=True)[..., 0]
    w = many * np.exp(q[..., 0].astype(np.float64) / np.sqrt(dim))
    want = ((w - (n - many)) / (w + (n - many)))[..., None] * 8 * np.sign(v[:, :1, :1].astype(np.float64) * np.where(sort[:, :, :1], 1, -1))
    tol = 8 * (2.0 ** -18 + n * 2.0 ** -27) + 2.0 ** -11 * np.abs(want) + 2.0 ** -25
    assert (np.abs(y - want) <= tol).all(), (np.abs(y - want) - tol).max()
