"""GPU tests of log probabilities (NativeOps.logprobs) against a plain implementation in
64 bits.

Tolerance, with u = 2^-24, m the row's largest logit, d = x - m, Z = sum e^d, c the number of
logits equal to m and R = Z - c.  d is rounded once (u |d|), its exponential to 2 u |d| + 4 u
of itself (a product with log2 e and the hardware's 2^x); a thread adds up at most V / 1024 +
40 of them after another, and 10 + 16 joins follow, each with a rescaling (4 u).  With
n = V / 1024 + 200 for all of these roundings together
  R is off by  u sum over x < m of e^d (2 |d| + n),
  S = sum e^d d by  u sum e^d |d| (2 |d| + n),
log Z = log c + log1p(R / c) by R's error over Z and 4 u of itself, a log probability by that
and 2 u (|d| + log Z), the entropy log Z - S / Z by that, S's error over Z, R's error times
|S| / Z^2 and 4 u of its terms.  Exponentials below fp32's normal range, 2^-126, count as 0:
at most V 2^-126 of R and, as |d| e^d falls from d = -87.4 on, V 2^-119 of S."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
NONE = 2 ** 31 - 1


def torch():
    import torch as t
    return t


def dev(a):
    return torch().from_numpy(np.ascontiguousarray(a)).cuda()


def host(x):
    torch().cuda.synchronize()
    return x.cpu().numpy()


def say(*args):
    print("[case]", *args, flush=True)


def row_of(x):
    """Order, log probabilities, entropy and their tolerances of one finite-maximum row."""
    x = np.where(np.isnan(x.astype(np.float64)), -np.inf, x.astype(np.float64))
    m = x.max()
    d = x - m
    e = np.exp(d)
    live = e > 0
    dl, el = d[live], e[live]
    below = dl < 0
    c, r = (~below).sum(), el[below].sum()
    z, s = c + r, (el * dl).sum()
    n = len(x) / 1024 + 200
    r_err = U * (el[below] * (2 * -dl[below] + n)).sum() + len(x) * 2.0 ** -126
    s_err = U * (el * -dl * (2 * -dl + n)).sum() + len(x) * 2.0 ** -119
    log_z = math.log(c) + math.log1p(r / c)
    z_err = r_err / z + 4 * U * abs(log_z)
    lp = d - log_z
    with np.errstate(invalid="ignore"):
        lp_tol = z_err + 2 * U * (np.abs(d) + log_z)
    entropy = log_z - s / z
    h_tol = z_err + s_err / z + r_err * -s / z ** 2 + 4 * U * (log_z - s / z)
    order = np.lexsort((np.arange(len(x)), -x))
    return order[:np.isfinite(x).sum()], lp, lp_tol, entropy, h_tol


def close(got, want, tol, what):
    both = np.isneginf(got) & np.isneginf(want)
    with np.errstate(invalid="ignore"):
        bad = ~both & ~(np.abs(got.astype(np.float64) - want) <= tol)
    assert not bad.any(), f"{what}: {got[bad][0]} against {want[bad][0]}, {np.broadcast_to(tol, got.shape)[bad][0]} allowed"


def check(ops, logits, tokens, top):
    lp, entropy, top_lp, top_tokens = (host(y) for y in ops.logprobs(dev(logits), dev(tokens), top=top))
    assert lp.shape == tokens.shape and entropy.shape == (len(logits),) and top_lp.shape == top_tokens.shape == (len(logits), top)
    many = tokens.reshape(len(logits), -1)
    for b, x in enumerate(logits):
        order, want, tol, h, h_tol = row_of(x)
        inside = (many[b] >= 0) & (many[b] < len(x))
        at = np.where(inside, many[b], 0)
        close(lp.reshape(many.shape)[b], np.where(inside, want[at], -np.inf), tol[at], f"row {b}")
        close(entropy[b:b + 1], np.array([h]), h_tol, f"entropy {b}")
        k = min(top, len(order))
        assert np.array_equal(top_tokens[b, :k], order[:k]), f"row {b}: {top_tokens[b, :k]} against {order[:k]}"
        close(top_lp[b, :k], want[order[:k]], tol[order[:k]], f"top {b}")
        assert (top_tokens[b, k:] == NONE).all() and np.isneginf(top_lp[b, k:]).all()


@pytest.mark.parametrize("batch,vocab,top", [
    (1, 1, 1), (2, 1, 0), (3, 2, 5), (2, 3, 64), (4, 7, 3), (3, 17, 20), (2, 64, 64), (5, 65, 64), (2, 1000, 1), (3, 1023, 5),
    (2, 4097, 33), (3, 16385, 20), (2, 50257, 0), (3, 50257, 5), (1, 50257, 64), (2, 65536, 17), (2, 128257, 20), (1, 2 ** 18, 64),
    (130, 50257, 5), (60, 50257, 20), (20, 131003, 64), (2, 32768, 33)])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_against_the_formula(ops, batch, vocab, top, dtype):
    say("logprobs", batch, vocab, top, dtype.__name__)
    rng = np.random.default_rng(vocab + top)
    logits = (rng.standard_normal((batch, vocab)) * 3).astype(dtype)
    check(ops, logits, rng.integers(0, vocab, batch).astype(np.int32), top)
    tokens = rng.integers(0, vocab, (batch, 5)).astype(np.int32)
    tokens[0, :4] = [0, vocab - 1, vocab, -1]
    check(ops, logits, tokens, top)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_rows_of_every_kind(ops, dtype):
    """Equal logits, rising and falling ones, few tokens left, sure rows, large values, ties of zeros."""
    say("kinds", dtype.__name__)
    vocab = 50257
    rng = np.random.default_rng(1)
    rows = [np.zeros(vocab), np.linspace(-20, 20, vocab), np.linspace(20, -20, vocab), np.full(vocab, -np.inf),
            np.full(vocab, -np.inf), rng.standard_normal(vocab), rng.standard_normal(vocab), rng.standard_normal(vocab) * 1000,
            np.where(rng.random(vocab) < 0.5, 0.0, -0.0), rng.integers(-3, 3, vocab).astype(float), np.full(vocab, 65504.0),
            rng.standard_normal(vocab)]
    rows[3][[7, 50000, 123]] = [1.0, 1.0, -60000.0]
    rows[4][50256] = -5.0
    rows[5][777] = 18.0
    rows[6][31] = 60.0
    rows[11][4096:] = np.linspace(5, 6, vocab - 4096)   # many above the first tokens' bar
    logits = np.stack(rows).astype(dtype)
    tokens = np.tile(np.array([[7, 50000, 0, 777, 31, 50256]], np.int32), (len(rows), 1))
    for top in (0, 1, 5, 64):
        check(ops, logits, tokens, top)


def test_sure_rows_keep_their_digits(ops):
    """log p of a token that is nearly certain, and the row's entropy, to relative accuracy."""
    say("sure")
    logits = np.full((3, 4000), -50.0, np.float32)
    logits[:, 1234] = 0.0
    logits[0, 5] = -16.0
    logits[1, 5] = -30.0
    lp, entropy, _, _ = (host(y) for y in ops.logprobs(dev(logits), dev(np.full(3, 1234, np.int32))))
    for b in range(3):
        x = logits[b].astype(np.longdouble)
        rest = np.exp(x[x < 0]).sum()
        assert abs(lp[b] / -np.log1p(rest) - 1) < 1e-4
        assert abs(entropy[b] / (np.log1p(rest) - (np.exp(x) * x).sum() / (1 + rest)) - 1) < 1e-4


def test_infinities_and_nan(ops):
    say("infinities")
    inf, nan = math.inf, math.nan
    for dtype in (np.float16, np.float32):
        logits = np.zeros((5, 300), dtype)
        logits[0] = -inf
        logits[1] = nan
        logits[2, [40, 9, 200]] = inf
        logits[2, 3] = nan
        logits[3, ::3] = nan
        logits[3, 1::3] = -inf
        logits[4, 17] = nan
        tokens = np.tile(np.array([[3, 9, 40, 5, 17]], np.int32), (5, 1))
        lp, h, top_lp, top = (host(y) for y in ops.logprobs(dev(logits), dev(tokens), top=4))
        assert np.isneginf(lp[:2]).all() and (h[:3] == 0).all() and (top[:2] == NONE).all() and np.isneginf(top_lp[:2]).all()
        assert lp[2].tolist() == [-inf, 0.0, -inf, -inf, -inf]
        assert top[2].tolist() == [9, 40, 200, 0] and top_lp[2].tolist() == [0.0, -inf, -inf, -inf]
        check(ops, logits[3:], tokens[3:], 4)


def test_unaligned_rows(ops):
    """Logits that start anywhere in memory, of odd lengths."""
    say("unaligned")
    rng = np.random.default_rng(8)
    for dtype in (np.float16, np.float32):
        for shift in (1, 3, 5, 7):
            flat = dev((rng.standard_normal(shift + 3 * 1537) * 2).astype(dtype))[shift:]
            x = flat.view(3, 1537)
            tokens = dev(np.array([0, 1536, 700], np.int32))
            for got, want in zip(ops.logprobs(x, tokens, top=20), ops.logprobs(x.clone(), tokens, top=20)):
                assert torch().allclose(got.double(), want.double(), rtol=1e-5, atol=1e-6)
            check(ops, host(x), host(tokens), 20)


def test_calls_on_streams_at_once(ops):
    """Rows split over workgroups, several calls in flight: each as on its own."""
    say("streams")
    t = torch()
    rng = np.random.default_rng(9)
    work = []
    for i, (batch, vocab, top) in enumerate([(1, 50257, 5), (32, 50257, 20), (9, 128257, 64), (40, 70001, 0)]):
        logits = dev((rng.standard_normal((batch, vocab)) * 3).astype(np.float16 if i % 2 else np.float32))
        tokens = dev(rng.integers(0, vocab, batch).astype(np.int32))
        work.append((logits, tokens, top, ops.logprobs(logits, tokens, top=top)))
    t.cuda.synchronize()
    streams = [t.cuda.Stream() for _ in range(4)]
    got = []
    for turn in range(6):
        for i, stream in enumerate(streams):
            logits, tokens, top, _ = work[(i + turn) % 4]
            with t.cuda.stream(stream):
                got.append(((i + turn) % 4, ops.logprobs(logits, tokens, top=top)))
    t.cuda.synchronize()
    for i, y in got:
        for a, b in zip(y, work[i][3]):
            assert t.equal(a, b), i


def test_an_answer_depends_on_its_row_alone(ops):
    """Rows that one workgroup reads whatever their number."""
    say("rows alone")
    t = torch()
    rng = np.random.default_rng(4)
    logits = dev(rng.standard_normal((300, 2000)).astype(np.float32))
    tokens = dev(rng.integers(0, 2000, 300).astype(np.int32))
    whole = ops.logprobs(logits, tokens, top=7)
    for b in (0, 150, 299):
        for got, want in zip(ops.logprobs(logits[b:b + 1].clone(), tokens[b:b + 1].clone(), top=7), whole):
            assert t.equal(got[0], want[b])
    for got, want in zip(ops.logprobs(logits, tokens, top=7), whole):
        assert t.equal(got, want)


def test_captured(ops):
    say("graph")
    t = torch()
    rng = np.random.default_rng(6)
    logits = dev(rng.standard_normal((8, 50257)).astype(np.float32))
    tokens = dev(rng.integers(0, 50257, 8).astype(np.int32))
    ops.logprobs(logits, tokens, top=5)
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        out = ops.logprobs(logits, tokens, top=5)
    for turn in range(3):
        logits.mul_(1.5)
        tokens.add_(1).remainder_(50257)
        want = ops.logprobs(logits, tokens, top=5)
        for y in out:
            y.zero_()
        graph.replay()
        t.cuda.synchronize()
        for got, w in zip(out, want):
            assert t.equal(got, w), turn
