"""GPU tests of NativeOps.sample against a plain 64-bit implementation in numpy.

Tokens have to be the reference's: the kernel's cumulative masses are right to
about 1e-12, so the two can differ only where the random number falls that near
a border; the reference checks that it does not (`far`), on inputs fixed before.
Probabilities are fp32: half a step (2^-24 relative) and the masses' 2^-44."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

NONE = 2 ** 31 - 1


def torch():
    import torch as t
    return t


def dev(a):
    return torch().from_numpy(np.ascontiguousarray(a)).cuda()


def say(*args):
    print("[case]", *args, flush=True)


def one(row, u, temperature, top_k, top_p, min_p):
    """(token, probability, distance of u from the nearest border) by the definition."""
    x = row.astype(np.float64)
    x[np.isnan(x)] = -np.inf
    if x.max() == -np.inf:
        return NONE, 0.0, 1.0
    if not temperature > 0 or x.max() == np.inf:
        return int(np.argmax(x)), 1.0, 1.0
    order = np.lexsort((np.arange(len(x)), -x))
    w = np.exp((x[order] - x.max()) / np.float64(temperature))
    n = len(x) if top_k <= 0 else min(top_k, len(x))
    far = 1.0
    if top_p < 1:
        c = np.cumsum(w[:n])
        goal = max(float(top_p), 0.0) * c[-1]
        far = min(far, float(np.abs(c - goal).min() / c[-1])) if top_p > 0 else far
        n = min(n, int(np.searchsorted(c, goal, side="left")) + 1)
    if min_p > 0:
        n = max(1, min(n, int((w >= min_p).sum())))
    c = np.cumsum(w[:n])
    u = min(max(float(u), 0.0), 1 - 2.0 ** -24) if u == u else 0.0
    at = min(int(np.searchsorted(c, u * c[-1], side="right")), n - 1)
    if u > 0:
        far = min(far, float(np.abs(c[:-1] - u * c[-1]).min() / c[-1]) if n > 1 else 1.0)
    return int(order[at]), float(w[at] / c[-1]), far


def check(ops, logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, borders=True):
    t = torch()
    batch = logits.shape[0]
    give = [dev(np.asarray(x, dt)) if np.ndim(x) else x for x, dt in
            ((temperature, np.float32), (top_k, np.int32), (top_p, np.float32), (min_p, np.float32))]
    tokens, probs = ops.sample(dev(logits), dev(np.asarray(uniforms, np.float32)), temperature=give[0], top_k=give[1],
                               top_p=give[2], min_p=give[3])
    t.cuda.synchronize()
    assert tokens.dtype == t.int32 and probs.dtype == t.float32
    tokens, probs = tokens.cpu().numpy(), probs.cpu().numpy()
    full = [np.broadcast_to(np.asarray(x, dt), batch) for x, dt in
            ((temperature, np.float32), (top_k, np.int32), (top_p, np.float32), (min_p, np.float32))]
    for b in range(batch):
        want, p, far = one(logits[b], np.float32(uniforms[b]), *(x[b] for x in full))
        assert not borders or far > 1e-11, "the input is too near a border"
        assert tokens[b] == want, f"row {b}: {tokens[b]} against {want}"
        assert abs(float(probs[b]) - p) <= (2.0 ** -24 + 1e-11) * p + 2.0 ** -140, (b, probs[b], p)
    return tokens


def rows_of(rng, batch, vocab, spread=3.0):
    return (rng.standard_normal((batch, vocab)) * spread).astype(np.float32)


@pytest.mark.parametrize("batch,vocab", [(1, 1), (3, 2), (2, 7), (5, 255), (4, 4096), (3, 4097), (2, 50257), (2, 131071),
                                         (1, 262144)])
@pytest.mark.parametrize("half", [False, True])
def test_vocabularies(ops, batch, vocab, half):
    say("vocab", batch, vocab, half)
    rng = np.random.default_rng(vocab + batch)
    x = rows_of(rng, batch, vocab)
    if half:
        x = x.astype(np.float16)
    for u in (rng.random(batch), rng.random(batch)):
        check(ops, x, u)
        check(ops, x, u, 0.7)
        check(ops, x, u, 1.0, 40)
        check(ops, x, u, 1.3, 0, 0.9)
        check(ops, x, u, 0.9, 0, 1.0, 0.05)
        check(ops, x, u, 0.8, 50, 0.95, 0.02)


def test_parameters_per_row(ops):
    say("per row")
    rng = np.random.default_rng(1)
    batch = 64
    x = rows_of(rng, batch, 5003)
    check(ops, x, rng.random(batch), rng.uniform(0.3, 2, batch), rng.integers(0, 3000, batch), rng.uniform(0.1, 1, batch),
          rng.uniform(0, 0.2, batch))


@pytest.mark.parametrize("top_k", [1, 2, 511, 512, 513, 2000, 4999, 5000, 6000, NONE])
def test_top_k(ops, top_k):
    say("top_k", top_k)
    rng = np.random.default_rng(top_k % 1000)
    x = rows_of(rng, 4, 5000)
    check(ops, x, rng.random(4), 1.0, top_k)
    check(ops, x, rng.random(4), 1.5, top_k, 0.8)


@pytest.mark.parametrize("top_p", [0.0, 1e-6, 0.5, 0.999, 0.9999999])
def test_top_p(ops, top_p):
    say("top_p", top_p)
    rng = np.random.default_rng(int(top_p * 1000))
    x = rows_of(rng, 4, 9000)
    check(ops, x, rng.random(4), 1.0, 0, top_p)
    check(ops, x, rng.random(4), 2.0, 700, top_p)


@pytest.mark.parametrize("min_p", [1e-6, 0.1, 1.0])
def test_min_p(ops, min_p):
    say("min_p", min_p)
    rng = np.random.default_rng(3)
    x = rows_of(rng, 4, 9000)
    x[1, 77] = x[1].max()          # two of the likeliest
    check(ops, x, rng.random(4), 1.0, 0, 1.0, min_p)


def test_uniforms_at_their_ends(ops):
    """0 takes the likeliest token, the largest number below 1 and what lies outside [0, 1)
    the nearest of them; kept tokens of tiny probability are at the end."""
    say("ends")
    rng = np.random.default_rng(4)
    x = rows_of(rng, 6, 3001)
    got = check(ops, x, [0.0, -1.0, np.nan, 1 - 2.0 ** -24, 1.0, 7.0], borders=False)
    assert list(got[:3]) == [int(r.argmax()) for r in x[:3]]
    check(ops, x, [0.0, 0.0, 0.0, 1 - 2.0 ** -24, 1.0, np.inf], 0.7, 20, borders=False)


@pytest.mark.parametrize("vocab", [600, 5000, 70001])
def test_equal_logits(ops, vocab):
    """Ties go to the lowest index, whole rows of them too: more equal tokens than any list holds."""
    say("ties", vocab)
    rng = np.random.default_rng(vocab)
    flat = np.zeros((4, vocab), np.float32)
    steps = np.round(rows_of(rng, 4, vocab))
    zeros = np.where(rng.random((4, vocab)) < 0.5, 0.0, -0.0).astype(np.float32)  # -0 equals 0
    for x in (flat, steps.astype(np.float32), zeros, steps.astype(np.float16)):
        check(ops, x, rng.random(4))
        check(ops, x, rng.random(4), 0.5, 300)
        check(ops, x, rng.random(4), 0.5, 577, 0.61)
        check(ops, x, rng.random(4), 1.0, 0, 0.37)


def test_near_equal_logits(ops):
    """Thousands of distinct logits within one bin, fp32 neighbours among them."""
    say("crowded bin")
    rng = np.random.default_rng(6)
    x = (1 + rng.integers(0, 4096, (3, 20000)) * 2.0 ** -23).astype(np.float32)
    x[2] = rng.uniform(0, 1e-30, 20000)
    check(ops, x, rng.random(3))
    # (Row 2's weights all round to 1 in 64 bits, so its sums are whole numbers, half of
    # 7000 of them is exactly a border, and both sides meet it exactly.)
    check(ops, x, rng.random(3), 0.9, 7000, 0.5, borders=False)


def test_masked_tokens(ops):
    """-inf and the types' lowest values are never chosen beside others; NaN never."""
    say("masks")
    rng = np.random.default_rng(7)
    for dt, low in ((np.float32, np.finfo(np.float32).min), (np.float16, np.finfo(np.float16).min)):
        x = rows_of(rng, 6, 3000).astype(dt)
        hide = rng.random((6, 3000)) < 0.9
        x[0][hide[0]] = -np.inf
        x[1][hide[1]] = low
        x[2][hide[2]] = np.nan
        x[3] = low                       # every token masked by the lowest value: all alike
        x[4], x[4, 1234] = -np.inf, -5   # one left
        x[5, 100], x[5, 200] = np.inf, np.inf
        got = check(ops, x, rng.random(6))
        assert got[4] == 1234 and got[5] == 100
        check(ops, x, rng.random(6), 0.6, 50, 0.9, 0.01)


def test_rows_without_a_token(ops):
    say("no token")
    x = np.full((4, 700), -np.inf, np.float32)
    x[1], x[2, :350] = np.nan, np.nan
    x[3, 5] = 1
    assert list(check(ops, x, [0.5] * 4)) == [NONE, NONE, NONE, 5]
    assert list(check(ops, x, [0.5] * 4, 0.0)) == [NONE, NONE, NONE, 5]


def test_temperatures(ops):
    """0 is greedy, tiny ones leave the likeliest, huge ones all alike; device values that are
    not above 0 are greedy too."""
    say("temperatures")
    rng = np.random.default_rng(8)
    x = rows_of(rng, 8, 2000)
    x[0, 30] = x[0, 20] = x[0].max()
    got = check(ops, x, rng.random(8), [0.0, 1e-6, 1e-30, -1.0, np.nan, 1e30, 0.01, 100.0])
    assert got[0] == 20 and got[3] == x[3].argmax() and got[4] == x[4].argmax()
    assert list(check(ops, x, rng.random(8), 0)) == [int(r.argmax()) for r in x]


def test_an_answer_depends_on_its_row_alone(ops):
    """The same row alone, in a batch, on another stream and captured gives the same bits."""
    say("row alone")
    t = torch()
    rng = np.random.default_rng(9)
    x, u = dev(rows_of(rng, 33, 50257)), dev(rng.random(33).astype(np.float32))
    tokens, probs = ops.sample(x, u, temperature=0.8, top_p=0.92)
    for b in (0, 7, 32):
        one_t, one_p = ops.sample(x[b:b + 1], u[b:b + 1], temperature=0.8, top_p=0.92)
        assert int(one_t) == int(tokens[b]) and float(one_p) == float(probs[b])
    side = t.cuda.Stream()
    side.wait_stream(t.cuda.current_stream())
    with t.cuda.stream(side):
        st, sp = ops.sample(x, u, temperature=0.8, top_p=0.92)
    side.synchronize()
    assert t.equal(st, tokens) and t.equal(sp, probs)
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        gt, gp = ops.sample(x, u, temperature=0.8, top_p=0.92)
    for turn in range(4):
        u.copy_(dev(rng.random(33).astype(np.float32)))
        graph.replay()
        t.cuda.synchronize()
        wt, wp = ops.sample(x, u, temperature=0.8, top_p=0.92)
        assert t.equal(gt, wt) and t.equal(gp, wp), turn


def test_frequencies(ops):
    """Over evenly spaced random numbers every token comes as often as its probability says, to one."""
    say("frequencies")
    x = np.log(np.array([0.5, 0.25, 0.125, 0.0625, 0.0625], np.float32))[None].repeat(1024, 0)
    u = (np.arange(1024) + 0.5) / 1024
    tokens, _ = ops.sample(dev(x), dev(u.astype(np.float32)))
    count = np.bincount(tokens.cpu().numpy(), minlength=5)
    assert np.abs(count - np.array([512, 256, 128, 64, 64])).max() <= 1


def test_refusals(ops):
    say("refusals")
    t = torch()
    x, u = t.zeros(2, 10, device="cuda"), t.zeros(2, device="cuda")
    bad = [
        (TypeError, lambda: ops.sample(x.double(), u)), (TypeError, lambda: ops.sample(x.t(), u)),
        (TypeError, lambda: ops.sample(x, u.double())), (ValueError, lambda: ops.sample(x, u[:1])),
        (ValueError, lambda: ops.sample(x[0], u)), (TypeError, lambda: ops.sample(x, 0.5)),
        (ValueError, lambda: ops.sample(x, u, temperature=-1.0)), (ValueError, lambda: ops.sample(x, u, temperature=float("nan"))),
        (ValueError, lambda: ops.sample(x, u, temperature=float("inf"))), (ValueError, lambda: ops.sample(x, u, temperature=None)),
        (ValueError, lambda: ops.sample(x, u, top_k=-1)), (ValueError, lambda: ops.sample(x, u, top_k=2.0)),
        (ValueError, lambda: ops.sample(x, u, top_p=1.5)), (ValueError, lambda: ops.sample(x, u, min_p=-0.1)),
        (TypeError, lambda: ops.sample(x, u, top_k=u)), (ValueError, lambda: ops.sample(x, u, top_p=u[:1])),
        (ValueError, lambda: ops.sample(x, u, min_p=True)),
        (ValueError, lambda: ops.sample(t.zeros(1, (1 << 18) + 1, device="cuda"), u[:1])),
        (ValueError, lambda: ops.sample(x.clone().requires_grad_(), u)),
    ]
    for i, (error, call) in enumerate(bad):
        with pytest.raises(error):
            call()
            pytest.fail(f"call {i} was accepted")


@pytest.mark.parametrize("vocab,top_k", [(399, 40), (400, 40), (401, 41), (16383, 256), (16384, 256), (16384, 257),
                                         (256, 256), (300, 256), (5, 3), (5, 4), (4, 4)])
def test_both_sides_of_the_one_pass_rule(ops, vocab, top_k):
    say("one pass rule", vocab, top_k)
    rng = np.random.default_rng(vocab + top_k)
    rows = rows_of(rng, 6, vocab)
    rows[4] = np.float32(0.25)                      # equal logits
    rows[5, ::2] = -np.inf                          # fewer tokens than a large top-k
    uniforms = (rng.random(6) * 0.999 + 0.0005).astype(np.float32)
    check(ops, rows, uniforms, 0.8, top_k)
    check(ops, rows, uniforms, 1.2, top_k, top_p=0.8, min_p=0.01)


@pytest.mark.parametrize("temperature", [1e-30, 1e-3, 0.7, 300.0, 1e30, float("inf")])
@pytest.mark.parametrize("shift,spread", [(0.0, 3.0), (1e5, 2.0), (-1e5, 2.0), (1e30, 1e28), (0.0, 1e-6), (-3.0, 1e-30)])
def test_scales_and_shifts(ops, temperature, shift, spread):
    """Where rounding moves logits and bins furthest against each other."""
    say("scales", temperature, shift, spread)
    rng = np.random.default_rng(int(abs(shift) % 97) + 7)
    rows = (rng.standard_normal((4, 9001)) * spread + shift).astype(np.float32)
    uniforms = (rng.random(4) * 0.999 + 0.0005).astype(np.float32)
    t = np.full(4, temperature, np.float32)
    check(ops, rows, uniforms, t, top_p=0.9, borders=False)
    check(ops, rows, uniforms, t, 2000, top_p=0.95, min_p=0.001, borders=False)
