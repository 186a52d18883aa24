"""GPU tests of NativeOps.sample on rows whose tokens crowd into few bins of the kernel's
histogram, up to the largest vocabulary, against the 64-bit implementation of
test_sample_gpu.

A token's weight is right to 1.4 * 2^-30 of itself: its fraction to 2^-23 of a bin, which
is 2^-31 of the weight; its loss of at most 1.02 * 2^-8 to three fp32 roundings (of the
fraction and the slack, and the last two steps), 3.1 * 2^-32, and a cut to 2^-34.  A bin's
mass is rounded to 2^-45 of the likeliest token's once, 8192 of them to 2^-32.  So a
cumulative mass and a total are right to r = 2^-29, a border to 2 r of the total for a
filter's goal and for the random number's, and a probability to 2^-24 (its fp32 rounding)
and 2 r of itself."""
import numpy as np
import pytest

from test_sample_gpu import dev, one, say, torch

pytestmark = pytest.mark.gpu

OFF = 2.0 ** -29
VOCAB = 1 << 18


def check(ops, logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    t = torch()
    tokens, probs = ops.sample(dev(logits), dev(np.asarray(uniforms, np.float32)), temperature=temperature, top_k=top_k,
                               top_p=top_p, min_p=min_p)
    t.cuda.synchronize()
    tokens, probs = tokens.cpu().numpy(), probs.cpu().numpy()
    for b, row in enumerate(logits):
        want, p, far = one(row, np.float32(uniforms[b]), np.float32(temperature), top_k, np.float32(top_p), np.float32(min_p))
        assert far > 4 * OFF, "the input is too near a border"
        assert tokens[b] == want, f"row {b}: {tokens[b]} against {want}"
        assert abs(float(probs[b]) - p) <= (2.0 ** -24 + 2 * OFF) * p, (b, probs[b], p)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("fraction", [0.0, 0.02, 0.5, 0.98, 0.999])
@pytest.mark.parametrize("bin_", [0, 1, 1280])
def test_a_whole_vocabulary_in_one_bin(ops, bin_, fraction, half):
    """One likeliest token, all others equal behind it at a bin's near edge, middle and far edge."""
    say("one bin", bin_, fraction, half)
    rng = np.random.default_rng(bin_ + int(1000 * fraction))
    x = np.full((4, VOCAB), -(bin_ + fraction) / 256, np.float32)
    x[np.arange(4), rng.integers(0, VOCAB, 4)] = 0
    if half:  # (a bin of 1280 is wider than an fp16 step there, so the fraction is another one)
        x = x.astype(np.float16)
    uniforms = np.array([0.0031, 0.4987, 0.9971, 1 - 2.0 ** -24], np.float32)
    check(ops, x, uniforms)
    check(ops, x, uniforms, top_p=0.97)
    check(ops, x, uniforms, min_p=0.001)
    check(ops, x, uniforms, top_k=VOCAB - 3)
    check(ops, x, uniforms, top_k=VOCAB - 3, top_p=0.6, min_p=0.0005)


@pytest.mark.parametrize("temperature", [0.5, 1.0])
def test_the_largest_vocabulary_of_few_distinct_logits(ops, temperature):
    """Equal ones, fp32 neighbours, and a few steps of one bin."""
    say("few distinct", temperature)
    rng = np.random.default_rng(3)
    x = np.zeros((4, VOCAB), np.float32)
    x[1] = 1 + rng.integers(0, 4096, VOCAB) * np.float32(2.0 ** -23)
    x[2] = rng.integers(0, 8, VOCAB) / np.float32(2048)
    x[3, 1:] = -rng.integers(250, 256, VOCAB - 1) / np.float32(65536)
    uniforms = np.array([0.99993, 0.2501, 0.7503, 0.99997], np.float32)
    check(ops, x, uniforms, temperature)
    check(ops, x, uniforms, temperature, top_k=200003)
    check(ops, x, uniforms, temperature, top_p=0.9137)
    check(ops, x, uniforms, temperature, top_k=250001, top_p=0.31, min_p=0.9)


@pytest.mark.parametrize("distance", [31.9, 32.5, 33.0])
def test_a_vocabulary_far_behind_the_likeliest(ops, distance):
    """Nearly all of the largest vocabulary about 32 temperatures behind the likeliest token:
    from 32 on they count as without weight, at most V e^-32 of the likeliest one's, which
    moves a border and a probability by as much (again for each goal)."""
    say("far behind", distance)
    rng = np.random.default_rng(int(10 * distance))
    x = (-distance - rng.random((4, VOCAB)) * 0.05).astype(np.float32)
    for row in x:
        row[rng.permutation(VOCAB)[:5]] = [0, -1.5, -4, -9, -11.5]
    uniforms = np.array([0.11, 0.79, 0.999, 1 - 2.0 ** -24], np.float32)
    off = OFF + 1.001 * VOCAB * np.exp(-32.0)
    for more in ({}, {"top_k": VOCAB - 100}, {"top_k": 3000}, {"min_p": 1e-14}, {"top_p": 0.9999}, {"top_k": 70000, "top_p": 0.87}):
        tokens, probs = ops.sample(dev(x), dev(uniforms), **more)
        torch().cuda.synchronize()
        for b in range(4):
            want, p, far = one(x[b], uniforms[b], np.float32(1), more.get("top_k", 0), np.float32(more.get("top_p", 1)),
                               np.float32(more.get("min_p", 0)))
            assert far > 4 * off, "the input is too near a border"
            assert int(tokens[b]) == want, (more, b)
            assert abs(float(probs[b]) - p) <= (2.0 ** -24 + 2 * off) * p, (more, b, float(probs[b]), p)
