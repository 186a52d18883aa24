"""GPU tests of rotary positions (NativeOps.rotary, rotate) against a plain implementation
with angles in 80-bit arithmetic.

Tolerance, from the operator's roundings.  An angle is t f / 2 pi turns with f / 2 pi held
to 2^-53 of itself (t f 2^-52 radians at most, both halves counted) and to 2^-65 turns; its
rest within a quarter turn is rounded to fp32 three times (3 * 2^-24 of at most pi / 4); the
polynomials are off by 2.5e-8 and round five times next to 1 (5 * 2^-24): a cosine or sine is
off by less than 2^-21 + t f 2^-52.  A turned value is the fp32 sum of two products (three
roundings of 2^-24 of their absolute values, one more for the amplitude), rounded to fp16
once (2^-11, or 2^-25 below fp16's normal range):
  |got - want| <= e + 2^-11 (|want| + e) + 2^-25,  e = amplitude (|a| + |b|) (2^-20 + t f 2^-52)"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


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


def frequencies(rotated, base=10000.0, how=None, factor=1.0, length=None, fast=32.0, slow=1.0):
    i = np.arange(rotated // 2, dtype=np.longdouble)
    base = np.longdouble(base)
    if how == "base" and rotated > 2:
        base = base * np.longdouble(factor) ** (np.longdouble(rotated) / (rotated - 2))
    f = base ** (-2 * i / rotated)
    if how == "linear":
        f = f / factor
    if how == "parts":
        turns = length * f / (2 * np.longdouble(math.pi))
        ramp = np.clip((turns - slow) / (fast - slow), 0, 1)
        f = ramp * f + (1 - ramp) * f / factor
    return f


TWO_PI = 8 * np.arctan(np.longdouble(1))


def turned(x, positions, f, interleaved, amplitude=1.0):
    """(values, their tolerance): x [B, H, Q, D] fp16, positions [B, Q]."""
    half = len(f)
    a = np.arange(half) * 2 if interleaved else np.arange(half)
    b = a + 1 if interleaved else a + half
    angle = np.mod(positions.astype(np.longdouble)[..., None] * f, TWO_PI)[:, None]
    c, s = np.cos(angle), np.sin(angle)
    y = x.astype(np.longdouble)
    want, tol = y.copy(), np.zeros(x.shape)
    u, v = y[..., a], y[..., b]
    want[..., a], want[..., b] = amplitude * (u * c - v * s), amplitude * (u * s + v * c)
    e = abs(amplitude) * (np.abs(u) + np.abs(v)) * (2.0 ** -20 + np.abs(positions[..., None] * f)[:, None] * 2.0 ** -52)
    for at in (a, b):
        tol[..., at] = e + 2.0 ** -11 * (np.abs(want[..., at]) + e) + 2.0 ** -25
    return want, tol


def check(got, want, tol, dims):
    bad = np.abs(got.astype(np.longdouble) - want) > tol
    assert not bad.any(), f"{bad.sum()} off, first at {np.argwhere(bad)[0]}: {got[bad][0]} against {want[bad][0]}"
    assert np.array_equal(got[..., dims:], want[..., dims:].astype(np.float16))


@pytest.mark.parametrize("batch,heads,rows,dim,rotated,interleaved", [
    (1, 1, 1, 64, 64, False), (3, 12, 1, 64, 64, True), (2, 5, 7, 128, 128, False), (2, 25, 33, 64, 32, False),
    (2, 3, 65, 128, 32, True), (1, 2, 300, 256, 64, False), (2, 4, 9, 80, 20, False), (2, 4, 9, 80, 40, True),
    (1, 3, 5, 96, 2, False), (2, 1, 3, 2, 2, True), (1, 2, 4, 7, 6, False), (2, 40, 17, 112, 112, True),
    (1, 2, 3, 16, 16, False), (33, 2, 2, 48, 16, True), (1, 8, 4100, 64, 64, False)])
def test_against_the_formula(ops, batch, heads, rows, dim, rotated, interleaved):
    say("rotate", batch, heads, rows, dim, rotated, interleaved)
    rng = np.random.default_rng(rows * dim + rotated)
    x = rng.standard_normal((batch, heads, rows, dim)).astype(np.float16)
    x[0, 0, 0, 0] = 65504
    x[-1, -1, -1, -1] = 2.0 ** -24
    first = rng.integers(0, 5000, batch).astype(np.int32)
    first[0] = 0
    rotary = ops.rotary(rotated, interleaved=interleaved)
    f, at = frequencies(rotated), first[:, None] + np.arange(rows)
    x[0, 0, 0, :rotated] = np.minimum(x[0, 0, 0, :rotated], 40000)  # (position 0 turns by nothing)
    want, tol = turned(x, at, f, interleaved)
    check(host(ops.rotate(dev(x), rotary, dev(first))), want, tol, rotated)
    check(host(ops.rotate(dev(x), rotary, first.tolist())), want, tol, rotated)
    each = rng.permutation(at.reshape(-1)).reshape(at.shape).astype(np.int32)
    want, tol = turned(x, each, f, interleaved)
    check(host(ops.rotate(dev(x), rotary, dev(each))), want, tol, rotated)


@pytest.mark.parametrize("far", [0, 1000, 131072, 2 ** 24 + 1, 2 ** 31 - 100])
@pytest.mark.parametrize("how", [dict(), dict(how="linear", factor=8.0), dict(how="base", factor=4.0),
                                 dict(how="parts", factor=4.0, length=8192)])
def test_far_positions_and_stretched_frequencies(ops, far, how):
    say("far", far, how)
    rng = np.random.default_rng(far % 1000)
    x = rng.standard_normal((1, 3, 50, 128)).astype(np.float16)
    args = {"scaling": how.get("how"), **({"factor": how["factor"]} if how else {}),
            **({"original_length": how["length"]} if "length" in how else {})}
    rotary = ops.rotary(128, base=500000.0, amplitude=1.25, **args)
    f = frequencies(128, base=500000.0, **how)
    assert np.allclose(np.array(rotary.frequencies), f.astype(float), rtol=1e-14)
    want, tol = turned(x, np.int64(far) + np.arange(50)[None], f, False, 1.25)
    check(host(ops.rotate(dev(x), rotary, far)), want, tol, 128)


def test_given_frequencies_and_negative_positions(ops):
    say("given frequencies")
    rng = np.random.default_rng(5)
    f = [0.0, 1.0, 2 * math.pi, -0.3, 7.5, 1e-9, 1e3, 0.25]
    rotary = ops.rotary(16, frequencies=f, amplitude=-0.5)
    x = rng.standard_normal((2, 2, 40, 64)).astype(np.float16)
    at = np.array([[-20], [1000]]) + np.arange(40)
    want, tol = turned(x, at, np.array(f, np.longdouble), False, -0.5)
    check(host(ops.rotate(dev(x), rotary, dev(at[:, 0].astype(np.int32)))), want, tol, 16)


@pytest.mark.parametrize("dim,rotated", [(64, 64), (80, 20)])
def test_any_strides(ops, dim, rotated):
    """Slices of a projection, expanded heads and odd offsets; a single row of odd strides."""
    say("strides", dim, rotated)
    t = torch()
    rng = np.random.default_rng(9)
    rotary = ops.rotary(rotated)
    whole = dev(rng.standard_normal(3 * 11 * 7 * dim + 3).astype(np.float16))
    view = whole[1:-2].view(3, 11, 7, dim).transpose(1, 2)[:, 2:5, ::2]
    flat = view.contiguous()
    for pos in (17, dev(np.arange(18, dtype=np.int32).reshape(3, 6) * 5)):
        assert t.equal(ops.rotate(view, rotary, pos), ops.rotate(flat, rotary, pos))
    spread = flat[:, :1].expand(3, 4, 6, dim)
    assert t.equal(ops.rotate(spread, rotary, 3), ops.rotate(spread.contiguous(), rotary, 3))
    assert ops.rotate(view, rotary, 17).is_contiguous()


def test_not_finite_values_stay_in_their_pair(ops):
    say("not finite")
    x = np.zeros((1, 1, 2, 64), np.float16)
    x[0, 0, 0, 5], x[0, 0, 1, 40] = np.nan, np.inf
    y = host(ops.rotate(dev(x), ops.rotary(64), 3))
    bad = ~np.isfinite(y)
    assert bad[0, 0, 0, [5, 37]].all() and bad[0, 0, 1, [8, 40]].all() and bad.sum() == 4


def test_captured_and_on_two_streams(ops):
    say("graph and streams")
    t = torch()
    rng = np.random.default_rng(2)
    rotary = ops.rotary(64)
    x = dev(rng.standard_normal((4, 12, 1, 64)).astype(np.float16))
    pos = dev(np.array([0, 7, 900, 5], np.int32))
    want = ops.rotate(x, rotary, pos)
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        y = ops.rotate(x, rotary, pos)
    for turn in range(3):
        pos += 1
        x.mul_(0.5)
        want = ops.rotate(x, rotary, pos)
        y.zero_()
        graph.replay()
        t.cuda.synchronize()
        assert t.equal(y, want), turn
    side = t.cuda.Stream()
    side.wait_stream(t.cuda.current_stream())
    with t.cuda.stream(side):
        other = ops.rotate(x, rotary, pos)
    side.synchronize()
    assert t.equal(other, want)
