"""GPU test of decoding with the int8 KV cache and the sampler together: prompts are appended,
then every step appends a token's rows, attends (to a shared prefix too), multiplies the output
by a vocabulary matrix and samples the next token, whose rows the step after it appends.

Attention is held against the 64-bit result over the tokens that were in fact sampled, tokens
against the 64-bit sampler of the logits that were in fact computed, so no error carries over."""
import numpy as np
import pytest

from test_int8_cache_gpu import check, dev, ends_of, held, host, i32, random_rows, say, torch
from test_sample_gpu import one

pytestmark = pytest.mark.gpu

VOCAB, STEPS = 1003, 6
TEMPERATURE, TOP_K, TOP_P, MIN_P = [0.7, 1.0, 1.3, 0.0], [0, 40, 300, 0], [0.95, 1.0, 0.9, 1.0], [0.0, 0.01, 0.0, 0.0]


@pytest.fixture(scope="module")
def ops():
    from tinyinfer_amd.native_ops import NativeOps
    return NativeOps()


class Held:
    """What the cache holds, in 64 bits."""

    def __init__(self, slots, kv_heads, capacity, dim):
        self.kv_heads, self.dim = kv_heads, dim
        self.hk, self.hv = (np.zeros((slots, kv_heads, capacity, dim)) for _ in range(2))

    def write(self, slots, positions, k, v, lengths):
        for b, (slot, at, n) in enumerate(zip(slots, positions, lengths)):
            self.hk[slot, :, at:at + n], self.hv[slot, :, at:at + n] = held(k)[0][b, :, :n], held(v)[0][b, :, :n]


@pytest.mark.parametrize("prefix", [0, 90])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 64), (6, 2, 128)])
def test_decode_loop(ops, heads, kv_heads, dim, prefix):
    say("decode loop", heads, kv_heads, dim, prefix)
    t = torch()
    rng = np.random.default_rng(heads + prefix)
    batch, capacity = 4, 128
    slots, prefix_slot = [3, 0, 4, 1], 2
    prompt = np.array([37, 1, 64, 9])
    # a token's q, k and v, and the vocabulary matrix
    table = rng.standard_normal((VOCAB, heads + 2 * kv_heads, dim)).astype(np.float16)
    weight = dev((rng.standard_normal((heads * dim, VOCAB)) * 4 / np.sqrt(heads * dim)).astype(np.float16))
    k, v = random_rows(rng, batch, kv_heads, 64, dim), random_rows(rng, batch, kv_heads, 64, dim)
    pk, pv = random_rows(rng, 1, kv_heads, capacity, dim), random_rows(rng, 1, kv_heads, capacity, dim)
    uniforms = rng.random((STEPS, batch)).astype(np.float32)
    first = rng.integers(0, VOCAB, batch).astype(np.int32)
    dtable, du = dev(table), dev(uniforms)
    dslots, lanes = i32(slots), [dev(np.asarray(x, d)) for x, d in
                                 ((TEMPERATURE, np.float32), (TOP_K, np.int32), (TOP_P, np.float32), (MIN_P, np.float32))]

    def filled():
        cache = ops.kv_cache_int8(5, kv_heads, capacity, dim)
        ops.kv_append_int8(cache, dev(k), dev(v), slots, 0, lengths=[int(n) for n in prompt])
        ops.kv_append_int8(cache, dev(pk), dev(pv), prefix_slot, 0)
        return cache

    def step(cache, tokens, lengths, u):
        """One step; the tokens and lengths that the next one takes, and what is checked."""
        rows = dtable[tokens.long()].view(batch, heads + 2 * kv_heads, 1, dim)
        q, nk, nv = (x.contiguous() for x in rows.split([heads, kv_heads, kv_heads], 1))
        ops.kv_append_int8(cache, nk, nv, dslots, lengths)
        after = lengths + 1
        if prefix:
            o = ops.attention_shared_prefix(q, cache, prefix_slot, prefix, dslots, after)
        else:
            o = ops.attention_int8kv(q, cache, dslots, after)
        logits = ops.gemm(o.view(batch, heads * dim), weight, output_dtype=t.float32)
        chosen, probs = ops.sample(logits, u, temperature=lanes[0], top_k=lanes[1], top_p=lanes[2], min_p=lanes[3])
        return chosen, after, o, logits, probs

    cache, want = filled(), Held(5, kv_heads, capacity, dim)
    want.write(slots, [0] * batch, k, v, prompt)
    want.write([prefix_slot], [0], pk, pv, [capacity])
    tokens, lengths, eager = dev(first), i32(prompt), []
    for n in range(STEPS):
        fed, at = host(tokens), host(lengths)
        tokens, lengths, o, logits, probs = step(cache, tokens, lengths, du[n])
        rows = table[fed][:, :, None]
        want.write(slots, at, rows[:, heads:heads + kv_heads], rows[:, heads + kv_heads:], [1] * batch)
        check(o, np.ascontiguousarray(rows[:, :heads]), want, slots, ends_of(at + 1, 1),
              prefix=(prefix_slot, prefix) if prefix else None)
        for b, (token, p) in enumerate(zip(host(tokens), host(probs))):
            expect, chance, far = one(host(logits)[b], uniforms[n, b], np.float32(TEMPERATURE[b]), TOP_K[b],
                                      np.float32(TOP_P[b]), np.float32(MIN_P[b]))
            assert far > 1e-11, "the input is too near a border"
            assert token == expect and abs(float(p) - chance) <= (2.0 ** -24 + 1e-11) * chance
        eager.append((host(tokens), host(o)))
    assert len({x[0].tobytes() for x in eager}) > 1

    # the step as a graph, replayed in place
    cache = filled()
    tokens, lengths, u = dev(first), i32(prompt), du[0].clone()
    side = t.cuda.Stream()
    side.wait_stream(t.cuda.current_stream())
    with t.cuda.stream(side):
        graph = t.cuda.CUDAGraph()
        with t.cuda.graph(graph, stream=side):
            chosen, after, o, _, _ = step(cache, tokens, lengths, u)
            tokens.copy_(chosen)
            lengths.copy_(after)
        for n in range(STEPS):
            u.copy_(du[n])
            graph.replay()
            side.synchronize()
            assert np.array_equal(tokens.cpu().numpy(), eager[n][0])
            assert np.array_equal(o.cpu().numpy(), eager[n][1])
