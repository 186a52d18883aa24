"""GPU tests of the paged cache's operators together, as a serving loop uses them, and of what
they refuse.

Every stage of a step is compared with its formula on that stage's own inputs: keys and
queries with ``rotate`` (bit for bit), the attention in 64 bits, a sampled token's
probability with its log probability."""
import ctypes
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def torch():
    import torch as t
    return t


def i32(values):
    return torch().tensor(values, dtype=torch().int32, device="cuda")


def say(*args):
    print("[case]", *args, flush=True)


class Model:
    """One layer of random weights: projection, attention, output, head; 4 query heads over 2."""

    def __init__(self, ops, dim, vocab, seed):
        t = torch()
        gen = t.Generator("cuda").manual_seed(seed)
        rand = lambda *s: t.randn(s, generator=gen, device="cuda", dtype=t.float16)  # noqa: E731
        self.ops, self.dim, self.hidden, self.vocab = ops, dim, 4 * dim, vocab
        self.embed = rand(vocab, self.hidden)
        self.qkv = rand(self.hidden, 8 * dim) * self.hidden ** -0.5
        self.out = t.randint(-127, 128, (self.hidden, self.hidden), generator=gen, device="cuda", dtype=t.int8)
        self.out_scale = t.full((self.hidden,), 0.01 * self.hidden ** -0.5, device="cuda")
        self.head = rand(self.hidden, vocab) * self.hidden ** -0.5
        self.rotary = ops.rotary(dim, base=500000.0, scaling="parts", factor=4.0, original_length=64)

    def step(self, tokens, cache, table, positions, lengths, uniforms):
        """tokens [B, Q]: rows i < lengths[b] are the request's tokens positions[b] + i."""
        t, ops = torch(), self.ops
        batch, rows = tokens.shape
        x = self.embed[tokens.long()].view(batch * rows, self.hidden)
        qkv = ops.gemm(x, self.qkv).view(batch, rows, 8, self.dim).transpose(1, 2)
        q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
        turned = ops.kv_append_paged(cache, k, v, table, positions, lengths=lengths, rotary=self.rotary, q=q)
        held = positions + lengths
        y = ops.attention_paged(turned, cache, table, held, q_lengths=lengths)
        last = y.transpose(1, 2).reshape(batch, rows, self.hidden)[t.arange(batch, device="cuda"), (lengths - 1).clamp(min=0).long()]
        x = ops.gemm_int8(last, self.out, self.out_scale)
        logits = ops.gemm(x, self.head, output_dtype=t.float32)
        tokens, probs = ops.sample(logits, uniforms)
        return {"q": q, "k": k, "turned": turned, "y": y, "logits": logits, "tokens": tokens, "probs": probs,
                "held": held, "scores": ops.logprobs(logits, tokens, top=3)}


def check_step(model, out, cache, table, positions, lengths):
    t, ops = torch(), model.ops
    batch, _, rows, dim = out["turned"].shape
    live = (t.arange(rows, device="cuda") < lengths[:, None])[:, None, :, None]
    zero = t.zeros((), dtype=t.float16, device="cuda")
    assert t.equal(out["turned"], t.where(live, ops.rotate(out["q"], model.rotary, positions), zero))
    k, _ = ops.kv_read_paged(cache, table, positions, lengths, rows)
    assert t.equal(k, t.where(live, ops.rotate(out["k"], model.rotary, positions), zero))
    held = out["held"]
    n = int(held.max())
    ck, cv = (x.double() for x in ops.kv_read_paged(cache, table, t.zeros_like(positions), held, n))
    for b in range(batch):
        for h in range(4):
            s = out["turned"][b, h].double() @ ck[b, h // 2].t() / math.sqrt(dim)
            end = positions[b] + t.arange(rows, device="cuda") + 1
            sees = (t.arange(n, device="cuda")[None] < end[:, None]) & (t.arange(rows, device="cuda") < lengths[b])[:, None]
            s = s.masked_fill(~sees, -math.inf)
            p = t.softmax(s, -1).nan_to_num(0.0)
            want, size = p @ cv[b, h // 2], p @ cv[b, h // 2].abs()
            # Weights and result are rounded to fp16 (2^-11 each, or absolutely by 2^-31 of the largest
            # value for a weight and 2^-25), scores are fp32 sums of D products (D + 8 roundings of their
            # absolute terms, in a power of e, above and below the line).
            terms = (out["turned"][b, h].double().abs() @ ck[b, h // 2].abs().t()).max() / math.sqrt(dim)
            d = 2 * (dim + 8) * 2.0 ** -24 * (terms + 32)
            tol = 1.02 * ((2.0 ** -11 + d) * size + n * 2.0 ** -31 * cv[b, h // 2].abs().max() + 2.0 ** -11 * want.abs() + 2.0 ** -25)
            assert ((out["y"][b, h].double() - want).abs() <= tol).all(), (b, h)
    lp, entropy, top_lp, top = out["scores"]
    exact = t.log_softmax(out["logits"].double(), -1)
    given = exact.gather(1, out["tokens"].long()[:, None])[:, 0]
    assert t.allclose(lp.double(), given, rtol=1e-5, atol=1e-5)
    assert t.allclose(out["probs"].double().log(), given, rtol=1e-5, atol=1e-5)
    assert t.allclose(entropy.double(), -(exact.exp() * exact).sum(-1), rtol=1e-5, atol=1e-5)
    assert t.equal(top.long(), t.sort(out["logits"], dim=-1, descending=True, stable=True).indices[:, :3])


def test_a_serving_loop(ops):
    """Ragged prompts in two chunks, then single tokens, eager and as a replayed graph whose page
    table, positions and tokens change in place; a request that ends gives its pages to another."""
    t = torch()
    for dim, page in ((64, 32), (128, 64)):
        say("serving", dim, page)
        model = Model(ops, dim, 1000, 7)
        batch, width = 3, 6
        cache = ops.kv_cache_paged(batch * width + 1, 2, page, dim)
        cache.buffer.fill_(math.nan)  # what no request has written is not looked at
        rng = np.random.default_rng(dim)
        order = rng.permutation(cache.pages)
        table = i32(order[:batch * width].reshape(batch, width).tolist())
        positions, lengths = i32([0, 0, 0]), i32([40, 7, 33])
        u = t.rand((batch,), device="cuda")
        prompt = t.randint(0, 1000, (batch, 40), device="cuda", dtype=t.int32)
        out = model.step(prompt, cache, table, positions, lengths, u)
        check_step(model, out, cache, table, positions, lengths)
        positions, lengths = positions + lengths, i32([20, 40, 0])
        out = model.step(prompt.flip(1).contiguous(), cache, table, positions, lengths, u)
        check_step(model, out, cache, table, positions, lengths)
        positions = positions + lengths
        ones = i32([1, 1, 1])
        tokens = out["tokens"].clone().view(batch, 1)
        eager_cache = ops.kv_cache_paged(cache.pages, 2, page, dim)
        eager_cache.buffer.copy_(cache.buffer)
        model.step(tokens, eager_cache, table, positions, ones, u)  # (warm)
        eager_cache.buffer.copy_(cache.buffer)
        graph = t.cuda.CUDAGraph()
        with t.cuda.graph(graph):
            captured = model.step(tokens, cache, table, positions, ones, u)
        for turn in range(4):
            if turn == 2:  # request 1 ends: its pages, in another order, are a new request's
                table[1] = table[1].flip(0)
                positions[1] = 0
            u.copy_(t.rand((batch,), device="cuda"))
            want = model.step(tokens, eager_cache, table, positions, ones, u)
            check_step(model, want, eager_cache, table, positions, ones)
            graph.replay()
            t.cuda.synchronize()
            for name in ("turned", "y", "logits", "tokens", "probs"):
                assert t.equal(captured[name], want[name]), (turn, name)
            for got, w in zip(captured["scores"], want["scores"]):
                assert t.equal(got, w), turn
            tokens.copy_(want["tokens"].view(batch, 1))
            positions.add_(1)


def test_requests_that_share_pages(ops):
    """Two requests over one instruction's pages answer as with copies of them."""
    t = torch()
    say("shared pages")
    gen = t.Generator("cuda").manual_seed(3)
    rand = lambda *s: t.randn(s, generator=gen, device="cuda", dtype=t.float16)  # noqa: E731
    cache = ops.kv_cache_paged(12, 4, 32, 64)
    k, v = rand(1, 4, 96, 64), rand(1, 4, 96, 64)
    ops.kv_append_paged(cache, k, v, i32([[4, 9, 2]]), 0)
    for i, j in ((4, 5), (9, 6), (2, 7)):
        cache.buffer[j] = cache.buffer[i]
    own_k, own_v = rand(2, 4, 5, 64), rand(2, 4, 5, 64)
    shared, apart = i32([[4, 9, 2, 0], [4, 9, 2, 1]]), i32([[4, 9, 2, 0], [5, 6, 7, 1]])
    ops.kv_append_paged(cache, own_k, own_v, shared, 96)
    q = rand(2, 8, 5, 64)
    assert t.equal(ops.attention_paged(q, cache, shared, 101), ops.attention_paged(q, cache, apart, 101))


def test_refusals(ops):
    t = torch()
    say("refusals")
    cache = ops.kv_cache_paged(4, 2, 32, 64)
    x, table, pos = t.zeros((2, 2, 3, 64), dtype=t.float16, device="cuda"), i32([[0, 1], [2, 3]]), i32([0, 0])
    q = t.zeros((2, 4, 3, 64), dtype=t.float16, device="cuda")
    rotary, odd = ops.rotary(64), ops.rotary(24)
    logits, tokens = t.zeros((2, 50), device="cuda"), i32([0, 1])
    lib, at = ops.lib, cache._at
    for call in (
            lambda: ops.rotate(x, ops.rotary(66), pos),                                   # wider than the rows
            lambda: ops.rotate(x, rotary, None),
            lambda: ops.rotate(x, rotary, [0, 2 ** 31]),
            lambda: ops.rotate(x, rotary, i32([0, 0, 0])),
            lambda: ops.rotate(x, rotary, i32([[0, 0]])),
            lambda: ops.rotate(x.view(2, 2, 192), rotary, pos),
            lambda: ops.rotate(x.detach().float().half().requires_grad_(), rotary, pos),
            lambda: ops.rotate(x[:, :, :0], rotary, pos),
            lambda: ops.kv_append_paged(cache, x[:, :1], x[:, :1], table, pos),           # heads
            lambda: ops.kv_append_paged(cache, x, x[:, :, :2], table, pos),               # v's shape
            lambda: ops.kv_append_paged(cache, x, x, table[:1], pos),                     # a row per request
            lambda: ops.kv_append_paged(cache, x, x, table.view(-1), pos),
            lambda: ops.kv_append_paged(cache, x, x, table, None),
            lambda: ops.kv_append_paged(cache, x, x, table, [0, 62]),                     # past the table
            lambda: ops.kv_append_paged(cache, x, x, table, -1),
            lambda: ops.kv_append_paged(cache, x, x, table, 0, lengths=4),
            lambda: ops.kv_append_paged(cache, *[x[:, :, :1].expand(2, 2, (1 << 20) + 1, 64)] * 2, table, pos),
            lambda: ops.kv_append_paged(cache, x, x, table, pos, q=q),                    # q without rotary
            lambda: ops.kv_append_paged(cache, x, x, table, pos, rotary=odd),
            lambda: ops.kv_append_paged(cache, x, x, table, pos, rotary=ops.rotary(128)),
            lambda: ops.kv_append_paged(cache, x, x, table, pos, rotary=rotary, q=q[:, :, :2]),
            lambda: ops.kv_read_paged(cache, table, pos, None, 0),
            lambda: ops.kv_read_paged(cache, table, [0], None, 3),
            lambda: ops.kv_read_paged(cache, table, 0, None, 65),
            lambda: ops.kv_read_paged(cache, table, pos, None, (1 << 20) + 1),
            lambda: ops.kv_read_paged(cache, table[:0], 0, None, 3),
            lambda: ops.attention_paged(q[:, :3].contiguous(), cache, table, 3),                       # heads
            lambda: ops.attention_paged(q[..., :32].contiguous(), cache, table, 3),
            lambda: ops.attention_paged(q, cache, table, None),
            lambda: ops.attention_paged(q, cache, table, 65),
            lambda: ops.attention_paged(q, cache, table, 3, q_lengths=4),
            lambda: ops.attention_paged(q, cache, table, 3, causal=1),
            lambda: ops.attention_paged(q, cache, table, 3, max_kv_length=-1),
            lambda: ops.logprobs(logits, tokens, top=65),
            lambda: ops.logprobs(logits, tokens, top=True),
            lambda: ops.logprobs(logits, i32([0])),
            lambda: ops.logprobs(logits, i32([[[0]], [[1]]])),
            lambda: ops.logprobs(t.zeros((2, (1 << 18) + 1), device="cuda"), tokens)):
        with pytest.raises(ValueError):
            call()
    for call in (
            lambda: ops.rotate(x.float(), rotary, pos), lambda: ops.rotate(x, None, pos),
            lambda: ops.rotate(x.transpose(2, 3), rotary, pos),                           # dims not contiguous
            lambda: ops.rotate(x, rotary, pos.long()),
            lambda: ops.kv_append_paged(cache, x, x, table.long(), pos),
            lambda: ops.kv_append_paged(cache, x, x, table.t(), pos),
            lambda: ops.kv_append_paged(ops.kv_cache_int8(1, 2, 64, 64), x, x, table, pos),
            lambda: ops.kv_append_int8(cache, x, x, 0, 0),
            lambda: ops.kv_append_paged(cache, x, x, table, pos, rotary=3),
            lambda: ops.kv_read_paged(cache, table.tolist(), pos, None, 3),
            lambda: ops.attention_paged(q.transpose(1, 2), cache, table, 3),
            lambda: ops.logprobs(logits.double(), tokens), lambda: ops.logprobs(logits, tokens.long()),
            lambda: ops.logprobs(logits.t(), tokens)):
        with pytest.raises(TypeError):
            call()
    # The C entry points' own checks: a status, a message, nothing queued.
    stream, dev = ctypes.c_size_t(0), 0
    p = lambda y: ctypes.c_void_p(y.data_ptr())  # noqa: E731
    s = (384, 192, 64)
    out = t.full_like(q, 7.0)
    rows = lambda **o: {"x": p(q), "s": (768, 192, 64), "y": p(out), "pos": p(pos), "each": 0, "turns": p(rotary.turns), "r": 64,  # noqa: E731
                        "il": 0, "amp": 1.0, "b": 2, "h": 4, "n": 3, "d": 64, **o}
    for o in (dict(x=None), dict(y=None), dict(pos=None), dict(turns=None), dict(r=0), dict(r=3), dict(r=66), dict(il=2), dict(each=2),
              dict(amp=math.nan), dict(b=0), dict(b=65536), dict(h=0), dict(n=0), dict(d=0), dict(s=(-1, 192, 64)), dict(n=1 << 30, d=64)):
        a = rows(**o)
        assert lib.ti_amd_rotate(a["x"], *a["s"], a["y"], a["pos"], a["each"], a["turns"], a["r"], a["il"], a["amp"], a["b"], a["h"],
                                 a["n"], a["d"], stream, dev) == 1, o
        assert lib.ti_v2_last_error()
    app = lambda **o: {"c": at, "k": p(x), "v": p(x), "s": s, "q": None, "qo": None, "t": p(table), "w": 2, "pos": p(pos), "turns": None,  # noqa: E731
                       "r": 0, "b": 2, "h": 0, "n": 3, **o}
    for o in (dict(c=None), dict(k=None), dict(v=None), dict(t=None), dict(w=0), dict(pos=None), dict(b=0), dict(n=0), dict(n=(1 << 20) + 1),
              dict(s=(384, -192, 64)), dict(q=p(q), qo=p(out), h=4), dict(turns=p(odd.turns), r=24),
              dict(turns=p(rotary.turns), r=64, q=p(q), qo=None, h=4), dict(turns=p(rotary.turns), r=64, q=p(q), qo=p(out), h=0)):
        a = app(**o)
        assert lib.ti_amd_kv_append_paged(a["c"], a["k"], *a["s"], a["v"], *a["s"], a["q"], 768, 192, 64, a["qo"], a["t"], a["w"], a["pos"], None,
                                          a["turns"], a["r"], 0, 1.0, a["b"], a["h"], a["n"], stream, dev) == 1, o
    lengths = i32([2000, 2000])
    wide = t.zeros((2, 64), dtype=t.int32, device="cuda")
    needed = lib.ti_amd_attention_paged_workspace(at, 64, 2, 4, 3, 0)
    work = t.zeros(needed + 16, dtype=t.uint8, device="cuda")
    ask = lambda **o: {"c": at, "q": p(q), "y": p(out), "t": p(wide), "w": 64, "kv": p(lengths), "ws": p(work), "n": needed, "h": 4, "l": 3,  # noqa: E731
                       "causal": 1, "max": 0, **o}
    assert needed > 0
    for o in (dict(c=None), dict(q=None), dict(y=None), dict(t=None), dict(w=0), dict(kv=None), dict(ws=None), dict(n=needed - 1),
              dict(ws=ctypes.c_void_p(work.data_ptr() + 4)), dict(h=3), dict(l=0), dict(l=1 << 21), dict(causal=2), dict(max=-1)):
        a = ask(**o)
        assert lib.ti_amd_attention_paged(a["c"], a["q"], a["y"], a["t"], a["w"], a["kv"], None, None, a["ws"], a["n"], 2, a["h"], a["l"], a["max"],
                                          a["causal"], stream, dev) == 1, o
    f = t.zeros(200, device="cuda")
    for o in (dict(dtype=2), dict(logits=None), dict(tokens=None), dict(lp=None), dict(h=None), dict(top=65), dict(top=-1), dict(top=3, tl=None),
              dict(given=0), dict(given=(1 << 16) + 1), dict(vocab=(1 << 18) + 1), dict(vocab=0), dict(batch=0)):
        a = {"logits": p(logits), "dtype": 1, "tokens": p(tokens), "lp": p(f), "h": p(f), "tl": p(f), "batch": 2, "vocab": 50, "given": 1, "top": 0, **o}
        assert lib.ti_amd_logprobs(a["logits"], a["dtype"], a["tokens"], a["lp"], a["h"], a["tl"], p(tokens), a["batch"], a["vocab"], a["given"],
                                   a["top"], stream, dev) == 1, o
    t.cuda.synchronize()
    assert (out == 7.0).all() and (f == 0).all() and (cache.buffer == 0).all()
