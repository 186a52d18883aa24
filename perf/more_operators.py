"""Rotary positions, a paged fp16 KV cache with the attention that reads it, and log
probabilities, as measurable cases.

``listed()`` gives the cases, ``draw(rng)`` another one of the same ranges,
``prepare`` what a serving program has in hand before the call, ``run`` one pass,
``work`` the bytes and operations it cannot do without and ``exact`` the same
outputs in 64-bit arithmetic.  Where ``own`` is false ``run`` computes the
operators in elementary torch operations, where it is true it calls ``NativeOps``:

* ``rotate``: rows turned by their positions, whole heads or part of them, in the
  half and the interleaved layout, with plain or stretched frequencies;
* ``write``: a step's or a prompt's new keys and values, cut out of the projection
  that made them, join a paged cache, keys and queries turned on the way; the
  written rows are read back;
* ``attention``: queries over a paged cache, single tokens and prompts' chunks;
* ``logprobs``: log probabilities of given tokens, the entropy of their row and the
  likeliest alternatives.
"""
import math
import random

import torch

own = False
DEV = "cuda"
VOCAB = 50257  # the GPT-2 vocabulary
_ops = None


def listed():
    return [
        # One decode step's queries and keys of a full batch, 12 heads, each at its own position.
        {"name": "rotate decode b32", "op": "rotate", "batch": 32, "heads": 24, "dim": 64, "q": 1, "rotated": 64,
         "interleaved": False, "scaling": None, "far": 1024},
        # Two long prompts' queries, interleaved pairs, frequencies stretched to four times the length.
        {"name": "rotate prompts long", "op": "rotate", "batch": 2, "heads": 32, "dim": 128, "q": 6001, "rotated": 128,
         "interleaved": True, "scaling": "parts", "far": 100000},
        # A batch of prompts of which only the first half of each head is turned.
        {"name": "rotate part of head", "op": "rotate", "batch": 8, "heads": 25, "dim": 64, "q": 777, "rotated": 32,
         "interleaved": False, "scaling": "linear", "far": 4096},
        # One decode step of a full batch: 32 tokens join their pages (one layer), their queries are turned.
        {"name": "paged write decode b32", "op": "write", "batch": 32, "heads": 12, "kv_heads": 12, "dim": 64, "q": 1,
         "page": 64, "rotated": 64, "interleaved": False, "scaling": None, "far": 1024, "low": 1},
        # Eight ragged prompts of up to 1000 tokens, 25 heads, join theirs.
        {"name": "paged write prompts", "op": "write", "batch": 8, "heads": 25, "kv_heads": 25, "dim": 64, "q": 1000,
         "page": 32, "rotated": 64, "interleaved": False, "scaling": "base", "far": 64, "low": 300},
        # One request's token over a short cache: the smallest call a decode loop makes.
        {"name": "paged attention decode b1", "op": "attention", "batch": 1, "heads": 12, "kv_heads": 12, "dim": 64,
         "q": 1, "page": 64, "kv": 300, "low": 300, "causal": True},
        # A full batch with ragged caches of up to 1024 keys.
        {"name": "paged attention decode b32", "op": "attention", "batch": 32, "heads": 12, "kv_heads": 12, "dim": 64,
         "q": 1, "page": 32, "kv": 1024, "low": 128, "causal": True},
        # Long contexts, four query heads to a key head.
        {"name": "paged attention decode long", "op": "attention", "batch": 16, "heads": 32, "kv_heads": 8, "dim": 128,
         "q": 1, "page": 64, "kv": 32768, "low": 12000, "causal": True},
        # A later chunk of two long prompts, an odd number of queries, four query heads to a key head.
        {"name": "paged attention chunk", "op": "attention", "batch": 2, "heads": 32, "kv_heads": 8, "dim": 128,
         "q": 777, "page": 128, "kv": 6001, "low": 4500, "causal": True},
        # What a step's sampled tokens had for probabilities, with five alternatives each.
        {"name": "logprobs b1", "op": "logprobs", "batch": 1, "vocab": VOCAB, "dtype": "f32", "given": 1, "top": 5,
         "masked": False},
        {"name": "logprobs b32", "op": "logprobs", "batch": 32, "vocab": VOCAB, "dtype": "f16", "given": 1, "top": 20,
         "masked": False},
        # Every token of 768 prompt positions scored over a large, odd vocabulary.
        {"name": "logprobs scoring", "op": "logprobs", "batch": 768, "vocab": 128257, "dtype": "f32", "given": 1,
         "top": 5, "masked": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _turn(rng, dim):
    """How heads are turned: a part or all of them, and the frequencies."""
    return {"rotated": rng.choice((dim, dim, dim // 2, dim // 4)), "interleaved": rng.random() < 0.4,
            "scaling": rng.choice((None, None, "linear", "base", "parts")), "far": _log(rng, 64, 131072)}


def draw(rng: random.Random):
    """A case of the listed ones' ranges."""
    op = rng.choice(("rotate", "rotate", "write", "write", "attention", "attention", "attention", "logprobs",
                     "logprobs"))
    if op == "logprobs":
        vocab = rng.choice((VOCAB, _log(rng, 1000, 160000)))
        batch = min(_log(rng, 1, 2048), 98_000_000 // vocab)
        return {"op": op, "batch": batch, "vocab": vocab, "dtype": rng.choice(("f32", "f16")),
                "given": rng.choice((1, 1, 1, 4)), "top": rng.choice((0, 1, 5, 5, 20)), "masked": rng.random() < 0.3}
    if op == "rotate":
        dim = rng.choice((64, 64, 128, 128, 80, 256))
        batch, heads, q = _log(rng, 1, 64), rng.choice((1, 8, 12, 25, 32, 40)), _log(rng, 1, 8192)
        q = max(1, min(q, 49_000_000 // (batch * heads * dim)))
        return {"op": op, "batch": batch, "heads": heads, "dim": dim, "q": q, **_turn(rng, dim)}
    dim = rng.choice((64, 128))
    kv_heads, group = rng.choice(((12, 1), (25, 1), (8, 4), (4, 7), (2, 8), (1, 12)))
    page = rng.choice((32, 64, 64, 128, 256))
    if op == "write":
        batch, n = _log(rng, 1, 64), _log(rng, 1, 16384)
        n = max(1, min(n, 29_000_000 // (batch * kv_heads * (group + 2) * dim)))
        return {"op": op, "batch": batch, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "q": n,
                "page": page, "low": max(1, int(n * rng.choice((0.1, 0.5, 1.0)))), **_turn(rng, dim)}
    heads = kv_heads * group
    if rng.random() < 0.65:  # single tokens, and the few of a checked draft
        q = rng.choice((1, 1, 1, 1, 2, 4, 5))
        batch, kv = _log(rng, 1, 64), _log(rng, 16, 32768)
        kv = max(16, min(kv, 370_000_000 // (batch * kv_heads * dim)))
    else:
        batch, q = _log(rng, 1, 16), _log(rng, 8, 2048)
        kv = q if rng.random() < 0.5 else q + _log(rng, 1, 4096)
        batch = max(1, min(batch, 210_000_000 // (heads * q * kv)))
    return {"op": "attention", "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim, "q": q, "page": page,
            "kv": kv, "low": max(q, int(kv * rng.choice((0.1, 0.5, 1.0)))), "causal": rng.random() < 0.8}


# -- inputs ---------------------------------------------------------------------
def _lengths(case, high):
    """Ragged lengths in [low, high], one of them high; the same for every seed (work() counts them)."""
    rng = random.Random(case["batch"] * 7919 + high)
    got = [rng.randint(min(case["low"], high), high) for _ in range(case["batch"])]
    got[rng.randrange(case["batch"])] = high
    return got


def _gen(seed):
    return torch.Generator(DEV).manual_seed(int(seed) * 2 + 1)


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float16)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _keys_values(gen, rows, kv_heads, n, dim):
    """fp16 keys with a few large channels, and values whose size varies from token to token."""
    k = _normal(gen, rows, kv_heads, n, dim)
    k += _normal(gen, 1, kv_heads, 1, dim) * (torch.arange(dim, device=DEV) % 16 == 3) * 4
    v = _normal(gen, rows, kv_heads, n, dim)
    v *= torch.rand((rows, kv_heads, n, 1), generator=gen, device=DEV, dtype=torch.float16) + 0.25
    return k, v


def _table(gen, batch, tokens, page):
    """Page tables [batch, ceil(tokens / page)] of a cache handed out in no order, and its number of pages."""
    width = -(-tokens // page)
    pages = batch * width + 3
    return torch.randperm(pages, generator=gen, device=DEV)[:batch * width].view(batch, width).int(), pages


def _inputs(case, seed):
    """The case's tensors, from the seed alone."""
    gen, op = _gen(seed), case["op"]
    if op == "logprobs":
        batch, vocab = case["batch"], case["vocab"]
        logits = torch.randn((batch, vocab), generator=gen, device=DEV) * 2.0
        # A few tokens stand out, as after a real prompt.
        logits += 9.0 * torch.rand((batch, vocab), generator=gen, device=DEV).pow(400.0)
        tokens = torch.randint(0, vocab, (batch, case["given"]), generator=gen, device=DEV, dtype=torch.int32)
        if case["masked"]:  # nine of ten tokens a grammar rules out, the given ones not among them
            out = torch.rand((batch, vocab), generator=gen, device=DEV) < 0.9
            logits[out.scatter_(1, tokens.long(), False)] = -math.inf
        return {"logits": logits.half() if case["dtype"] == "f16" else logits,
                "tokens": tokens if case["given"] > 1 else tokens[:, 0].contiguous()}
    batch, dim, q = case["batch"], case["dim"], case["q"]
    if op == "rotate":
        return {"x": _normal(gen, batch, case["heads"], q, dim),
                "positions": (torch.rand((batch,), generator=gen, device=DEV) * case["far"]).int()}
    kv_heads, heads = case["kv_heads"], case["heads"]
    if op == "write":
        # The projection of a step's or a prompt's rows: queries, keys and values side by side.
        qkv = _normal(gen, batch, q, heads + 2 * kv_heads, dim).transpose(1, 2)
        far = min(case["far"], 4 * q + 2048)
        table, pages = _table(gen, batch, far + q, case["page"])
        return {"q": qkv[:, :heads], "k": qkv[:, heads:heads + kv_heads], "v": qkv[:, heads + kv_heads:],
                "table": table, "pages": pages, "lengths": _ints(_lengths(case, q)),
                "positions": (torch.rand((batch,), generator=gen, device=DEV) * far).int()}
    k, v = _keys_values(gen, batch, kv_heads, case["kv"], dim)
    table, pages = _table(gen, batch, case["kv"], case["page"])
    return {"k": k, "v": v, "table": table, "pages": pages, "lengths": _ints(_lengths(case, case["kv"])),
            "q": _normal(gen, batch, heads, q, dim) * 1.5}


SCALE = {"linear": {"factor": 8.0}, "base": {"factor": 4.0}, "parts": {"factor": 4.0, "original_length": 8192}}


def prepare(case, seed):
    state = {"case": dict(case), **_inputs(case, seed)}
    op, ops = case["op"], _native() if own else None
    state["ops"] = ops
    if op in ("rotate", "write"):
        if own:
            state["rotary"] = ops.rotary(case["rotated"], interleaved=case["interleaved"], scaling=case["scaling"],
                                         **SCALE.get(case["scaling"], {}))
        else:
            state["rotary"] = _frequencies(case)
    if op in ("write", "attention"):
        pages = state.pop("pages")
        if own:  # the cache that the serving program keeps
            cache = state["cache"] = ops.kv_cache_paged(pages, case["kv_heads"], case["page"], case["dim"])
        else:
            shape = (pages, case["kv_heads"], case["page"], case["dim"])
            cache = state["cache"] = {"k": torch.zeros(shape, dtype=torch.float16, device=DEV),
                                      "v": torch.zeros(shape, dtype=torch.float16, device=DEV)}
    if op == "attention":  # filled by earlier steps
        k, v = state.pop("k"), state.pop("v")
        zeros = torch.zeros(case["batch"], dtype=torch.int32, device=DEV)
        if own:
            ops.kv_append_paged(cache, k, v, state["table"], zeros)
        else:
            _append(cache, k, v, state["table"], zeros, zeros + case["kv"])
    return state


def _native():
    global _ops
    if _ops is None:
        from tinyinfer_amd.native_ops import NativeOps
        _ops = NativeOps()
    return _ops


# -- the plain forms --------------------------------------------------------------
def _frequencies(case):
    """Angle per position of every pair, and the factor on turned values."""
    count, base, how = case["rotated"] // 2, 10000.0, case["scaling"]
    got = SCALE.get(how, {})
    if how == "base":
        base *= got["factor"] ** (2 * count / max(2 * count - 2, 1))
    f = base ** (-torch.arange(count, dtype=torch.float64, device=DEV) / count)
    if how == "linear":
        f = f / got["factor"]
    if how == "parts":  # pairs that turn often over the original length keep their frequency, slow ones are stretched
        turns = got["original_length"] * f / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        f = f * keep + f / got["factor"] * (1 - keep)
    return f


def _rotate(x, frequencies, positions, rotated, interleaved):
    """x [B, H, Q, D]: row i is token positions[b] + i.  Angles in 64 bits."""
    at = positions.double()[:, None] + torch.arange(x.shape[2], device=DEV)
    angle = (at[..., None] * frequencies)[:, None]
    cos, sin = angle.cos().float(), angle.sin().float()
    part = x[..., :rotated].float()
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = part[..., :rotated // 2], part[..., rotated // 2:]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((turned.half(), x[..., rotated:]), -1)


def _at(table, page, heads, n, positions):
    """Index of tokens positions[b] .. + n - 1 in the first three axes of a cache, [B, G, n]."""
    t = positions.long()[:, None] + torch.arange(n, device=DEV)
    where = table.long().gather(1, t // page)
    return where[:, None, :], torch.arange(heads, device=DEV)[None, :, None], (t % page)[:, None, :]


def _live(n, lengths):
    return (torch.arange(n, device=DEV) < lengths[:, None])[:, None, :, None]


def _append(cache, k, v, table, positions, lengths):
    at = _at(table, cache["k"].shape[2], k.shape[1], k.shape[2], positions)
    live = _live(k.shape[2], lengths)
    for name, x in (("k", k), ("v", v)):
        cache[name][at] = torch.where(live, x, cache[name][at])


def _write(state):
    case, cache, table, positions, lengths = (state[x] for x in ("case", "cache", "table", "positions", "lengths"))
    n = case["q"]
    if own:
        ops = state["ops"]
        q = ops.kv_append_paged(cache, state["k"], state["v"], table, positions, lengths=lengths,
                                rotary=state["rotary"], q=state["q"])
        return (q, *ops.kv_read_paged(cache, table, positions, lengths, n))
    turn = lambda x: _rotate(x, state["rotary"], positions, case["rotated"], case["interleaved"])  # noqa: E731
    q = torch.where(_live(n, lengths), turn(state["q"]), torch.zeros_like(state["q"]))
    _append(cache, turn(state["k"]), state["v"], table, positions, lengths)
    at, live = _at(table, case["page"], case["kv_heads"], n, positions), _live(n, lengths)
    read = [torch.where(live, cache[name][at], torch.zeros((), dtype=torch.float16, device=DEV)) for name in ("k", "v")]
    return (q, *read)


def _attention(state):
    case, cache, table, lengths = (state[x] for x in ("case", "cache", "table", "lengths"))
    if own:
        return state["ops"].attention_paged(state["q"], cache, table, lengths, causal=case["causal"])
    batch, heads, kv_heads, q, n, dim = (case[x] for x in ("batch", "heads", "kv_heads", "q", "kv", "dim"))
    k, v = (cache[name][table.long()].transpose(1, 2).reshape(batch, kv_heads, -1, dim)[:, :, :n].float()
            for name in ("k", "v"))
    key, end = torch.arange(n, device=DEV), lengths[:, None].expand(-1, q)
    if case["causal"]:  # the queries are each request's last ones
        end = end - q + 1 + torch.arange(q, device=DEV)
    rows = state["q"].float().view(batch, kv_heads, -1, dim)
    s = torch.matmul(rows, k.transpose(-1, -2)) * (1.0 / math.sqrt(dim))
    s = s.view(batch, kv_heads, heads // kv_heads, q, n).masked_fill(~(key < end[..., None])[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    total = p.sum(-1).view(batch, heads, -1, 1)
    return (torch.matmul(p.view(batch, kv_heads, -1, n), v).view(batch, heads, -1, dim) / total).half()


def _logprobs(state):
    logits, tokens, top = state["logits"], state["tokens"], state["case"]["top"]
    if own:
        return state["ops"].logprobs(logits, tokens, top=top)
    x = logits.float()
    x = x - x.amax(-1, keepdim=True)
    e = torch.exp(x)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    entropy = (log_total - (e * torch.where(e > 0, x, 0.0)).sum(-1, keepdim=True) / total)[:, 0]
    given = x.gather(1, tokens.long().view(x.shape[0], -1)) - log_total
    # The order of tokens: by logit, ties by index, as one whole number each.
    bits = (logits.float() + 0.0).view(torch.int32)
    rank = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long() * 2 ** 31 - torch.arange(x.shape[1], device=DEV)
    best = torch.topk(rank, top, -1).indices
    return given.view(tokens.shape), entropy, x.gather(1, best) - log_total, best.int()


def run(state):
    op = state["case"]["op"]
    if op == "rotate":
        case = state["case"]
        if own:
            return state["ops"].rotate(state["x"], state["rotary"], state["positions"])
        return _rotate(state["x"], state["rotary"], state["positions"], case["rotated"], case["interleaved"])
    return {"write": _write, "attention": _attention, "logprobs": _logprobs}[op](state)


def work(case):
    op, batch = case["op"], case["batch"]
    if op == "logprobs":
        size = 2 if case["dtype"] == "f16" else 4
        return {"bytes": batch * (case["vocab"] * size + 8 * case["given"] + 4 + 8 * case["top"]),
                "flops": 5 * batch * case["vocab"]}
    dim, q = case["dim"], case["q"]
    if op == "rotate":
        values = batch * case["heads"] * q
        return {"bytes": 4 * dim * values, "flops": 3 * case["rotated"] * values}
    kv_heads, heads = case["kv_heads"], case["heads"]
    if op == "write":
        live = sum(_lengths(case, q))
        rows = live * (heads + 2 * kv_heads * 3) + batch * q * (heads + 2 * kv_heads)  # read, cached, read back; put out
        return {"bytes": 2 * dim * rows, "flops": 3 * case["rotated"] * live * (heads + kv_heads)}
    lengths = _lengths(case, case["kv"])
    pairs = sum(n * q - (q * (q - 1) // 2 if case["causal"] else 0) for n in lengths)
    return {"bytes": sum(lengths) * kv_heads * 4 * dim + batch * heads * q * dim * 4, "flops": 4 * dim * heads * pairs}


# -- the definitions in 64 bits ----------------------------------------------------
def _exact_turned(case, x, positions):
    """Each pair as a complex number, times e^(i angle)."""
    half, out = case["rotated"] // 2, x.double().clone()
    i = torch.arange(half, dtype=torch.float64, device=DEV)
    scale = SCALE.get(case["scaling"], {})
    base = math.log(10000.0)
    if case["scaling"] == "base":
        base += math.log(scale["factor"]) * half / (half - 1)
    f = torch.exp(-base * i / half)
    if case["scaling"] == "linear":
        f /= scale["factor"]
    if case["scaling"] == "parts":
        w = torch.clamp((scale["original_length"] / (2 * math.pi) * f - 1) / 31, min=0, max=1)
        f *= w + (1 - w) / scale["factor"]
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["interleaved"] else (slice(0, half),
                                                                                               slice(half, 2 * half))
    for b in range(x.shape[0]):
        t = float(positions[b]) + torch.arange(x.shape[2], dtype=torch.float64, device=DEV)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV).expand(t.numel(), half), torch.outer(t, f))
        z = torch.complex(out[b, ..., first].clone(), out[b, ..., second].clone()) * turn
        out[b, ..., first], out[b, ..., second] = z.real, z.imag
    return out


def exact(case, seed):
    x, op = _inputs(case, seed), case["op"]
    if op == "rotate":
        return _exact_turned(case, x["x"], x["positions"])
    if op == "logprobs":
        given, entropy, best, index = [], [], [], []
        for b in range(case["batch"]):
            row = x["logits"][b].double()
            lp = torch.log_softmax(row, 0)
            given.append(lp[x["tokens"][b].long()])
            entropy.append(-torch.special.xlogy(lp.exp(), lp.exp()).sum())
            # Everything from the last kept value on, put in order: by value, ties by index.
            keep = max(case["top"], 1)
            at = torch.nonzero(row >= torch.topk(row, keep).values[-1])[:, 0]
            at = at[torch.argsort(row[at], descending=True, stable=True)][:case["top"]]
            best.append(lp[at])
            index.append(at.int())
        return tuple(torch.stack(y) for y in (given, entropy, best, index))
    lengths = x["lengths"].tolist()
    if op == "write":
        out = [_exact_turned(case, x["q"], x["positions"]), _exact_turned(case, x["k"], x["positions"]),
               x["v"].double()]
        for y in out:
            for b, n in enumerate(lengths):
                y[b, :, n:] = 0
        return tuple(out)
    heads, kv_heads, q = case["heads"], case["kv_heads"], case["q"]
    group = heads // kv_heads
    out = torch.zeros(x["q"].shape, dtype=torch.float64, device=DEV)
    for b, n in enumerate(lengths):
        ends = (n - q + 1 + torch.arange(q, device=DEV)) if case["causal"] else torch.full((q,), n, device=DEV)
        unseen = torch.arange(n, device=DEV)[None, :] >= ends.repeat(group)[:, None]
        for g in range(kv_heads):
            rows = x["q"][b, g * group:(g + 1) * group].double().reshape(-1, case["dim"])
            s = (rows @ x["k"][b, g, :n].double().t() / math.sqrt(case["dim"])).masked_fill(unseen, -math.inf)
            out[b, g * group:(g + 1) * group] = (torch.softmax(s, -1) @ x["v"][b, g, :n].double()).view(group, q, -1)
    return out
