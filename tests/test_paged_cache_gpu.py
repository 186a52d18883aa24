"""GPU tests of the paged fp16 KV cache (kv_append_paged, kv_read_paged): contents bit for
bit against a plain cache in numpy; turned keys and queries equal ``rotate``'s (which has
its own test against 80-bit angles) bit for bit."""
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


class Plain:
    """The same cache in numpy: [pages, heads, page, D] twice."""

    def __init__(self, pages, heads, page, dim):
        self.k = np.zeros((pages, heads, page, dim), np.float16)
        self.v = self.k.copy()
        self.page = page

    def append(self, k, v, table, positions, lengths):
        for b, n in enumerate(lengths):
            for i in range(max(n, 0)):
                t = int(positions[b]) + i
                if 0 <= t < table.shape[1] * self.page and 0 <= table[b, t // self.page] < len(self.k):
                    self.k[table[b, t // self.page], :, t % self.page] = k[b, :, i]
                    self.v[table[b, t // self.page], :, t % self.page] = v[b, :, i]

    def read(self, table, positions, lengths, rows):
        out = np.zeros((2, len(table), self.k.shape[1], rows, self.k.shape[3]), np.float16)
        for b, n in enumerate(lengths):
            for i in range(min(max(n, 0), rows)):
                t = int(positions[b]) + i
                if 0 <= t < table.shape[1] * self.page and 0 <= table[b, t // self.page] < len(self.k):
                    out[0, b, :, i] = self.k[table[b, t // self.page], :, t % self.page]
                    out[1, b, :, i] = self.v[table[b, t // self.page], :, t % self.page]
        return out


def same(got, want):
    got, want = np.ascontiguousarray(got).view(np.uint16), np.ascontiguousarray(want).view(np.uint16)
    bad = got != want
    assert not bad.any(), f"{bad.sum()} differ, first at {np.argwhere(bad)[0]}"


def tables(rng, batch, width, spare=2):
    pages = batch * width + spare
    return rng.permutation(pages)[:batch * width].reshape(batch, width).astype(np.int32), pages


@pytest.mark.parametrize("dim,heads,batch,rows,page,width", [
    (64, 12, 3, 1, 32, 4), (128, 2, 5, 1, 64, 2), (64, 3, 2, 8, 32, 3), (64, 3, 2, 9, 64, 2), (128, 5, 2, 8, 256, 1),
    (64, 2, 2, 64, 32, 5), (64, 1, 3, 65, 64, 4), (128, 3, 2, 130, 128, 3), (64, 25, 1, 200, 32, 9), (128, 1, 1, 1, 1024, 1),
    (128, 7, 2, 100, 32, 6), (64, 5, 4, 33, 1024, 1)])
def test_append_then_read(ops, dim, heads, batch, rows, page, width):
    say("append/read", dim, heads, batch, rows, page, width)
    rng = np.random.default_rng(dim + 7 * heads + rows)
    table, pages = tables(rng, batch, width)
    cache = ops.kv_cache_paged(pages, heads, page, dim)
    plain = Plain(pages, heads, page, dim)
    for turn in range(4):
        k, v = (rng.standard_normal((batch, heads, rows, dim)).astype(np.float16) for _ in range(2))
        k[0, 0, 0, :3], v[-1, -1, -1, -3:] = [np.nan, np.inf, -0.0], [65504, -np.inf, 2.0 ** -24]
        pos = rng.integers(0, width * page - rows + 1, batch).astype(np.int32)
        lens = rng.integers(0, rows + 1, batch).astype(np.int32) if turn else np.full(batch, rows, np.int32)
        assert ops.kv_append_paged(cache, dev(k), dev(v), dev(table), dev(pos), lengths=dev(lens) if turn else None) is None
        plain.append(k, v, table, pos, lens)
        # Every token of every page, in another order, and the ragged window.
        other = rng.permutation(pages).astype(np.int32).reshape(1, -1)
        got = ops.kv_read_paged(cache, dev(other), 0, pages * page, pages * page)
        want = plain.read(other, [0], [pages * page], pages * page)
        same(host(got[0]), want[0])
        same(host(got[1]), want[1])
        got = ops.kv_read_paged(cache, dev(table), dev(pos), dev(lens), rows)
        want = plain.read(table, pos, lens, rows)
        same(host(got[0]), want[0])
        same(host(got[1]), want[1])


@pytest.mark.parametrize("dim,heads,q_heads,rows,rotated,interleaved", [
    (64, 12, 12, 1, 64, False), (128, 8, 32, 1, 128, True), (64, 1, 71, 5, 16, False), (128, 4, 28, 77, 64, False),
    (64, 25, 25, 40, 32, True), (128, 2, 1, 300, 128, False), (64, 30, 2, 3, 48, False)])
def test_rotation_on_the_way(ops, dim, heads, q_heads, rows, rotated, interleaved):
    """From slices of one projection: keys and queries are turned as rotate turns them."""
    say("rotation", dim, heads, q_heads, rows, rotated, interleaved)
    t = torch()
    rng = np.random.default_rng(rows + rotated)
    batch, page = 3, 32
    width = (rows + 50) // page + 2
    table, pages = tables(rng, batch, width)
    cache = ops.kv_cache_paged(pages, heads, page, dim)
    rotary = ops.rotary(rotated, interleaved=interleaved, amplitude=1.125)
    qkv = dev(rng.standard_normal((batch, rows, q_heads + 2 * heads, dim)).astype(np.float16)).transpose(1, 2)
    q, k, v = qkv[:, :q_heads], qkv[:, q_heads:q_heads + heads], qkv[:, q_heads + heads:]
    pos, lens = i32([0, 31, 50]), i32([rows, max(rows - 1, 1), 0])
    turned = ops.kv_append_paged(cache, k, v, dev(table), pos, lengths=lens, rotary=rotary, q=q)
    gk, gv = ops.kv_read_paged(cache, dev(table), pos, lens, rows)
    live = (t.arange(rows, device="cuda") < lens[:, None])[:, None, :, None]
    zero = t.zeros((), dtype=t.float16, device="cuda")
    for got, want in ((turned, ops.rotate(q, rotary, pos)), (gk, ops.rotate(k, rotary, pos)), (gv, v)):
        same(host(got), host(t.where(live, want, zero)))
    # Without queries, and contiguous keys: the same cache.
    again = ops.kv_cache_paged(pages, heads, page, dim)
    assert ops.kv_append_paged(again, k.contiguous(), v.contiguous(), dev(table), pos, lengths=lens, rotary=rotary) is None
    assert t.equal(again.buffer, cache.buffer)


def test_what_lies_outside_is_not_written(ops):
    """Pages outside the cache, positions outside the table, lengths below 0 and above the rows."""
    say("outside")
    rng = np.random.default_rng(11)
    heads, dim, page, rows = 2, 64, 32, 40
    cache, plain = ops.kv_cache_paged(6, heads, page, dim), Plain(6, heads, page, dim)
    table = np.array([[0, -1, 1], [6, 2, 2 ** 31 - 1], [3, 4, 5], [-2 ** 31, 1 << 20, -5]], np.int32)
    for pos, lens in (([0, 20, 90, 0], [40, 40, 40, 40]), ([-10, 31, -2 ** 31, 5], [40, -3, 40, 9]),
                      ([95, 64, 2 ** 31 - 1, 2 ** 31 - 20], [2, 41, 40, 40])):
        k, v = (rng.standard_normal((4, heads, rows, dim)).astype(np.float16) for _ in range(2))
        ops.kv_append_paged(cache, dev(k), dev(v), dev(table), i32(pos), lengths=i32(lens))
        plain.append(k, v, table, pos, np.minimum(lens, rows))
        ops.kv_append_paged(cache, dev(k[:, :, :2]), dev(v[:, :, :2]), dev(table), i32(pos), lengths=i32(np.minimum(lens, 2)))
        plain.append(k[:, :, :2], v[:, :, :2], table, pos, np.minimum(lens, 2))
        everything = np.arange(6, dtype=np.int32)[None]
        got, want = ops.kv_read_paged(cache, dev(everything), 0, 192, 192), plain.read(everything, [0], [192], 192)
        same(host(got[0]), want[0])
        same(host(got[1]), want[1])
        got, want = ops.kv_read_paged(cache, dev(table), i32(pos), i32(lens), rows), plain.read(table, pos, lens, rows)
        same(host(got[0]), want[0])
        same(host(got[1]), want[1])


def test_pages_are_copied_as_rows_of_the_buffer(ops):
    say("page copy")
    t = torch()
    rng = np.random.default_rng(3)
    cache = ops.kv_cache_paged(4, 3, 64, 128)
    k, v = (dev(rng.standard_normal((1, 3, 64, 128)).astype(np.float16)) for _ in range(2))
    ops.kv_append_paged(cache, k, v, i32([[1]]), 0)
    cache.buffer[3] = cache.buffer[1]
    gk, gv = ops.kv_read_paged(cache, i32([[3]]), 0, 64, 64)
    assert t.equal(gk, k) and t.equal(gv, v)


def test_unaligned_inputs(ops):
    """Rows that start at any even address."""
    say("unaligned")
    t = torch()
    rng = np.random.default_rng(13)
    rotary = ops.rotary(32)
    for rows in (1, 40):
        flat = dev(rng.standard_normal(3 + 3 * 2 * 5 * rows * 64).astype(np.float16))
        q, k, v = flat[3:].view(3, 2, 5, rows, 64)
        table = i32([[0, 1, 2], [3, 4, 5]])
        a, b = ops.kv_cache_paged(6, 5, 32, 64), ops.kv_cache_paged(6, 5, 32, 64)
        x = ops.kv_append_paged(a, k, v, table, [3, 50], rotary=rotary, q=q)
        y = ops.kv_append_paged(b, k.clone(), v.clone(), table, [3, 50], rotary=rotary, q=q.clone())
        assert t.equal(x, y) and t.equal(a.buffer, b.buffer)


def test_a_cache_beyond_32_bits(ops):
    """Pages whose values lie more than 2^32 values, and 2^33 bytes, into the buffer."""
    say("large cache")
    t = torch()
    pages = (2 ** 32 // (8 * 2 * 1024 * 128)) + 40
    cache = ops.kv_cache_paged(pages, 8, 1024, 128)
    rng = np.random.default_rng(17)
    k, v = (dev(rng.standard_normal((2, 8, 1500, 128)).astype(np.float16)) for _ in range(2))
    table = i32([[pages - 1, 0], [pages - 2, pages - 3]])
    ops.kv_append_paged(cache, k, v, table, 100)
    gk, gv = ops.kv_read_paged(cache, table, 100, 1500, 1500)
    assert t.equal(gk, k) and t.equal(gv, v)
    q = dev(rng.standard_normal((2, 16, 1, 128)).astype(np.float16))
    small = ops.kv_cache_paged(4, 8, 1024, 128)
    near = i32([[0, 1], [2, 3]])
    ops.kv_append_paged(small, k, v, near, 100)
    assert t.equal(ops.attention_paged(q, cache, table, 1600), ops.attention_paged(q, small, near, 1600))
    del cache
    t.cuda.empty_cache()


def test_the_longest_append(ops):
    """2^20 rows in one call, all the same in memory, of which the last lie where they belong."""
    t = torch()
    say("2^20 rows")
    rows, page = 1 << 20, 1024
    cache = ops.kv_cache_paged(rows // page, 1, page, 128)
    table = i32(np.arange(rows // page)[::-1].reshape(1, -1).copy())
    row = t.randn((1, 1, 1, 128), device="cuda", dtype=t.float16)
    k = row.expand(1, 1, rows, 128)
    rotary = ops.rotary(128)
    ops.kv_append_paged(cache, k, -row.expand(1, 1, rows, 128), table, 0, rotary=rotary)
    for at in (0, 4096, rows - 3):
        got_k, got_v = ops.kv_read_paged(cache, table, at, None, 3)
        assert t.equal(got_k, ops.rotate(k[:, :, :3], rotary, at)) and t.equal(got_v, -row.expand(1, 1, 3, 128)), at
