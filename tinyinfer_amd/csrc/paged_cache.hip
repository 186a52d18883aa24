// The paged fp16 KV cache: rows join it, keys turned by their positions on the way, and
// are read back.  Layout in paged_cache.hpp, angles in rotary.hpp.
//
// Keys (and queries, into their own output) are taken 16 values to a lane, which walks
// over heads with one set of cosines and sines.  Values are taken 8 dims by 8 tokens to a
// lane: eight loads of 16 bytes, an 8 x 8 turn in registers (32 byte permutations, the rest
// of it is naming), eight stores of 16 bytes that with the neighbouring lanes' fill whole
// records.  Tokens that are not the call's own keep what they hold: a lane whose 8 are not
// all to be written stores single values.  One launch: a workgroup takes some heads of the
// queries, the keys or the values of a range of tokens that starts where a record does, and
// neighbouring ones the same tokens of other heads, which lie side by side where q, k and v are
// slices of one projection.
//
// What bounds it: memory (8 prompts of up to 1000 tokens, 25 heads of 64: append 26 us, of which the
// same bytes copied take 23; read back 20.5, 4.1 TB/s, or 16.6 where the rows are still in the last
// cache), and the launch for single tokens (32 requests of 12 heads of 64: 4.7 and 4.1 us).
#include "paged_cache.hpp"
#include "rotary.hpp"

namespace tia {
namespace {

typedef unsigned short u16x8_t __attribute__((ext_vector_type(8)));

__device__ __forceinline__ int live_rows(const int32_t* lengths, int b, int rows) {
  return lengths ? min(max(lengths[b], 0), rows) : rows;
}

// Where head `head` of token t of request b lies, or null: its page's K (V is page_size * D behind).
__device__ __forceinline__ uint16_t* head_at(const KvPaged& c, const PageTable& p, int b, int64_t t, int head) {
  if (t < 0 || t >= int64_t(p.width) * c.page_size) return nullptr;
  const int page = p.table[int64_t(b) * p.width + (t >> __builtin_ctz(c.page_size))];
  if (page < 0 || page >= c.page_count) return nullptr;
  return c.pages + (int64_t(page) * c.kv_heads + head) * paged_head_size(c);
}

// 16 values of heads [h0, h1) of one row of the queries (keys: false) or the keys.
template <int D, int HC>
__device__ __forceinline__ void append_turned(const PagedAppendArgs& a, bool keys, int b, int row, int u, int h0, int h1) {
  const Rows& from = keys ? a.k : a.q;
  const uint16_t* x = from.at + b * from.batch + row * from.row;
  const bool live = row < live_rows(a.lengths, b, a.rows);
  const int64_t t = int64_t(a.positions[b]) + row;
  const RowUnit unit = row_unit(a.rotary, u);
  uint16_t* y;
  int64_t step;
  int second;  // the second piece's place behind the first's
  if (keys) {
    if (!live || !(y = head_at(a.cache, a.pages, b, t, 0))) return;
    const int r = int(t) & (a.cache.page_size - 1), first = paged_k_at(r, unit.first, D);
    y += first;
    second = paged_k_at(r, unit.second, D) - first;
    step = paged_head_size(a.cache);
  } else {
    y = a.q_out + (int64_t(b) * a.heads * a.rows + row) * D + unit.first;
    second = unit.second - unit.first;
    step = int64_t(a.rows) * D;
    if (!live) {
      for (int h = h0; h < h1; ++h) {
        store_half8(y + h * step, half8_t{});
        store_half8(y + h * step + second, half8_t{});
      }
      return;
    }
  }
  turn_heads<HC>(a.rotary, unit, u, t, x, from.head, y, step, second, h0, h1);
}

// 8 rows of 8 values the other way round.
__device__ __forceinline__ void transpose8(u32x4_t (&x)[8]) {
  u32x4_t y[8];
#pragma unroll
  for (int r = 0; r < 8; ++r)
#pragma unroll
    for (int c = 0; c < 4; ++c)
      y[r][c] = __builtin_amdgcn_perm(x[2 * c + 1][r >> 1], x[2 * c][r >> 1], r & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
  for (int r = 0; r < 8; ++r) x[r] = y[r];
}

// Token number i (0 .. 7) of a lane's 8 of a block of 32.
__device__ __forceinline__ int block_token(int g, int i) { return 16 * (i >> 2) + 4 * g + (i & 3); }

// 8 dims (from 8 s) of 8 tokens (group g of the block of 32 from t0 on) of one head's values.
template <int D>
__device__ __forceinline__ void append_values(const PagedAppendArgs& a, int b, int64_t t0, int head, int s, int g) {
  constexpr int PER = D / 16;
  const int n = live_rows(a.lengths, b, a.rows);
  const int64_t pos = a.positions[b];
  if (n <= 0 || t0 >= pos + n || t0 + 32 <= pos) return;
  uint16_t* y = head_at(a.cache, a.pages, b, t0, head);
  if (!y) return;
  y += int64_t(a.cache.page_size) * D + paged_v_at(int(t0) & (a.cache.page_size - 1), 0, D) + 128 * g;
  const uint16_t* x = a.v.at + b * a.v.batch + head * a.v.head + 8 * s;
  u32x4_t v[8];
  bool all = true, live[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = t0 + block_token(g, i) - pos;
    live[i] = row >= 0 && row < n;
    all = all && live[i];
    v[i] = __builtin_bit_cast(u32x4_t, load_half8(x + min(max(row, int64_t(0)), int64_t(n - 1)) * a.v.row));
  }
  if (all) {
    transpose8(v);
#pragma unroll
    for (int e = 0; e < 8; ++e) *reinterpret_cast<u32x4_t*>(y + (8 * s + e) % PER * 512 + (8 * s + e) / PER * 8) = v[e];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (!live[i]) continue;
#pragma unroll
      for (int e = 0; e < 8; ++e) y[(8 * s + e) % PER * 512 + (8 * s + e) / PER * 8 + i] = uint16_t(v[i][e >> 1] >> (16 * (e & 1)));
    }
  }
}

// Many rows.  A workgroup takes the tokens [t0, t0 + RANGE), t0 a multiple of 32, of `chunk`
// heads (of the values: v_chunk).  Grid: (chunks of q, k and v, ranges, batch).
template <int D>
struct Range {
  static constexpr int LANES = D / 16, RANGE = 256 / LANES;                // 64 or 32 tokens
  static constexpr int BLOCKS = RANGE / 32, HEADS = 256 / (D / 2) / BLOCKS;  // of values: heads at a time
};
template <int D, int HC>
__global__ __launch_bounds__(256) void append_range_kernel(PagedAppendArgs a, int q_chunks, int k_chunks, int chunk, int v_chunk) {
  using R = Range<D>;
  const int b = int(blockIdx.z), tid = int(threadIdx.x);
  const int64_t pos = a.positions[b], t0 = (pos & ~int64_t(31)) + int64_t(blockIdx.y) * R::RANGE;
  if (t0 >= pos + a.rows) return;
  int c = int(blockIdx.x);
  if (c < q_chunks + k_chunks) {
    const bool keys = c >= q_chunks;
    if (keys) c -= q_chunks;
    const int64_t row = t0 + tid / R::LANES - pos;
    if (row < 0 || row >= a.rows) return;
    append_turned<D, HC>(a, keys, b, int(row), tid % R::LANES, c * chunk, min(keys ? a.cache.kv_heads : a.heads, (c + 1) * chunk));
    return;
  }
  c -= q_chunks + k_chunks;
  const int lane = tid % (D / 2), block = tid / (D / 2) % R::BLOCKS;
  for (int h = c * v_chunk + tid / (D / 2) / R::BLOCKS; h < min(a.cache.kv_heads, (c + 1) * v_chunk); h += R::HEADS)
    append_values<D>(a, b, t0 + 32 * block, h, lane % (D / 8), lane / (D / 8));
}

// A few rows (single tokens): a lane has 16 values of a query or key, or 8 of a value, which it
// stores one by one.  Grid: (lanes, batch).
template <int D>
__global__ __launch_bounds__(256) void append_few_kernel(PagedAppendArgs a) {
  constexpr unsigned UNITS = D / 16, PIECES = D / 8;
  constexpr int PER = D / 16;
  const unsigned rows = unsigned(a.rows), turned = unsigned(a.heads + a.cache.kv_heads) * rows * UNITS;
  unsigned at = blockIdx.x * 256 + threadIdx.x;
  const int b = int(blockIdx.y);
  if (at < turned) {
    const unsigned u = at % UNITS, hr = at / UNITS, head = hr / rows;
    const bool keys = int(head) >= a.heads;
    const int h = int(head) - (keys ? a.heads : 0);
    append_turned<D, 1>(a, keys, b, int(hr % rows), int(u), h, h + 1);
    return;
  }
  at -= turned;
  const int s = int(at % PIECES);
  const unsigned hr = at / PIECES;
  const int head = int(hr / rows), row = int(hr % rows);
  if (head >= a.cache.kv_heads || row >= live_rows(a.lengths, b, a.rows)) return;
  const int64_t t = int64_t(a.positions[b]) + row;
  uint16_t* y = head_at(a.cache, a.pages, b, t, head);
  if (!y) return;
  const u16x8_t v = __builtin_bit_cast(u16x8_t, load_half8(a.v.at + b * a.v.batch + head * a.v.head + row * a.v.row + 8 * s));
  y += int64_t(a.cache.page_size) * D + paged_v_at(int(t) & (a.cache.page_size - 1), 0, D);
#pragma unroll
  for (int e = 0; e < 8; ++e) y[(8 * s + e) % PER * 512 + (8 * s + e) / PER * 8] = v[e];
}

// Rows back: a lane takes 8 dims of a token's key and turns 8 dims of 8 tokens' values
// around.  Grid: (blocks of 32 tokens, head groups, batch).
template <int D>
__global__ __launch_bounds__(256) void read_kernel(PagedReadArgs a) {
  constexpr int LPB = D / 2, HEADS = 256 / LPB, PIECES = D / 8, PER = D / 16;
  const int b = int(blockIdx.z), lane = int(threadIdx.x) % LPB, s = lane % PIECES, g = lane / PIECES;
  const int head = int(blockIdx.y) * HEADS + int(threadIdx.x) / LPB;
  const int64_t pos = a.positions[b], t0 = ((pos >> 5) + blockIdx.x) << 5;
  if (head >= a.cache.kv_heads || t0 >= pos + a.rows) return;
  const uint16_t* x = t0 < pos + live_rows(a.lengths, b, a.rows) ? head_at(a.cache, a.pages, b, t0, head) : nullptr;
  const int n = x ? live_rows(a.lengths, b, a.rows) : 0, first = int(t0) & (a.cache.page_size - 1);
  const int64_t out = (int64_t(b) * a.cache.kv_heads + head) * a.rows;
  u32x4_t k[8] = {}, v[8] = {};
  if (x) {
    const uint16_t* xv = x + int64_t(a.cache.page_size) * D + paged_v_at(first, 0, D) + 128 * g;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int dim = 8 * s + i;
      k[i] = *reinterpret_cast<const u32x4_t*>(x + paged_k_at(first + block_token(g, i), 8 * s, D));
      v[i] = *reinterpret_cast<const u32x4_t*>(xv + dim % PER * 512 + dim / PER * 8);
    }
    transpose8(v);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = t0 + block_token(g, i) - pos;
    if (row < 0 || row >= a.rows) continue;
    const bool live = row < n;
    store_half8(a.k + (out + row) * D + 8 * s, live ? __builtin_bit_cast(half8_t, k[i]) : half8_t{});
    store_half8(a.v + (out + row) * D + 8 * s, live ? __builtin_bit_cast(half8_t, v[i]) : half8_t{});
  }
}

// Blocks of 32 tokens that `rows` rows from any position on can touch.
unsigned blocks_of(int rows) { return unsigned((int64_t(rows) + 30) / 32 + 1); }

// Whether a row's lanes lie side by side, values stored one by one, in place of whole records:
// few rows to a request leave most of a range idle, and few rows in all are done sooner by more
// lanes.  One by one against ranges, us, with queries: 32 requests of 25 heads of 64, 4 / 16 / 64
// rows 5.4 / 7.2 / 13.8 and 7.8 / 14.9 / 21.3; 64 of 32 over 8 of 128, 5.5 / 10 / 25.2 and 8.4 /
// 15.5 / 25.7; one of 12 heads, 1000 rows 5.8 and 6.1; 8 of 12, 200 / 400 / 1000 rows 8.0 / 12.2 /
// 20.1 and 9.0 / 11.5 / 18.7; 16 of 32 over 8, 128 / 200 / 1000 14.5 / 19.2 / 93 and 15.3 /
// 18.4 / 83.
bool one_by_one(const PagedAppendArgs& a) { return a.rows <= 64 || int64_t(a.batch) * a.rows <= 2048; }

template <int D>
hipError_t append(const PagedAppendArgs& a, hipStream_t stream) {
  using R = Range<D>;
  const int q_heads = a.heads, kv_heads = a.cache.kv_heads;
  if (one_by_one(a)) {
    const int64_t lanes = int64_t(a.rows) * ((q_heads + kv_heads) * (D / 16) + kv_heads * (D / 8));
    hipLaunchKernelGGL((append_few_kernel<D>), dim3(unsigned((lanes + 255) / 256), unsigned(a.batch)), dim3(256), 0, stream, a);
    return hipGetLastError();
  }
  // (From any position on, rows touch one range more than they fill, or two.)
  const int64_t ranges = (int64_t(a.rows) + 30) / R::RANGE + 1;
  const auto chunks = [](int heads, int chunk) { return (heads + chunk - 1) / chunk; };
  const int v_chunk = R::HEADS, v_chunks = chunks(kv_heads, v_chunk);
  // Heads that share a lane's angles: 4, or fewer where that leaves fewer than 1024 workgroups.
  int chunk = 4;
  while (chunk > 1 && ranges * a.batch * (chunks(q_heads, chunk) + chunks(kv_heads, chunk) + v_chunks) < 1024) chunk /= 2;
  const int q_chunks = chunks(q_heads, chunk), k_chunks = chunks(kv_heads, chunk);
  const dim3 grid(unsigned(q_chunks + k_chunks + v_chunks), unsigned(ranges), unsigned(a.batch));
  const auto kernel = chunk == 1 ? append_range_kernel<D, 1> : chunk == 2 ? append_range_kernel<D, 2> : append_range_kernel<D, 4>;
  hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, a, q_chunks, k_chunks, chunk, v_chunk);
  return hipGetLastError();
}

}  // namespace

hipError_t paged_append(const PagedAppendArgs& a, hipStream_t stream) {
  return a.cache.head_dim == 64 ? append<64>(a, stream) : append<128>(a, stream);
}

hipError_t paged_read(const PagedReadArgs& a, hipStream_t stream) {
  const int heads = 512 / a.cache.head_dim;
  const dim3 grid(blocks_of(a.rows), unsigned((a.cache.kv_heads + heads - 1) / heads), unsigned(a.batch));
  if (a.cache.head_dim == 64) hipLaunchKernelGGL((read_kernel<64>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((read_kernel<128>), grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace tia
