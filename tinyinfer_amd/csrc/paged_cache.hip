// The paged fp16 KV cache: rows join it, keys turned by their positions on the way, and
// are read back.  Layout in paged_cache.hpp, angles in rotary.hpp.
//
// Keys (and queries, into their own output) are taken 16 values to a lane, which walks
// over heads with one set of cosines and sines.  Values are taken 8 dims by 8 tokens to a
// lane: eight loads of 16 bytes, an 8 x 8 turn in registers (32 byte permutations, the rest
// of it is naming), eight stores of 16 bytes that with the neighbouring lanes' fill whole
// records.  Tokens that are not the call's own keep what they hold: a lane whose 8 are not
// all to be written stores single values.
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

// Queries and keys, 16 values to a lane.  Grid: (rows x D / 16, chunks of heads, batch); a
// chunk holds query heads or key heads.
template <int D>
__global__ __launch_bounds__(256) void append_turned_kernel(PagedAppendArgs a, int q_chunks, int chunk) {
  constexpr unsigned units = D / 16;
  const unsigned at = blockIdx.x * 256 + threadIdx.x;
  const int b = int(blockIdx.z), row = int(at / units), u = int(at % units);
  if (row >= a.rows) return;
  const bool keys = int(blockIdx.y) >= q_chunks;
  const int heads = keys ? a.cache.kv_heads : a.heads;
  const int h0 = (int(blockIdx.y) - (keys ? q_chunks : 0)) * chunk, h1 = min(heads, h0 + chunk);
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
  if (!unit.turned) {
#pragma unroll 4
    for (int h = h0; h < h1; ++h) {
      store_half8(y + h * step, load_half8(x + h * from.head + unit.first));
      store_half8(y + h * step + second, load_half8(x + h * from.head + unit.second));
    }
    return;
  }
  const Turns turns(a.rotary, u, t);
#pragma unroll 4
  for (int h = h0; h < h1; ++h) {
    half8_t p = load_half8(x + h * from.head + unit.first), q = load_half8(x + h * from.head + unit.second);
    turn_unit(turns, a.rotary.interleaved, p, q);
    store_half8(y + h * step, p);
    store_half8(y + h * step + second, q);
  }
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

// Values: D / 2 lanes to a head's block of 32 tokens.  Grid: (blocks, head groups, batch).
template <int D>
__global__ __launch_bounds__(256) void append_values_kernel(PagedAppendArgs a) {
  constexpr int LPB = D / 2, HEADS = 256 / LPB, PIECES = D / 8, PER = D / 16;
  const int b = int(blockIdx.z), lane = int(threadIdx.x) % LPB, s = lane % PIECES, g = lane / PIECES;
  const int head = int(blockIdx.y) * HEADS + int(threadIdx.x) / LPB;
  const int n = live_rows(a.lengths, b, a.rows);
  const int64_t pos = a.positions[b], t0 = ((pos >> 5) + blockIdx.x) << 5;
  if (head >= a.cache.kv_heads || n <= 0 || t0 >= pos + n) return;
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
  if (all) transpose8(v);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int dim = 8 * s + e;
    if (all) {
      *reinterpret_cast<u32x4_t*>(y + dim % PER * 512 + dim / PER * 8) = v[e];
    } else {
      // (Value e of token i.)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (live[i]) y[dim % PER * 512 + dim / PER * 8 + i] = uint16_t(v[i][e >> 1] >> (16 * (e & 1)));
    }
  }
}

// A few rows (single tokens): 8 dims of one row to a lane, stored one by one.
template <int D>
__global__ __launch_bounds__(256) void append_value_rows_kernel(PagedAppendArgs a) {
  constexpr unsigned PIECES = D / 8;
  constexpr int PER = D / 16;
  const unsigned at = blockIdx.x * 256 + threadIdx.x;
  const int b = int(blockIdx.y), s = int(at % PIECES);
  const unsigned hr = at / PIECES;
  const int head = int(hr / unsigned(a.rows)), row = int(hr % unsigned(a.rows));
  if (head >= a.cache.kv_heads || row >= live_rows(a.lengths, b, a.rows)) return;
  const int64_t t = int64_t(a.positions[b]) + row;
  uint16_t* y = head_at(a.cache, a.pages, b, t, head);
  if (!y) return;
  const u16x8_t v = __builtin_bit_cast(u16x8_t, load_half8(a.v.at + b * a.v.batch + head * a.v.head + row * a.v.row + 8 * s));
  y += int64_t(a.cache.page_size) * D + paged_v_at(int(t) & (a.cache.page_size - 1), 0, D);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int dim = 8 * s + e;
    y[dim % PER * 512 + dim / PER * 8] = v[e];
  }
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

constexpr int kValueRowsMax = 8;

template <int D>
hipError_t append(const PagedAppendArgs& a, hipStream_t stream) {
  constexpr int HEADS = 512 / D;
  const int64_t groups = (int64_t(a.rows) * (D / 16) + 255) / 256;
  const int q_heads = a.q.at ? a.heads : 0, kv_heads = a.cache.kv_heads;
  int chunk = q_heads > kv_heads ? q_heads : kv_heads;
  while (chunk > 1 && groups * a.batch * ((q_heads + chunk - 1) / chunk + (kv_heads + chunk - 1) / chunk) < 1024) chunk = (chunk + 1) / 2;
  const int q_chunks = (q_heads + chunk - 1) / chunk, k_chunks = (kv_heads + chunk - 1) / chunk;
  hipLaunchKernelGGL((append_turned_kernel<D>), dim3(unsigned(groups), unsigned(q_chunks + k_chunks), unsigned(a.batch)), dim3(256), 0,
                     stream, a, q_chunks, chunk);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (a.rows <= kValueRowsMax) {
    const int64_t lanes = int64_t(kv_heads) * a.rows * (D / 8);
    hipLaunchKernelGGL((append_value_rows_kernel<D>), dim3(unsigned((lanes + 255) / 256), unsigned(a.batch)), dim3(256), 0, stream, a);
  } else {
    hipLaunchKernelGGL((append_values_kernel<D>), dim3(blocks_of(a.rows), unsigned((kv_heads + HEADS - 1) / HEADS), unsigned(a.batch)),
                       dim3(256), 0, stream, a);
  }
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
