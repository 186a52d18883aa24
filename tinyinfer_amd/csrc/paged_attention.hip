// Attention over the paged fp16 KV cache for gfx950: single tokens and prompts.
//
//   o[r] = sum_j p_rj V_j / sum_j p_rj,  p_rj = 2^(x_rj - m_r),  x_rj = (q_r . K_j) D^-1/2 log2 e
//
// in one pass over the keys with a running reference m_r.  A query row is (request,
// query, query head of the key head's group): the rows of a group share their keys, so they
// fill the 16 columns of a matrix operand.  Per tile of 64 keys a wave computes, for each
// of its QB blocks of 16 rows,
//   S^T = K Q^T   v_mfma_f32_16x16x32_f16: A = 16 keys x 32 dims of K, B = Q^T;
//                 lane (j, g) receives the scores of row j for keys 4g .. 4g + 3
//                 of each 16;
//   P^T           two 16-key blocks of it side by side are the B operand of
//   O^T += V^T P^T with A = 16 dims x 32 keys of V^T.
// The cache holds K and V in these operands' order (paged_cache.hpp), so both come straight
// from memory into registers, 16 bytes per lane, and nothing moves between lanes or through
// LDS but the running maximum, when it rises.
//
// Pages: a tile is two halves of 32 tokens, each on one page.  A wave reads the page numbers
// of its next 64 tiles at once, one per lane, and broadcasts one per half: no load waits for
// a table.  A half on no page of the cache is masked like keys past the end.
//
// What memory holds in masked places is anybody's, an infinity or NaN too, and 0 times that
// is NaN: a tile in which something is masked is searched for such values, and if it has one
// they count as some number, times a weight of 0, and a product of ones, over the keys that a
// row sees, says which sums must be NaN all the same.
//
// What bounds it.  Single tokens: memory where caches are long (16 requests of 8 x 128, 12000
// to 32768 keys: 248 us, 6.3 TB/s), launch and one tile's chain of latencies where they are
// short (one request of 12 heads, 300 keys: 6.0 us; 32 of them, 128 to 1024 keys: 14 us, 5.6 of
// them without keys).  Prompts: a tile of 64 keys x 32 rows at D 128 is 68 matrix instructions, 1088
// cycles of a SIMD, about 105 vector instructions and 32 exponentials, 700 cycles, and 32 KB
// from LDS, 128 of the CU's cycles and 512 for four waves; two workgroups a CU overlap these in part.  2
// requests of 777 queries, 32 heads over 8 of 128, 4500 to 6001 keys: 165 us, 817 TFLOP/s (400
// workgroups on 256 CUs); 2 of 1024 over 5120 159 us, 973 TFLOP/s, 86 % of what a large library
// product reaches; 4 prompts of 1024, 25 heads of 64: 28 us, 480 TFLOP/s; prompts on their own last as long
// as their longest block's chain of tiles (one of 1000, 32 heads over 8 of 128: 27 us, 306).  Left out (wrong values), 166
// us becomes: the exponentials 158, the maximum 164, the loads 155, the second product 122.  One row
// block's products stand beside the other's exponentials (172 with both blocks in step).  Tried for the
// shared tiles and no faster: the next tile's scores under this one's weights (192 us for 179 then),
// eight waves of which four multiply while four work out weights (169, but 46 for 30 at D 64), operands
// read from LDS 4 to 16 ahead by hand (181), the loads spread over the tile (165 to 171), wave
// priorities (167).
#include <algorithm>

#include "divisor.hpp"
#include "lds_limit.hpp"
#include "paged_cache.hpp"

namespace tia {
namespace {

constexpr int kTile = 64;   // keys per wave and step
constexpr float kNegInf = -__builtin_huge_valf();
// The reference of a row's exponents: 6 below its largest x when set, raised when one is
// more than 14 above it.  Weights then lie around 2^6 and below 2^15: rounded to fp16, whose
// smallest normal number is 2^-14, a weight 2^-20 times the heaviest still keeps 11 bits.
// A weight's exponent is one fused multiply-add of a score and the reference, which was set from
// a rounded product: the two are apart by up to 1.5 half steps of x, a factor that all weights
// share and that cancels, but not out of fp16's range.  From a reference of 2^22 on, steps of
// half a unit, it is the rounded product less the reference: a number of at most 14, exactly.
constexpr float kBelow = 6.f, kRaise = 14.f, kFar = 4194304.f;

struct AttnPlan {
  PagedAttnArgs a;
  float scale;             // D^-1/2 log2 e
  int page_shift;          // log2(page_size / 32)
  Divisor group, rows;     // query heads per key head; rows of one request and key head
  Divisor heads, pairs;    // key heads; (request, key head) pairs
  Divisor row_block_div;   // row blocks of a pair
  int splits;              // of a request's keys
  int tail;                // kMixed: row blocks of a pair, from the first on, that are walked two by two
  int64_t workgroups;
  int64_t all_rows;        // batch * heads * q_len
};

typedef unsigned short u16x8_t __attribute__((ext_vector_type(8)));
typedef unsigned long long u64;

typedef __attribute__((address_space(1))) void* global_ptr;
typedef __attribute__((address_space(3))) void* lds_ptr;

template <bool NT>
__device__ __forceinline__ half8_t load16(const uint16_t* p) {
  if constexpr (NT) return __builtin_bit_cast(half8_t, __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(p)));
  return *reinterpret_cast<const half8_t*>(p);
}

// The largest |x| bits of 8 values, with `top`.
__device__ __forceinline__ u16x8_t top_bits(u16x8_t top, half8_t x) {
  return __builtin_elementwise_max(top, __builtin_bit_cast(u16x8_t, x) & uint16_t(0x7fff));
}
__device__ __forceinline__ bool any_not_finite(u16x8_t top) {
  bool inside = true;
#pragma unroll
  for (int e = 0; e < 8; ++e) inside = inside && top[e] < 0x7c00;
  return !inside;
}

// The output of weighted values o of `total` probability (inv: its reciprocal).  It lies
// between values, of at most 65504: what the rounded weights of finite ones sum up to beyond
// is cut off.
__device__ __forceinline__ half4_t output_of(float4_t o, float total, float inv) {
  constexpr float most = 65504.f;
  float x[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = total == 0.f ? 0.f : o[e] * inv;
  if (__ballot(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))) > most)) {
#pragma unroll
    for (int e = 0; e < 4; ++e)  // (infinities and NaN stay)
      x[e] = fabsf(x[e]) == -kNegInf ? x[e] : x[e] > most ? most : x[e] < -most ? -most : x[e];
  }
  return half4_t{f16r(x[0]), f16r(x[1]), f16r(x[2]), f16r(x[3])};
}

// x y, rounded: a difference behind it is not made one operation with it.
__device__ __forceinline__ float rounded_product(float x, float y) {
  float z = x * y;
  asm("" : "+v"(z));
  return z;
}

// A wave's rows, QB blocks of 16, lane (j, g) holding its part of row j of each: what they
// ask, see and have summed up.
template <int D, int QB>
struct Rows {
  static constexpr int PER = D / 16, ROWS = 16 * QB;
  // One block of rows (always where a key head has 16 rows or fewer, as of single tokens): a second
  // product with what the weights' rounding to fp16 leaves out costs nothing that shows, so the
  // result is as near as fp32 weights would bring it.  Two blocks (prompts, and single tokens of more
  // heads where a call is large: 32 requests of 32 heads over one, 9000 keys 36.7 us, one block 37.8;
  // 64 over 16384 100 and 113) take the rounded weights alone, a third less matrix work, and sum up
  // these too: by one more product, with ones, in place of 32 additions.  (Twice rounded the chunk
  // above takes 235 us in place of 167, and its error against 64 bits is 2.1e-4 in place of 2.9e-4,
  // most of both the result's own rounding.)
  static constexpr bool FINE = QB == 1;

  const AttnPlan& p;
  int lane, j, g, b, head, kv, ql;
  int64_t off;
  int row_id[QB];  // in q's order, -1 past the last row
  int end[QB];     // keys [0, end) are visible
  int last, first; // keys that some row of the wave sees, and that every row with a query sees
  half8_t qf[QB][D / 32];
  float m[QB];
  float4_t l[QB];  // FINE: [0] is this lane's part of the sum; else all are the row's sum
  float4_t acc[QB][PER];
  u64 far[QB];     // which lanes' references are far from 0 (the same in all of them)
  unsigned spoilt[QB];  // bit 4 d + e: the sum acc[u][d][e] is over an infinity or NaN that is not in it
  half8_t pp[QB][2], rest[2];

  // Keys that query qi sees, and keys that some of `rows` rows from `from` on see.
  __device__ __forceinline__ int seen(int qi) const {
    return int(max(p.a.causal ? min(int64_t(kv), off + qi + 1) : int64_t(kv), int64_t(0)));
  }
  __device__ __forceinline__ int last_of(int from, int rows) const {
    const int count = int(p.rows.d), q_last = min(div_by(min(from + rows, count) - 1, p.group), ql - 1);
    return from >= count || q_last < div_by(from, p.group) ? 0 : seen(q_last);
  }
  __device__ __forceinline__ int first_of(int from) const { return seen(div_by(min(from, int(p.rows.d) - 1), p.group)); }

  __device__ __forceinline__ Rows(const AttnPlan& plan, int request, int kv_head, int r0)
      : p(plan), lane(int(threadIdx.x & 63)), j(lane & 15), g(lane >> 4), b(request), head(kv_head) {
    const PagedAttnArgs& a = p.a;
    kv = int(min(int64_t(max(a.kv_lengths[b], 0)), int64_t(a.pages.width) * a.cache.page_size));
    ql = a.q_lengths ? min(max(a.q_lengths[b], 0), a.q_len) : a.q_len;
    off = int64_t(a.offsets ? a.offsets[b] : a.kv_lengths[b]) - (a.offsets ? 0 : ql);
    const int count = int(p.rows.d), group = int(p.group.d);
#pragma unroll
    for (int u = 0; u < QB; ++u) {
      const int r = r0 + 16 * u + j, rc = min(r, count - 1), qi = div_by(rc, p.group);
      row_id[u] = r < count ? (b * a.heads + head * group + rc - qi * group) * a.q_len + qi : -1;
      end[u] = r < count && qi < ql ? seen(qi) : 0;
    }
    last = last_of(r0, ROWS);
    // (A row without a query may compute anything: it is cleared at the end.)
    first = last == 0 ? 0 : first_of(r0);
  }
  __device__ __forceinline__ void load() {
#pragma unroll
    for (int u = 0; u < QB; ++u) {
      u16x8_t top = {};
      const uint16_t* qp = p.a.q + int64_t(max(row_id[u], 0)) * D + 8 * g;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        half8_t x;
        __builtin_memcpy(&x, qp + 32 * c, 16);
        top = top_bits(top, x);
        qf[u][c] = end[u] > 0 ? x : half8_t{};
      }
      // A row's sum starts at NaN if its query has an infinity or NaN: its scores are infinite, of
      // either sign, or NaN (and all of -inf would pass for a row without a key).
      const float start = __ballot(any_not_finite(top)) >> j & 0x0001000100010001u ? __builtin_nanf("") : 0.f;
      l[u] = float4_t{start, start, start, start};
      m[u] = kNegInf;
      far[u] = 0;
      spoilt[u] = 0;
#pragma unroll
      for (int d = 0; d < PER; ++d) acc[u][d] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
  }

  // Key 16 kb + v of this lane, of tile t, is visible to row (u, j) iff it is below its half's limit.
  __device__ __forceinline__ bool sees(int u, int t, bool held0, bool held1, int kb, int v) const {
    return 16 * kb + v < ((kb < 2 ? held0 : held1) ? end[u] - t * kTile - 4 * g : 0);
  }
  __device__ __forceinline__ bool full(int t, bool held0, bool held1) const { return (t + 1) * kTile <= first && held0 && held1; }

  // Scores of block u, key(kb, c) being the operand of 16 keys x 32 dims.
  template <typename K>
  __device__ __forceinline__ void score(int u, float4_t (&sc)[QB][4], K key) const {
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
      sc[u][kb] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < D / 32; ++c) sc[u][kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(key(kb, c), qf[u][c], sc[u][kb], 0, 0, 0);
    }
  }
  // Masks the scores of block u and raises its reference where it must be.  (Scores far from 0 are
  // scaled here; one branch for both, taken rarely.)
  __device__ __forceinline__ void refer(int u, float4_t (&sc)[QB][4], int t, bool held0, bool held1) {
    if (!full(t, held0, held1)) {
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int v = 0; v < 4; ++v) sc[u][kb][v] = sees(u, t, held0, held1, kb, v) ? sc[u][kb][v] : kNegInf;
    }
    float high = kNegInf;
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int v = 0; v < 4; ++v) high = fmaxf(high, sc[u][kb][v]);
    if (__builtin_expect((__ballot(fmaf(high, p.scale, -m[u]) > kRaise) | far[u]) != 0, 0)) {
      high = rounded_product(high, p.scale);
      high = fmaxf(high, __shfl_xor(high, 16, 64));
      high = fmaxf(high, __shfl_xor(high, 32, 64));
      const float nm = high - m[u] > kRaise ? high - kBelow : m[u];
      const float f = m[u] == kNegInf ? 0.f : __builtin_amdgcn_exp2f(m[u] - nm);
      l[u] *= f;
#pragma unroll
      for (int d = 0; d < PER; ++d) acc[u][d] *= f;
      m[u] = nm;
      far[u] = __ballot(fabsf(nm) >= kFar && fabsf(nm) < -kNegInf);
      if (far[u]) {
#pragma unroll
        for (int kb = 0; kb < 4; ++kb)
#pragma unroll
          for (int v = 0; v < 4; ++v) sc[u][kb][v] = rounded_product(sc[u][kb][v], p.scale);
      }
    }
  }
  // Its weights.
  __device__ __forceinline__ void weigh(int u, const float4_t (&sc)[QB][4]) {
    const float ref = m[u] == kNegInf ? 0.f : -m[u];  // -inf while every key so far is masked
    const float scale = far[u] ? 1.f : p.scale;
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float w = __builtin_amdgcn_exp2f(fmaf(sc[u][kb][v], scale, ref));
        pp[u][kb >> 1][4 * (kb & 1) + v] = f16(w);
        if constexpr (FINE) {
          l[u][0] += w;
          rest[kb >> 1][4 * (kb & 1) + v] = f16(w - float(f16(w)));
        }
      }
  }
  // Adds the tile's values to block u, value(d, h) being the operand of 16 dims x 32 keys.
  template <typename V>
  __device__ __forceinline__ void product(int u, V value) {
    if constexpr (!FINE) {
      const f16 one = f16(1.f);
      const half8_t ones = {one, one, one, one, one, one, one, one};
#pragma unroll
      for (int h = 0; h < 2; ++h) l[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pp[u][h], l[u], 0, 0, 0);
    }
#pragma unroll
    for (int d = 0; d < PER; ++d)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const half8_t vf = value(d, h);
        acc[u][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pp[u][h], acc[u][d], 0, 0, 0);
        if constexpr (FINE) acc[u][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, rest[h], acc[u][d], 0, 0, 0);
      }
  }
  // Of a tile of which a row may not see everything: whether it has an infinity or NaN, and the
  // sums that must be NaN for one that their row sees.
  template <typename V>
  __device__ __forceinline__ bool any_odd(V value) const {
    u16x8_t top = {};
#pragma unroll
    for (int d = 0; d < PER; ++d) top = top_bits(top_bits(top, value(d, 0)), value(d, 1));
    return __ballot(any_not_finite(top)) != 0;
  }
  template <typename V>
  __device__ __forceinline__ void spoil(int t, bool held0, bool held1, V value) {
    half8_t seen_ones[QB][2];
#pragma unroll
    for (int u = 0; u < QB; ++u)
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int v = 0; v < 4; ++v) seen_ones[u][kb >> 1][4 * (kb & 1) + v] = sees(u, t, held0, held1, kb, v) ? f16(1.f) : f16(0.f);
    // (Rolled, and the values read once more: this is rare, and registers are not.)
#pragma unroll 1
    for (int d = 0; d < PER; ++d) {
      float4_t hits[QB];
#pragma unroll
      for (int u = 0; u < QB; ++u) hits[u] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const half8_t x = value(d, h);
        half8_t bad;
#pragma unroll
        for (int e = 0; e < 8; ++e) bad[e] = (__builtin_bit_cast(u16x8_t, x)[e] & 0x7fff) >= 0x7c00 ? f16(1.f) : f16(0.f);
#pragma unroll
        for (int u = 0; u < QB; ++u) hits[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bad, seen_ones[u][h], hits[u], 0, 0, 0);
      }
#pragma unroll
      for (int u = 0; u < QB; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) spoilt[u] |= hits[u][e] > 0.f ? 1u << (4 * d + e) : 0u;
    }
  }
  // The rows' sums of weights in l[u][0], 0 for rows without a key, and of spoilt ones NaN.
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int u = 0; u < QB; ++u) {
      if constexpr (FINE) {
        l[u][0] += __shfl_xor(l[u][0], 16, 64);
        l[u][0] += __shfl_xor(l[u][0], 32, 64);
      }
      if (end[u] == 0) l[u][0] = 0.f;
      if (__ballot(spoilt[u] != 0)) {
#pragma unroll
        for (int d = 0; d < PER; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[u][d][e] = spoilt[u] >> (4 * d + e) & 1 ? __builtin_nanf("") : acc[u][d][e];
      }
    }
  }
  // Of this lane's dims: D / 16 (4 g + v) + 4 c .. + 3.
  __device__ __forceinline__ float4_t piece(int u, int v, int c) const {
    return float4_t{acc[u][4 * c][v], acc[u][4 * c + 1][v], acc[u][4 * c + 2][v], acc[u][4 * c + 3][v]};
  }
  // These of row (u, j), of `total` weight, to the output.
  __device__ __forceinline__ void put(int u, int v, int c, float4_t o, float total) const {
    if (row_id[u] < 0) return;
    const float inv = total == 0.f ? 0.f : 1.f / total;
    const half4_t y = output_of(o, total, inv);
    __builtin_memcpy(p.a.out + int64_t(row_id[u]) * D + PER * (4 * g + v) + 4 * c, &y, 8);
  }
  // To the state of a split, and their exponents' reference.
  __device__ __forceinline__ void keep(int u, int v, int c, int split, float4_t o, float total) const {
    if (row_id[u] < 0 || total == 0.f) return;
    const int64_t at = int64_t(split) * p.all_rows + row_id[u];
    *reinterpret_cast<float4_t*>(p.a.workspace + at * D + PER * (4 * g + v) + 4 * c) = o;
  }
  __device__ __forceinline__ void keep_weight(int u, int split, float top, float total) const {
    if (g != 0 || row_id[u] < 0) return;
    float* ml = p.a.workspace + p.splits * p.all_rows * D + 2 * (int64_t(split) * p.all_rows + row_id[u]);
    ml[0] = top;
    ml[1] = total;
  }
};

__device__ __forceinline__ half8_t finite(half8_t x) {  // an infinity or NaN: some number
  const f16 most = f16(65504.f);
  const half8_t high = {most, most, most, most, most, most, most, most};
  return __builtin_elementwise_max(__builtin_elementwise_min(x, high), -high);
}

// Where a (request, key head)'s tiles lie.  The pages of the halves of the wave's next 64
// tiles, STEP apart, are read at once, one tile to a lane.
template <int D, int STEP>
struct Pages {
  const AttnPlan& p;
  const int32_t* table;
  int head, ids[2], from;

  __device__ __forceinline__ Pages(const AttnPlan& plan, int b, int kv_head)
      : p(plan), table(plan.a.pages.table + int64_t(b) * plan.a.pages.width), head(kv_head) {}
  __device__ __forceinline__ void look_up(int t0) {
    from = t0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int entry = (2 * (t0 + STEP * int(threadIdx.x & 63)) + h) >> p.page_shift;
      const int id = entry < p.a.pages.width ? table[entry] : -1;
      ids[h] = id < p.a.cache.page_count ? id : -1;
    }
  }
  // (Behind these calls tiles in front of t are no longer at hand.)
  __device__ __forceinline__ void reach(int t) {
    if (t - from >= 64 * STEP) look_up(t);
  }
  __device__ __forceinline__ int page(int t, int h) const {
    return __builtin_amdgcn_readlane(h ? ids[1] : ids[0], (t - from) / STEP & 63);
  }
  __device__ __forceinline__ bool held(int t, int h) const { return page(t, h) >= 0; }
  // Tokens 64 t + 32 h .. + 31 of the head on a page (none: the first): the number of their
  // keys' block of 32 x D, and that of their values.
  __device__ __forceinline__ int block(int page, int t, int h) const {
    const int blocks = 1 << p.page_shift;
    return (max(page, 0) * p.a.cache.kv_heads + head) * 2 * blocks + ((2 * t + h) & (blocks - 1));
  }
  __device__ __forceinline__ int values(int block) const { return block + (1 << p.page_shift); }
  __device__ __forceinline__ const uint16_t* at(int block) const { return p.a.cache.pages + int64_t(block) * (32 * D); }
};

// Four waves share a row block, each with its own tiles.  Their states meet in LDS: of lane
// (j, g)'s dims, number v of 4 and b of D / 16 lie next to each other in b.
constexpr int kWaves = 4;
template <int D, int QB>
struct Merge {
  float4_t acc[kWaves][QB][4][D / 64][64];
  float m[kWaves][QB][16], l[kWaves][QB][16];
};
template <int D, int QB>
__device__ __forceinline__ void attend(const AttnPlan& p, uint8_t* lds, int b, int head, int rb, int split) {
  constexpr int PER = D / 16;
  const int lane = int(threadIdx.x & 63), wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
  Pages<D, kWaves> pages(p, b, head);
  if (p.splits == 1) pages.look_up(wave);  // (the lengths are still on their way)
  Rows<D, QB> rows(p, b, head, rb * 16 * QB);
  const int tiles = (rows.last + kTile - 1) / kTile, per = (tiles + p.splits - 1) / p.splits, t_end = min(tiles, (split + 1) * per);
  int t = split * per + wave;

  // One block: memory has no use for the keys again.  The next tile's keys are loaded once the
  // scores have used this one's; two blocks of 128 dims leave no registers for that.
  constexpr bool NT = QB == 1, AHEAD = QB == 1 || D == 64;
  half8_t kr[4][D / 32], vr[PER][2];
  const auto load_k = [&](int tt) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint16_t* at = pages.at(pages.block(pages.page(tt, h), tt, h));
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int c = 0; c < D / 32; ++c) kr[2 * h + kb][c] = load16<NT>(at + 16 * kb * D + 512 * c + uint32_t(8 * lane));
    }
  };
  const auto load_v = [&](int tt) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint16_t* at = pages.at(pages.values(pages.block(pages.page(tt, h), tt, h)));
#pragma unroll
      for (int d = 0; d < PER; ++d) vr[d][h] = load16<NT>(at + 512 * d + uint32_t(8 * lane));
    }
  };
  if (t < t_end) {
    if (p.splits > 1) pages.look_up(t);
    if (AHEAD) load_k(t);
  }
  rows.load();
  for (; t < t_end; t += kWaves) {
    const bool held0 = pages.held(t, 0), held1 = pages.held(t, 1);
    if (!AHEAD) load_k(t);
    else load_v(t);
    __builtin_amdgcn_sched_barrier(0);
    float4_t sc[QB][4];
#pragma unroll
    for (int u = 0; u < QB; ++u) rows.score(u, sc, [&](int kb, int c) { return kr[kb][c]; });
    __builtin_amdgcn_sched_barrier(0);
    if (!AHEAD) load_v(t);
    if (t + kWaves < t_end) {
      pages.reach(t + kWaves);
      if (AHEAD) load_k(t + kWaves);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < QB; ++u) {
      rows.refer(u, sc, t, held0, held1);
      rows.weigh(u, sc);
    }
    const auto value = [&](int d, int h) { return vr[d][h]; };
    if (!rows.full(t, held0, held1) && rows.any_odd(value)) {
      rows.spoil(t, held0, held1, [&](int d, int h) {
        const int page = (h ? held1 : held0) ? pages.table[(2 * t + h) >> p.page_shift] : 0;
        return load16<false>(pages.at(pages.values(pages.block(page, t, h))) + 512 * d + uint32_t(8 * lane));
      });
#pragma unroll
      for (int d = 0; d < PER; ++d)
#pragma unroll
        for (int h = 0; h < 2; ++h) vr[d][h] = finite(vr[d][h]);
    }
#pragma unroll
    for (int u = 0; u < QB; ++u) rows.product(u, value);
  }
  rows.finish();

  auto& mg = *reinterpret_cast<Merge<D, QB>*>(lds);
#pragma unroll
  for (int u = 0; u < QB; ++u) {
#pragma unroll
    for (int v = 0; v < 4; ++v)
#pragma unroll
      for (int c = 0; c < D / 64; ++c) mg.acc[wave][u][v][c][lane] = rows.piece(u, v, c);
    if (rows.g == 0) {
      mg.m[wave][u][rows.j] = rows.m[u];
      mg.l[wave][u][rows.j] = rows.l[u][0];
    }
  }
  __syncthreads();
  // Wave w joins number v = w of the dims.
#pragma unroll
  for (int u = 0; u < QB; ++u) {
    float top = kNegInf, total = 0.f, f[kWaves];
    bool empty[kWaves];  // (what it holds is no row's; a state with keys counts however little it weighs: 0 times NaN is NaN)
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = mg.l[w][u][rows.j] == 0.f ? top : fmaxf(top, mg.m[w][u][rows.j]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float lw = mg.l[w][u][rows.j];
      empty[w] = lw == 0.f;
      f[w] = empty[w] ? 0.f : __builtin_amdgcn_exp2f(mg.m[w][u][rows.j] - top);
      total += lw * f[w];
    }
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float4_t x = mg.acc[w][u][wave][c][lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = empty[w] ? o[e] : fmaf(x[e], f[w], o[e]);
      }
      if (p.splits > 1) rows.keep(u, wave, c, split, o, total);
      else rows.put(u, wave, c, o, total);
    }
    if (p.splits > 1 && wave == 0) rows.keep_weight(u, split, top, total);
  }
}

// Four waves have a pair of row blocks each and share every tile, brought into LDS operand by
// operand, one conflict-free kilobyte each, straight from memory: the next one while all work on
// this one, two buffers and one barrier a tile.
constexpr int kSharers = 4;
template <int D>
struct Tiles {
  half8_t k[2][4 * D / 32][64], v[2][2 * D / 16][64];
};
template <int D>
__device__ __forceinline__ void attend_shared(const AttnPlan& p, uint8_t* lds, int b, int head, int rb) {
  constexpr int QB = 2, PER = D / 16, GROUP = kSharers * 16 * QB, PIECE = D / 32;  // PIECE: records of keys, and of values, that a wave loads
  const int lane = int(threadIdx.x & 63), wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)), half = wave >> 1;
  auto& shared = *reinterpret_cast<Tiles<D>*>(lds);
  Pages<D, 1> pages(p, b, head);
  pages.look_up(0);
  Rows<D, QB> rows(p, b, head, rb * GROUP + wave * 16 * QB);
  const int group_last = rows.last_of(rb * GROUP, GROUP), group_first = rows.first_of(rb * GROUP);
  const int tiles = (group_last + kTile - 1) / kTile;

  // This wave's quarter of a tile's keys or values (records PIECE * wave .. of it, all of them of
  // half `wave / 2`) from their half's block to a buffer.
  const auto bring = [&](int block, half8_t (*to)[64]) {
    const global_ptr from = (global_ptr)(pages.at(block) + (wave & 1) * (PIECE * 512) + uint32_t(8 * lane));
    const lds_ptr in = (lds_ptr)&to[PIECE * wave][0];
    __builtin_amdgcn_global_load_lds(from, in, 16, 0, 0);  // (the offset counts on both sides)
    __builtin_amdgcn_global_load_lds(from, in, 16, 1024, 0);
    if constexpr (PIECE == 4) {
      __builtin_amdgcn_global_load_lds(from, in, 16, 2 * 1024, 0);
      __builtin_amdgcn_global_load_lds(from, in, 16, 3 * 1024, 0);
    }
  };
  int flags = 0;  // two bits for each of tiles t and t + 1: their halves are on a page
  const auto fetch = [&](int tt, int buf) {
    const int block = pages.block(pages.page(tt, half), tt, half);
    bring(block, shared.k[buf]);
    bring(pages.values(block), shared.v[buf]);
    flags |= int(pages.held(tt, 0)) << 2 | int(pages.held(tt, 1)) << 3;
  };
  if (tiles > 0) fetch(0, 0);
  rows.load();
  for (int t = 0, buf = 0; t < tiles; ++t, buf ^= 1) {
    flags >>= 2;
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): what this wave has brought
    lds_barrier();                        // everyone's has landed, and nobody reads the other buffer any more
    if (t + 1 < tiles) {
      pages.reach(t + 1);
      fetch(t + 1, buf ^ 1);
    }
    const auto value = [&](int d, int h) { return shared.v[buf][h * PER + d][lane]; };
    // (The same for all waves: what they find lies in LDS.)
    if (((t + 1) * kTile > group_first || (flags & 3) != 3) && rows.any_odd(value)) {
      rows.spoil(t, flags & 1, flags & 2, value);
      lds_barrier();
#pragma unroll
      for (int i = 0; i < PIECE; ++i) {
        half8_t& x = shared.v[buf][PIECE * wave + i][lane];
        x = finite(x);
      }
      lds_barrier();
    }
    if (t * kTile >= rows.last) continue;
    // One block's matrix instructions stand next to the other one's exponentials; the operands
    // stay in registers from the first block to the second.
    float4_t sc[QB][4];
    half8_t kf[4][D / 32], vf[PER][2];
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int c = 0; c < D / 32; ++c) kf[kb][c] = shared.k[buf][kb * (D / 32) + c][lane];
    const auto key = [&](int kb, int c) { return kf[kb][c]; };
    const auto held_value = [&](int d, int h) { return vf[d][h]; };
    rows.score(0, sc, key);
    rows.refer(0, sc, t, flags & 1, flags & 2);
    __builtin_amdgcn_sched_barrier(0);
    rows.score(1, sc, key);
    rows.weigh(0, sc);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int d = 0; d < PER; ++d)
#pragma unroll
      for (int h = 0; h < 2; ++h) vf[d][h] = value(d, h);
    rows.refer(1, sc, t, flags & 1, flags & 2);
    __builtin_amdgcn_sched_barrier(0);
    rows.product(0, held_value);
    rows.weigh(1, sc);
    __builtin_amdgcn_sched_barrier(0);
    rows.product(1, held_value);
  }
  rows.finish();
#pragma unroll
  for (int u = 0; u < QB; ++u)
#pragma unroll
    for (int v = 0; v < 4; ++v)
#pragma unroll
      for (int c = 0; c < D / 64; ++c) rows.put(u, v, c, rows.piece(u, v, c), rows.l[u][0]);
}

// Waves per SIMD that the registers are budgeted for.  What the compiler takes: 64 dims, one
// block 149 of 168, two 206, shared 154, mixed 207; 128 dims 240, 253, 234 and 256, none spilled.
constexpr int waves_for(int dim, int qb) { return dim == 64 && qb == 1 ? 3 : 2; }

// QB: blocks of 16 rows per wave; kShared: waves that share tiles, kMixed: and for the last
// workgroups ones of two blocks.
constexpr int kShared = 0, kMixed = -1;
static_assert(kSharers == kWaves, "one size of workgroup");
template <int D, int QB>
__global__ __launch_bounds__(64 * kWaves, waves_for(D, QB)) void paged_attention_kernel(AttnPlan p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  // The last row blocks of all (request, key head) pairs first: under the causal mask
  // they are the longest.
  const int id = int(blockIdx.x), block = div_by(id, p.pairs), at = id - block * int(p.pairs.d), b = div_by(at, p.heads);
  const int blocks = int(p.row_block_div.d), head = at - b * int(p.heads.d);
  if constexpr (QB == kMixed) {
    const int behind = block - (blocks - p.tail);
    if (behind < 0) attend_shared<D>(p, lds, b, head, blocks - 1 - block);
    else attend<D, 2>(p, lds, b, head, kSharers * p.tail - 1 - behind, 0);
  } else if constexpr (QB == kShared) {
    attend_shared<D>(p, lds, b, head, blocks - 1 - block);
  } else {
    const int split = div_by(block, p.row_block_div);
    attend<D, QB>(p, lds, b, head, blocks - 1 - (block - split * blocks), split);
  }
}

// W waves of a workgroup of 4 join a row's states: D / 4 lanes a state, 2 or 4 states at a
// time and wave.
template <int D, int W>
__global__ __launch_bounds__(256) void paged_attention_join_kernel(AttnPlan p) {
  constexpr int LPR = D / 4, PARTS = 64 / LPR;
  __shared__ float4_t sums[W][LPR];
  __shared__ float weights[W];
  const int lane = int(threadIdx.x & 63), wave = int(threadIdx.x >> 6) % W, part = lane / LPR, at = 4 * (lane % LPR);
  const int64_t row = int64_t(blockIdx.x) * (4 / W) + int(threadIdx.x >> 6) / W;
  if (row >= p.all_rows) return;  // (a workgroup of one row has it)
  const float* ml = p.a.workspace + p.splits * p.all_rows * D;
  float top = kNegInf;
  for (int s = lane; s < p.splits; s += 64) {
    const float* x = ml + 2 * (s * p.all_rows + row);
    if (x[1] != 0.f) top = fmaxf(top, x[0]);
  }
  top = wave_max(top);
  float total = 0.f;
  float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = wave * PARTS + part; s < p.splits; s += W * PARTS) {
    const float* x = ml + 2 * (s * p.all_rows + row);
    const float lw = x[1], f = lw == 0.f ? 0.f : __builtin_amdgcn_exp2f(x[0] - top);
    // (A state without weight was not written.)
    const float4_t y = *reinterpret_cast<const float4_t*>(p.a.workspace + (s * p.all_rows + row) * D + at);
    total = fmaf(lw, f, total);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = lw == 0.f ? o[e] : fmaf(y[e], f, o[e]);
  }
#pragma unroll
  for (int x = LPR; x < 64; x <<= 1) {
    total += __shfl_xor(total, x, 64);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], x, 64);
  }
  if constexpr (W > 1) {
    if (part == 0) sums[wave][lane % LPR] = o;
    if (lane == 0) weights[wave] = total;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < W; ++w) {
      total += weights[w];
      o += sums[w][lane % LPR];
    }
  }
  if (part != 0) return;
  const float inv = total == 0.f ? 0.f : 1.f / total;
  const half4_t y = output_of(o, total, inv);
  __builtin_memcpy(p.a.out + row * D + at, &y, 8);
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// How a call is walked: `blocks` row blocks of 16 per wave, kShared or kMixed, `splits` workgroups
// to its keys; kMixed: `tail` blocks of 128 rows of every pair by waves of two.
struct Walk {
  int blocks, splits, tail = 0;
};
// From the number of (request, key head) pairs, the rows of one, the tiles of 64 keys of the
// longest, and whether rows see about as many keys (even); us, of the ways that follow.
// Two blocks of 16 rows use every key and value twice.  They pay where one block to a
// workgroup makes many workgroups of many tiles (D 64: 12 pairs of 300 rows over 4096 keys 18.5
// against 22.5, 192 of 40 over 4096 56 and 87; not 48 of 40 over 1024, 9.9 and 8.5, nor 192 of 20
// over 256, 7.3 and 6.9), or at 128 dims, of which a CU holds two, more than one a CU (32 pairs
// of 400 rows over 256 keys 11.7 and 14.1, 128 of 80 over 4096 87 and 164; 8 of 400 over 1024 12.9
// and 10.8, 32 of 32 over 4096 21.5 and 19.9).
// Tiles shared by 128 rows pay from about one such block a CU on: the blocks that are launched, a pair's
// last one as long as a full one however few rows it has (D 64: 75 pairs of 269 rows, 225 blocks, over 269
// keys 12.2 against 18.7; 250 of 66 over 2558 44 and 75; D 128: 144 of 200 over 320 19.7 and 22.2), but of
// pairs with 64 rows and fewer, half a block at most, the part of it that they fill (D 64: 192 of 32 over
// 1024 20 and 13.8, 384 of 40 27 and 32).
// From which number on (shared against two blocks).  Short caches or many pairs, whose keys and values
// waves on their own read more often: 192 (D 128: 24 pairs of 1024 rows over 256 keys 14.7 and 19.6, 16 of
// 1536 over 512 19.0 and 21.3, 192 of 128 over 1024 30.5 and 47; D 64: 100 of 256 over 256 11.8 and 15.9).
// Long ones of few pairs: more (D 128: 16 of 1536 over 2048 45.7 and 40.6, of 1792 46.0 and 47.7; D 64: 16
// of 1536 over 4096 55 and 43, 32 of 1024 61.6 and 53.4, 256 of 128 59 and 151).  And prompts on their own,
// whose longest block is twice the average: a CU works on more than one at a time, and four waves
// that share its keys are through with it sooner (D 128: 8 of 4000 over 1000 28.2 and 27.4, 36 of 1000 over 1000 30.2
// and 35.0, 4 of 8192 over 2048 46.4 and 37.8, 20 of 2048 49.1 and 46.7, 2 of 16384 over 4096 81 and 57; D 64: 24 of
// 1000 21.8 and 17.7, 9 of 4096 63 and 41.6, but 25 of 2048, 400 blocks, 35.4 and 50).
// Mixed: a CU works on two blocks in 1.35 times one's time, so a few more blocks than CUs, or than
// a multiple of them, cost nearly a round.  Up to half a round is done by waves of two blocks
// instead, four workgroups to 128 rows, which spread over all CUs (D 128, 4096 keys, blocks: 288
// 89.7 against 113.6 shared, 384 112 and 123, 528 148 and 198, 800 214 and 247, but 448 133 and
// 130; over 512 keys 320 23 and 27, 384 28.2 and 27.8; 40 pairs of 900 rows, 320 blocks, over 4096 95 and
// 112; D 64: 288 58 and 79, 528 91 and 109, 2080 319 and 324, 3104 479 and 466; 128 pairs of 270 71 and 81).
// At D 128 of few pairs alone (100 of 330 over 4096 keys 154 and 117, 64 of 520 95 and 117).  Blocks of
// uneven rows, a prompt on its own, fill the CUs by themselves (25 heads of 64, 4 of 1024 rows: 33 and 27).
// Splits: a second launch and the states' traffic cost 2 us and more, and 4 us of the
// caller's time, so short caches are not split (12 pairs of 1 row over 1024 keys 8.7 us).
// Longer ones are, into at most one workgroup a CU (12 pairs over 4096 keys 10.1, over 16384
// 15.3; 8 pairs of 4 rows over 32768, D 128, 30) and 64 splits.  Workgroups for more than half of the
// CUs are cut in three where that fills two a CU (D 128: 160 of one token over 8192 to 16384 keys 164
// against 184 whole and 175 in four, 144 of two blocks over 6000 33.6, 39.5 and 39.7), else left whole
// (192 over 4096 to 8192 105 against 112 in two and 115 in three, 240 of two blocks over 6000 40 and 42).
Walk walk_for(int64_t pairs, int rows, int keys, bool even, int dim) {
  constexpr int kCus = 256;
  const int64_t tiles = ceil_div(keys, kTile), ones = pairs * ceil_div(rows, 16);
  Walk w{1, 1};
  if (rows > 16 && (dim == 64 ? ones * tiles > 5000 : ones > 256 || ones * tiles > 8000)) w.blocks = 2;
  const int64_t shared = rows > 64 ? pairs * ceil_div(rows, 32 * kSharers) : ceil_div(pairs * ceil_div(rows, 32), kSharers);
  int64_t least = 192;
  if (!even && tiles >= 16 && pairs <= 64) least = tiles < 32 ? kCus + 1 : 330;
  else if (dim == 64 && tiles >= 32 && pairs < 128) least = kCus + 1;
  else if (dim == 128 && tiles >= 16 && pairs <= 64) least = 224;
  if (w.blocks == 2 && shared >= least) {
    const int64_t more = shared % kCus, tail = ceil_div(more, pairs);
    if (even && (dim == 64 || pairs <= 64) && more > 0 && shared > kCus && shared < 9 * kCus &&
        pairs * tail <= (tiles >= 16 ? kCus / 2 : kCus / 4))
      return {kMixed, 1, int(tail)};
    return {kShared, 1};
  }
  const int64_t wgs = pairs * ceil_div(rows, 16 * w.blocks);
  if (wgs > kCus / 2) w.splits = tiles >= 64 && 3 * wgs <= 2 * kCus ? 3 : 1;
  else if (tiles > (dim == 64 ? 24 : 16)) w.splits = int(std::max<int64_t>(1, std::min<int64_t>({kCus / wgs, tiles / 4, 64})));
  return w;
}

AttnPlan plan_of(const PagedAttnArgs& a, Walk& w) {
  AttnPlan p{};
  p.a = a;
  p.scale = float(1.4426950408889634 / __builtin_sqrt(double(a.cache.head_dim)));
  p.page_shift = __builtin_ctz(unsigned(a.cache.page_size) / 32);
  const int group = a.heads / a.cache.kv_heads, rows = group * a.q_len;
  const int64_t pairs = int64_t(a.batch) * a.cache.kv_heads;
  p.group = divisor(group);
  p.rows = divisor(rows);
  p.heads = divisor(a.cache.kv_heads);
  p.pairs = divisor(uint32_t(pairs));
  p.all_rows = pairs * rows;
  w = walk_for(pairs, rows, a.max_kv, !a.causal || a.max_kv / 2 >= a.q_len, a.cache.head_dim);
  const int64_t blocks = ceil_div(rows, w.blocks <= kShared ? 32 * kSharers : 16 * w.blocks);
  p.row_block_div = divisor(uint32_t(blocks));
  p.workgroups = pairs * (blocks * w.splits + (kSharers - 1) * w.tail);
  p.tail = w.tail;
  p.splits = w.splits;
  return p;
}

template <int D, int QB>
hipError_t launch(const AttnPlan& p, hipStream_t stream) {
  constexpr int tiles = QB <= kShared ? int(sizeof(Tiles<D>)) : 0, merge = QB == kShared ? 0 : int(sizeof(Merge<D, QB == 1 ? 1 : 2>));
  constexpr int bytes = tiles > merge ? tiles : merge;
  if constexpr (bytes > 64 * 1024) {  // (two blocks of 128-dim rows)
    static LdsLimit limit;
    const hipError_t e = limit.raise(reinterpret_cast<const void*>(&paged_attention_kernel<D, QB>), bytes);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((paged_attention_kernel<D, QB>), dim3(unsigned(p.workgroups)), dim3(64 * kWaves), bytes, stream, p);
  hipError_t e = hipGetLastError();
  if (QB <= kShared || e != hipSuccess || p.splits == 1) return e;
  if (p.splits > 16)
    hipLaunchKernelGGL((paged_attention_join_kernel<D, 4>), dim3(unsigned(p.all_rows)), dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((paged_attention_join_kernel<D, 1>), dim3(unsigned(ceil_div(p.all_rows, 4))), dim3(256), 0, stream, p);
  return hipGetLastError();
}

template <int D>
hipError_t launch_walk(const AttnPlan& p, const Walk& w, hipStream_t stream) {
  if (w.blocks == kMixed) return launch<D, kMixed>(p, stream);
  if (w.blocks == kShared) return launch<D, kShared>(p, stream);
  return w.blocks == 1 ? launch<D, 1>(p, stream) : launch<D, 2>(p, stream);
}

}  // namespace

int64_t paged_attention_workspace(const PagedAttnArgs& a) {
  Walk w;
  const AttnPlan p = plan_of(a, w);
  return p.splits > 1 ? int64_t(p.splits) * p.all_rows * (a.cache.head_dim + 2) * 4 : 0;
}

hipError_t paged_attention(const PagedAttnArgs& a, hipStream_t stream) {
  Walk w;
  const AttnPlan p = plan_of(a, w);
  return a.cache.head_dim == 64 ? launch_walk<64>(p, w, stream) : launch_walk<128>(p, w, stream);
}

}  // namespace tia
