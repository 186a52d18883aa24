// Attention over the int8 KV cache for gfx950: single tokens, prompts, and a
// prefix that a batch shares, by one kernel.
//
//   o[r] = sum_j w_rj d_j / sum_j p_rj,  p_rj = 2^(x_rj - m_r),  w_rj = p_rj vs_j,
//   x_rj = (q_r . c_j) * ks_j * D^-1/2 * log2 e,  V_j = vs_j * d_j
// with c, d the whole numbers that the cache holds (exact in fp16) and ks, vs the
// fp32 scales of token j: a key's scale is applied to its score, a value's to its
// probability, so neither c nor d is rounded.  The weights w are, to fp16: the reference m_r
// follows the largest x + log2 vs of the keys that row r sees, not the largest x, so the
// rounding is relative to what the row weighs, whatever values others see.
//
// A query row is (request, query, query head of the key head's group): the rows
// of a group share their keys, so they fill the 16 columns of a matrix operand.
// Per 64 keys a wave computes, for each of its QB blocks of 16 rows,
//   S^T = K Q^T   v_mfma_f32_16x16x32_f16: A = 16 keys x 32 dims of K, B = Q^T;
//                 lane (j, g) receives the scores of row j for keys 4g .. 4g + 3
//                 of each 16;
//   P^T           two 16-key blocks of it side by side are the B operand of
//   O^T += V^T P^T with A = 16 dims x 32 keys of V^T.
// The cache keeps V in that operand's order and K's dims are summed in the order
// in which a lane finds them (16 bytes at a time, q's to match), so both come
// straight from memory into registers, 16 bytes per lane, and nothing moves
// between lanes or through LDS but the running maximum, when it rises.
//
// Waves (walk_for has the rules and both sides' times).  Two or four waves share a row
// block: each takes every second or fourth tile of 64 keys, and their states (m, l, O)
// merge through LDS.  Where row blocks are plenty four waves have one each and share the
// tiles instead: each widens a quarter of the next one into LDS (operand by operand, a
// conflict-free kilobyte) while all work on this one, two buffers and one barrier a tile.
// With few row blocks the keys are cut into splits as well, each split's state goes to the
// caller's workspace and a second kernel joins them.  A prefix is one such set of splits,
// its row blocks running over the whole batch: its keys are read once for all requests (but
// for a few short ones, whose rows walk it in front of their own keys: prefix_inline).
//
// What bounds it.  Single tokens: memory where caches are long (16 requests of 8 x 128,
// 12000 to 32768 keys: 135 us, 6.0 TB/s; the loads are the plain ones of a stream,
// past the caches), launch and one tile's chain of latencies where they are short (one
// request of 12 heads, 300 keys: 6 us).  Prompts: vector instructions beside the matrix
// products.  Of a tile of 64 keys x 32 rows at D 128 the 64 matrix instructions are 1024
// cycles of a SIMD; widening K and V is 192 vector instructions and a score takes 6 and an
// exponential, 1900 cycles together.  2 requests of 777 queries, 32 heads over 8 of 128,
// 4500 to 6001 keys: 197 us, 685 TFLOP/s; 4 prompts of 1024, 25 heads of 64: 31 us, 430
// TFLOP/s, its scores' exponentials and scales more than the products.
#include <algorithm>

#include "common.hpp"
#include "divisor.hpp"
#include "kernels.hpp"
#include "lds_limit.hpp"

namespace tia {
namespace {

constexpr int kTile = 64;   // keys per wave and step
constexpr float kNegInf = -__builtin_huge_valf();
// The reference of a row's exponents: 6 below its largest x + log2 vs when set, raised
// when one is more than 14 above it.  Weights then lie around 2^6 and below 2^14: rounded to
// fp16, whose smallest normal number is 2^-14, a weight 2^-20 times the heaviest
// still keeps 11 bits.  The scale of a row of zeros counts as 2^kLeast, below every
// other (2^-24 / 127 at least): probabilities are fp32 and stay below 2^(14 - kLeast).
constexpr float kBelow = 6.f, kRaise = 14.f, kLeast = -40.f;

struct AttnPlan {
  KvAttnArgs a;
  float scale;                   // D^-1/2 log2 e
  Divisor group, rows;           // query heads per key head; rows of one request and key head
  Divisor heads, pairs;          // key heads; (request, key head) pairs
  Divisor row_block_div, prefix_block_div;  // row blocks of a pair, and of the prefix
  int splits, prefix_splits;     // of the requests' own keys, and of the prefix's
  int64_t own_wgs, prefix_wgs;
  int64_t all_rows;              // batch * heads * q_len
  bool parts;                    // states to the workspace, joined by the second kernel
};

typedef unsigned short u16x8_t __attribute__((ext_vector_type(8)));

// Whole numbers c of 4 stored bytes c + 128, as fp16.
__device__ __forceinline__ void widen4(uint32_t w, half2_t& lo, half2_t& hi) {
  const half2_t bias = {f16(-1152.f), f16(-1152.f)};
  lo = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) + bias;
  hi = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) + bias;
}
__device__ __forceinline__ half8_t widen8(uint32_t w0, uint32_t w1) {
  half2_t a, b, c, d;
  widen4(w0, a, b);
  widen4(w1, c, d);
  return half8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// The same bytes as the whole numbers c + 1152: half the work.
__device__ __forceinline__ half8_t raise8(uint32_t w0, uint32_t w1) {
  const u32x4_t r = {__builtin_amdgcn_perm(0x64646464u, w0, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, w0, 0x04030402u),
                     __builtin_amdgcn_perm(0x64646464u, w1, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, w1, 0x04030402u)};
  return __builtin_bit_cast(half8_t, r);
}

// x times the value that lane N of this lane's row of 16 holds (the broadcast is an
// operand modifier of the multiplication).
template <int N>
__device__ __forceinline__ float mul_row_lane(float x, float of) {
  const float y = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, of), 0x150 + N, 0xF, 0xF, true));
  return x * y;
}
template <int N>
__device__ __forceinline__ float add_row_lane(float x, float of) {
  return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, of), 0x150 + N, 0xF, 0xF, true));
}
// x[kb][v] times lane 4 kb + v's value.
__device__ __forceinline__ void mul_row(float4_t (&x)[4], float of) {
#define TIA_MUL(kb, v) x[kb][v] = mul_row_lane<4 * kb + v>(x[kb][v], of);
#define TIA_MUL4(kb) TIA_MUL(kb, 0) TIA_MUL(kb, 1) TIA_MUL(kb, 2) TIA_MUL(kb, 3)
  TIA_MUL4(0) TIA_MUL4(1) TIA_MUL4(2) TIA_MUL4(3)
#undef TIA_MUL4
#undef TIA_MUL
}

// The largest x[kb][v] + lane 4 kb + v's value.
__device__ __forceinline__ float max_row_sum(const float4_t (&x)[4], float of) {
  float high = kNegInf;
#define TIA_MAX(kb, v) high = fmaxf(high, add_row_lane<4 * kb + v>(x[kb][v], of));
#define TIA_MAX4(kb) TIA_MAX(kb, 0) TIA_MAX(kb, 1) TIA_MAX(kb, 2) TIA_MAX(kb, 3)
  TIA_MAX4(0) TIA_MAX4(1) TIA_MAX4(2) TIA_MAX4(3)
#undef TIA_MAX4
#undef TIA_MAX
  return high;
}

template <bool NT>
__device__ __forceinline__ u32x4_t load16(const uint8_t* p) {
  if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(p));
  return *reinterpret_cast<const u32x4_t*>(p);
}

// The output of weighted values o of `total` probability (inv: its reciprocal).  It lies
// between values, of at most 65504: what the rounded weights sum up to beyond is cut off.
__device__ __forceinline__ half4_t output_of(float4_t o, float total, float inv) {
  constexpr float most = 65504.f;
  float x[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = total == 0.f ? 0.f : o[e] * inv;
  if (__ballot(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))) > most)) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = x[e] > most ? most : x[e] < -most ? -most : x[e];  // (NaN stays)
  }
  return half4_t{f16r(x[0]), f16r(x[1]), f16r(x[2]), f16r(x[3])};
}

template <int D, int QB, int KW>
struct Merge {
  float4_t acc[KW][QB * D / 16][64];
  float m[KW][QB][16], l[KW][QB][16];
};

// A tile's operands as the waves of a workgroup share them, in the order in which a
// lane reads them: 16 bytes per lane, one conflict-free kilobyte per operand.
template <int D>
struct Tiles {
  half8_t k[2][4][D / 32][64], v[2][D / 16][2][64];
};

// Row block `rb` of one set of keys.  kPrefix: rows run over the batch, key head
// `head`, the keys are the prefix's; else over request b's, the keys its own, behind the
// prefix's for kBoth.
// KW waves share the row block, each with its own tiles; kShared: 4 waves have a row
// block each (`rb` counts those groups) and share every tile, each widening a quarter of
// it into LDS while the tile before is worked on.
constexpr int kShared = 0;
enum Keys { kOwn, kPrefix, kBoth };
template <int D, int QB, int KW, Keys KEYS>
__device__ void attend(const AttnPlan& p, uint8_t* lds, int b0, int head, int rb, int split, int splits, int state) {
  constexpr bool PREFIX = KEYS == kPrefix, BOTH = KEYS == kBoth;
  const KvAttnArgs& a = p.a;
  const int lane = int(threadIdx.x & 63), wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
  const int j = lane & 15, g = lane >> 4;
  constexpr int ROWS = 16 * QB, GROUP = KW == kShared ? 4 * ROWS : ROWS;
  const int group0 = rb * GROUP, r0 = KW == kShared ? group0 + wave * ROWS : group0, row_count = PREFIX ? a.batch * int(p.rows.d) : int(p.rows.d);

  int slot, kv;
  if constexpr (PREFIX) {
    slot = a.prefix_slot;
    kv = a.prefix_len;
  } else {
    slot = a.slots[b0];
    kv = min(max(a.kv_lengths[b0], 0), a.cache.capacity);
    if (slot < 0 || slot >= a.cache.slots) slot = kv = 0;
  }

  // This lane's rows: block u, column j.
  int row_id[QB];  // in q's order, -1 past the last row
  int end[QB];     // keys [0, end) are visible
  bool asks[QB];   // it has a query
#pragma unroll
  for (int u = 0; u < QB; ++u) {
    const int r = r0 + 16 * u + j, rc = min(r, row_count - 1);
    const int b = PREFIX ? div_by(rc, p.rows) : b0, rr = PREFIX ? rc - b * int(p.rows.d) : rc;
    const int qi = div_by(rr, p.group), hg = rr - qi * int(p.group.d);
    row_id[u] = r < row_count ? (b * a.heads + head * int(p.group.d) + hg) * a.q_len + qi : -1;
    const int ql = a.q_lengths ? min(max(a.q_lengths[b], 0), a.q_len) : a.q_len;
    int64_t e = kv;
    if (!PREFIX && a.causal) e = min(e, (a.offsets ? int64_t(a.offsets[b]) : int64_t(kv) - ql) + qi + 1);
    asks[u] = r < row_count && qi < ql;
    end[u] = asks[u] ? int(max(e, int64_t(0))) : 0;
  }
  // Keys that some row of the wave sees, and keys that every row of it with a query sees
  // (a row without one may compute anything: it is cleared at the end); keys that some
  // row of the workgroup sees.
  int last, first, group_last;
  if constexpr (PREFIX) {
    last = r0 < row_count ? kv : 0;
    first = group_last = kv;
  } else {
    const int ql = a.q_lengths ? min(max(a.q_lengths[b0], 0), a.q_len) : a.q_len;
    const int64_t off = a.offsets ? int64_t(a.offsets[b0]) : int64_t(kv) - ql;
    const auto seen = [&](int qi) { return int(max(a.causal ? min(int64_t(kv), off + qi + 1) : int64_t(kv), int64_t(0))); };
    const auto last_of = [&](int from, int rows) {
      const int q_last = min(div_by(min(from + rows, row_count) - 1, p.group), ql - 1);
      return from >= row_count || q_last < div_by(from, p.group) ? 0 : seen(q_last);
    };
    last = last_of(r0, ROWS);
    first = last == 0 ? 0 : seen(div_by(r0, p.group));
    group_last = KW == kShared ? last_of(group0, GROUP) : last;
  }
  // (kBoth: tiles [0, shift) are the prefix's.)
  const int shift = BOTH ? (a.prefix_len + kTile - 1) / kTile : 0;
  const int tiles = shift + (group_last + kTile - 1) / kTile, per = (tiles + splits - 1) / splits;
  const int t_end = min(tiles, (split + 1) * per);
  int t = split * per + (KW == kShared ? 0 : wave);

  // The first tile of the slot's head; kBoth: in front of it by `shift`, and the prefix's.
  const int64_t base = (int64_t(slot) * a.cache.kv_heads + head) * (a.cache.capacity / kTile) - shift;
  const int64_t prefix_base = (int64_t(a.prefix_slot) * a.cache.kv_heads + head) * (a.cache.capacity / kTile);
  const auto tile_of = [&](int tt) { return (BOTH && tt < shift ? prefix_base : base) + tt; };
  const uint32_t k_lane = j * 64 + 16 * g, v_lane = lane * 16;
  // Lane (j, g) holds the scales of the tile's key 16 (j / 4) + 4 g + j % 4: of row g's
  // 16 scores of a tile, number 4 kb + v in order, lane 4 kb + v has the scale.
  const int my_key = 16 * (j >> 2) + 4 * g + (j & 3);
  // One block of rows (single tokens): memory has no use for the keys again, and a second
  // product with what the weights' rounding to fp16 leaves out costs nothing that shows,
  // so the result is as near as fp32 weights would bring it.  Two blocks (prompts) take
  // the rounded weights alone: a third less matrix work, 1.3 times the error.
  constexpr bool NT = KEYS == kOwn && QB == 1, FINE = QB == 1;
  // The next tile's K and scales are loaded once the scores have used this one's (one token
  // of 12 heads, 1000 keys: 8.0 us, 9.3 without; 32 of them 11.2 and 12.7), but for two
  // blocks of 64 dims, whose third wave per SIMD that would cost (12 pairs of 4096 rows:
  // 62 us, 57 without).
  constexpr bool AHEAD = QB == 1 || D == 128;
  // Two blocks whose waves widen every tile themselves are bound by that, so K stays at
  // c + 1152 and q . c is summed from -1152 sum_d q_d on: sums of up to 1152 / 127 times the
  // terms of q . c, which are fp32 sums still (their last place 2^-20 of q . c's terms).
  constexpr bool RAISED = QB == 2 && KW != kShared;
  u32x4_t kr[KW == kShared ? 1 : 4][D / 64], vr[KW == kShared ? D / 64 : D / 16];
  float ksr = 0.f, vsr = 0.f;
  auto& shared = *reinterpret_cast<Tiles<D>*>(lds);
  // A tile's bytes, or this wave's quarter of them: 16 keys, and a quarter of the dims of
  // all values.
  auto load_k = [&](int tt) {
    const uint8_t* at = a.cache.k + tile_of(tt) * (kTile * D) + (KW == kShared ? 16 * wave * D : 0);
#pragma unroll
    for (int kb = 0; kb < (KW == kShared ? 1 : 4); ++kb)
#pragma unroll
      for (int c = 0; c < D / 64; ++c) kr[kb][c] = load16<NT>(at + 16 * kb * D + 1024 * c + k_lane);
  };
  auto load_v = [&](int tt) {
    const uint8_t* at = a.cache.v + tile_of(tt) * (kTile * D) + (KW == kShared ? 1024 * wave * (D / 64) : 0);
#pragma unroll
    for (int d = 0; d < (KW == kShared ? D / 64 : D / 16); ++d) vr[d] = load16<NT>(at + 1024 * d + v_lane);
  };
  auto load_scales = [&](int tt) {
    ksr = (a.cache.k_scales + tile_of(tt) * kTile)[uint32_t(my_key)];
    vsr = (a.cache.v_scales + tile_of(tt) * kTile)[uint32_t(my_key)];
  };
  auto share = [&](int buf) {
#pragma unroll
    for (int c = 0; c < D / 64; ++c)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        shared.k[buf][wave][2 * c + s][lane] = widen8(kr[0][c][2 * s], kr[0][c][2 * s + 1]);
        shared.v[buf][wave * (D / 64) + c][s][lane] = widen8(vr[c][2 * s], vr[c][2 * s + 1]);
      }
  };
  if (KW == kShared && t < t_end) {
    load_k(t);
    load_v(t);
  }

  // Step (c, s) of a dot product takes dims 64 c + 16 g + 8 s .. + 7 from lane (., g).
  half8_t qf[QB][D / 32];
  // A row's sum starts at NaN if its query has an infinity or NaN: its scores are infinite, of
  // either sign, or NaN (and all of -inf would pass for a row without a key).
  float l[QB];
#pragma unroll
  for (int u = 0; u < QB; ++u) {
    u16x8_t top = {};
    const uint16_t* qp = a.q + int64_t(max(row_id[u], 0)) * D + 16 * g;
#pragma unroll
    for (int c = 0; c < D / 64; ++c)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        half8_t x;
        __builtin_memcpy(&x, qp + 64 * c + 8 * s, 16);
        top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x8_t, x) & uint16_t(0x7fff));
        qf[u][2 * c + s] = (BOTH ? asks[u] : end[u] > 0) ? x : half8_t{};
      }
    bool inside = true;
#pragma unroll
    for (int e = 0; e < 8; ++e) inside = inside && top[e] < 0x7c00;
    l[u] = __ballot(!inside) >> j & 0x0001000100010001u ? __builtin_nanf("") : 0.f;
  }

  float4_t from[QB];  // where the sums of S start
#pragma unroll
  for (int u = 0; u < QB; ++u) {
    from[u] = float4_t{0.f, 0.f, 0.f, 0.f};
    if constexpr (RAISED) {
      const f16 o = f16(-1152.f);
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
        from[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(half8_t{o, o, o, o, o, o, o, o}, qf[u][i], from[u], 0, 0, 0);
    }
  }

  float m[QB];
  float4_t acc[QB][D / 16];
#pragma unroll
  for (int u = 0; u < QB; ++u) {
    m[u] = kNegInf;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) acc[u][d] = float4_t{0.f, 0.f, 0.f, 0.f};
  }
  // A bound on the value scales so far, those of keys that only some rows see among them: a
  // row's largest score is `room` above its reference, or more, before x + log2 vs can be
  // kRaise above it.  It only spares the exact sums.
  float bound = 0.f, room = kRaise - kLeast;

  const auto tile = [&](int t, int buf, float ks, float vs_, auto after_scores) {
    const bool of_prefix = BOTH && t < shift;
    const int key0 = (t - (of_prefix ? 0 : shift)) * kTile;  // the tile's first key
    const bool full = key0 + kTile <= (of_prefix ? a.prefix_len : first);
    float4_t sc[QB][4];
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
#pragma unroll
      for (int u = 0; u < QB; ++u) sc[u][kb] = from[u];
#pragma unroll
      for (int c = 0; c < D / 64; ++c)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const u32x4_t w = kr[KW == kShared ? 0 : kb][c];
          const half8_t kf = KW == kShared ? shared.k[buf][kb][2 * c + s][lane]
                             : RAISED      ? raise8(w[2 * s], w[2 * s + 1])
                                           : widen8(w[2 * s], w[2 * s + 1]);
#pragma unroll
          for (int u = 0; u < QB; ++u)
            sc[u][kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[u][2 * c + s], sc[u][kb], 0, 0, 0);
        }
      if constexpr (KW != kShared) __builtin_amdgcn_sched_barrier(0);  // (widen one block of 16 keys at a time)
    }
    after_scores();
    const float ck = ks * p.scale;
    // (Past the last key any row sees, scales may be anything.)
    const float vs = key0 + my_key < (of_prefix ? a.prefix_len : last) ? vs_ : 0.f;
    if (__ballot(vs > bound)) {
      const int e = __builtin_amdgcn_frexp_expf(wave_max(vs));
      bound = __builtin_amdgcn_ldexpf(1.f, e);  // > every scale
      room = kRaise - fmaxf(float(e), kLeast);
    }
    half8_t pp[QB][2], rest[2];
#pragma unroll
    for (int u = 0; u < QB; ++u) {
      mul_row(sc[u], ck);
      const int lim = (of_prefix ? a.prefix_len : end[u]) - key0 - 4 * g;  // key 16 kb + v of this lane is visible iff < lim
      const auto mask = [&](float with) {
#pragma unroll
        for (int kb = 0; kb < 4; ++kb)
#pragma unroll
          for (int v = 0; v < 4; ++v) sc[u][kb][v] = 16 * kb + v < lim ? sc[u][kb][v] : with;
      };
      if (!full) mask(kNegInf);
      float high = kNegInf;
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int v = 0; v < 4; ++v) high = fmaxf(high, sc[u][kb][v]);
      if (__ballot(high - m[u] > room)) {  // (m + room would be rounded: far from 0 by more than fp16's range has left)
        high = max_row_sum(sc[u], fmaxf(__builtin_amdgcn_logf(vs), kLeast));
        high = fmaxf(high, __shfl_xor(high, 16, 64));
        high = fmaxf(high, __shfl_xor(high, 32, 64));
        const float nm = high - m[u] > kRaise ? high - kBelow : m[u];
        const float f = m[u] == kNegInf ? 0.f : __builtin_amdgcn_exp2f(m[u] - nm);
        l[u] *= f;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) acc[u][d] *= f;
        m[u] = nm;
      }
      const float ref = m[u] == kNegInf ? 0.f : m[u];  // -inf while every key so far is masked
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          sc[u][kb][v] = __builtin_amdgcn_exp2f(sc[u][kb][v] - ref);
          l[u] += sc[u][kb][v];
        }
      mul_row(sc[u], vs);
      if (!full) mask(0.f);  // (0 times a scale that is not finite)
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int v = 0; v < 4; ++v)
          pp[u][kb >> 1][4 * (kb & 1) + v] = f16(sc[u][kb][v]);
      if constexpr (FINE) {
#pragma unroll
        for (int kb = 0; kb < 4; ++kb)
#pragma unroll
          for (int v = 0; v < 4; ++v)
            rest[kb >> 1][4 * (kb & 1) + v] = f16(sc[u][kb][v] - float(pp[u][kb >> 1][4 * (kb & 1) + v]));
      }
    }
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const half8_t vf = KW == kShared ? shared.v[buf][d][c][lane] : widen8(vr[KW == kShared ? 0 : d][2 * c], vr[KW == kShared ? 0 : d][2 * c + 1]);
#pragma unroll
        for (int u = 0; u < QB; ++u) acc[u][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pp[u][c], acc[u][d], 0, 0, 0);
        if constexpr (FINE) acc[0][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, rest[c], acc[0][d], 0, 0, 0);
      }
      if constexpr (KW != kShared) __builtin_amdgcn_sched_barrier(0);
    }
  };
  if constexpr (KW == kShared) {
    if (t < t_end) {
      share(0);
      load_scales(t);
      if (t + 1 < t_end) {
        load_k(t + 1);
        load_v(t + 1);
      }
    }
    for (int buf = 0; t < t_end; ++t, buf ^= 1) {
      lds_barrier();  // (the next tile's loads stay in flight)
      const float ks = ksr, vs = vsr;
      if (t + 1 < t_end) {
        share(buf ^ 1);
        load_scales(t + 1);
        if (t + 2 < t_end) {
          load_k(t + 2);
          load_v(t + 2);
        }
      }
      if (t * kTile < last) tile(t, buf, ks, vs, [] {});
    }
  } else {
    if (AHEAD && t < t_end) {
      load_k(t);
      load_scales(t);
    }
    for (; t < t_end; t += KW) {
      if (!AHEAD) {
        load_k(t);
        load_scales(t);
      }
      const float ks = ksr, vs = vsr;
      load_v(t);
      __builtin_amdgcn_sched_barrier(0);
      tile(t, 0, ks, vs, [&] {
        if constexpr (AHEAD) {
          if (t + KW < t_end) {
            load_k(t + KW);
            load_scales(t + KW);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      });
    }
  }

#pragma unroll
  for (int u = 0; u < QB; ++u) {
    l[u] += __shfl_xor(l[u], 16, 64);
    l[u] += __shfl_xor(l[u], 32, 64);
    if (BOTH ? !asks[u] : end[u] == 0) l[u] = 0.f;
  }
  // Dims 16 d + 4 g .. + 3 of row (u, j), of `total` weight at exponent reference `top`.
  const auto put = [&](int u, int d, float4_t o, float total) {
    if (row_id[u] < 0) return;
    if (p.parts) {
      const int64_t at = int64_t(state) * p.all_rows + row_id[u];
      if (total != 0.f) *reinterpret_cast<float4_t*>(a.workspace + at * D + 16 * d + 4 * g) = o;
      return;
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    const half4_t y = output_of(o, total, inv);
    __builtin_memcpy(a.out + int64_t(row_id[u]) * D + 16 * d + 4 * g, &y, 8);
  };
  const auto put_weight = [&](int u, float top, float total) {
    if (!p.parts || g != 0 || row_id[u] < 0) return;
    const int64_t states = int64_t(p.splits + p.prefix_splits) * p.all_rows;
    float* ml = a.workspace + states * D + 2 * (int64_t(state) * p.all_rows + row_id[u]);
    ml[0] = top;
    ml[1] = total;
  };
  if constexpr (KW == kShared) {
#pragma unroll
    for (int u = 0; u < QB; ++u) {
#pragma unroll
      for (int d = 0; d < D / 16; ++d) put(u, d, acc[u][d], l[u]);
      put_weight(u, m[u], l[u]);
    }
  } else {
    // The waves' states meet in LDS; wave w joins every KW-th piece of 16 dims.
    auto& mg = *reinterpret_cast<Merge<D, QB, KW>*>(lds);
#pragma unroll
    for (int u = 0; u < QB; ++u) {
#pragma unroll
      for (int d = 0; d < D / 16; ++d) mg.acc[wave][u * (D / 16) + d][lane] = acc[u][d];
      if (g == 0) {
        mg.m[wave][u][j] = m[u];
        mg.l[wave][u][j] = l[u];
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < QB; ++u) {
      float top = kNegInf, total = 0.f, f[KW];
      bool empty[KW];  // (what it holds is no row's; a state with keys counts however little it weighs: 0 times NaN is NaN)
#pragma unroll
      for (int w = 0; w < KW; ++w) top = mg.l[w][u][j] == 0.f ? top : fmaxf(top, mg.m[w][u][j]);
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        const float lw = mg.l[w][u][j];
        empty[w] = lw == 0.f;
        f[w] = empty[w] ? 0.f : __builtin_amdgcn_exp2f(mg.m[w][u][j] - top);
        total += lw * f[w];
      }
#pragma unroll
      for (int d0 = 0; d0 < D / 16; d0 += KW) {
        const int d = d0 + wave;
        float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < KW; ++w) {
          const float4_t x = mg.acc[w][u * (D / 16) + d][lane];
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = empty[w] ? o[e] : fmaf(x[e], f[w], o[e]);
        }
        put(u, d, o, total);
      }
      if (wave == 0) put_weight(u, top, total);
    }
  }
}

// Waves per SIMD that the registers are budgeted for.  What the compiler takes: 64 dims, one
// block 121 registers of 128 (four waves), two 158 to 164 of 256 (three waves fit); 128 dims,
// one block 177 of 256, two sharing tiles 218, two that widen for themselves all 256 and 1 to 5
// more that are spilled (8 to 24 bytes a lane).
constexpr int waves_for(int dim, int qb) { return dim == 64 && qb == 1 ? 4 : 2; }

// QB, PB: row blocks of 16 per wave over the requests' own keys and the prefix's (0:
// no prefix, kInline: walked in front of the own keys); KW: waves that share a row block's
// keys.
constexpr int kInline = -1;
template <int D, int QB, int PB, int KW>
__global__ __launch_bounds__(KW == kShared ? 256 : 64 * KW, waves_for(D, QB > PB ? QB : PB)) void kv_attention_kernel(AttnPlan p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  int id = int(blockIdx.x);
  const int heads = p.a.cache.kv_heads;
  if constexpr (PB > 0) {
    if (id < p.prefix_wgs) {
      const int blocks = div_by(id, p.heads), split = div_by(blocks, p.prefix_block_div);
      attend<D, PB, KW, kPrefix>(p, lds, 0, id - blocks * heads, blocks - split * int(p.prefix_block_div.d), split, p.prefix_splits,
                              p.splits + split);
      return;
    }
    id -= int(p.prefix_wgs);
  }
  // The last row blocks of all (request, key head) pairs first: under the causal mask
  // they are the longest.
  const int block = div_by(id, p.pairs), at = id - block * int(p.pairs.d), b = div_by(at, p.heads);
  const int split = div_by(block, p.row_block_div), blocks = int(p.row_block_div.d);
  attend<D, QB, KW, PB == kInline ? kBoth : kOwn>(p, lds, b, at - b * heads, blocks - 1 - (block - split * blocks), split, p.splits, split);
}

// W waves of a workgroup of 4 join a row's states: D / 4 lanes a state, 2 or 4 states at a
// time and wave.  A launch and its dependent loads: 3.2 us for 384 rows of 3 states of 64,
// 4.2 for 512 rows of 4 and 4.3 for 2048 rows of 5 of 128.  Four waves from 17 states on:
// one token of 12 heads over 9000 keys in 36 splits takes 11.2 us, 13.3 with one wave.
template <int D, int W>
__global__ __launch_bounds__(256) void kv_attention_join_kernel(AttnPlan p) {
  constexpr int LPR = D / 4, PARTS = 64 / LPR;
  __shared__ float4_t sums[W][LPR];
  __shared__ float weights[W];
  const int lane = int(threadIdx.x & 63), wave = int(threadIdx.x >> 6) % W, part = lane / LPR, at = 4 * (lane % LPR);
  const int64_t row = int64_t(blockIdx.x) * (4 / W) + int(threadIdx.x >> 6) / W;
  if (row >= p.all_rows) return;  // (a workgroup of one row has it)
  const int states = p.splits + p.prefix_splits;
  const float* ml = p.a.workspace + int64_t(states) * p.all_rows * D;
  float top = kNegInf;
  for (int s = lane; s < states; s += 64) {
    const float* x = ml + 2 * (s * p.all_rows + row);
    if (x[1] != 0.f) top = fmaxf(top, x[0]);
  }
  top = wave_max(top);
  float total = 0.f;
  float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = wave * PARTS + part; s < states; s += W * PARTS) {
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

// How a set of keys is walked: `blocks` row blocks of 16 per wave, `waves` waves to a
// row block or kShared, `splits` workgroups to its keys.
struct Walk {
  int blocks, waves, splits;
};

// From the number of (request, key head) pairs, the rows of one and the tiles of 64 keys
// of the longest.  Two blocks of 16 rows use every widened key and value twice; they
// pay where there are plenty of row blocks (100 pairs of 1024 rows: 31 us against 60; 288
// pairs of 100 rows: 8.9 against 10.7), or many keys to them (128 pairs of 64 rows over 2000
// keys, D 128: 22 against 30; 8 pairs of 256 rows over 16000: 37 against 52), not where
// both are few (12 pairs of 512 rows: 8.2 against 6.9; 128 pairs of 20 rows over 2000 keys,
// D 128: 20 against 19).
// Waves: with row blocks to fill every SIMD twice a workgroup takes four of them and its
// waves share the tiles, each widened once instead of four times and nothing merged (100
// pairs of 1024 rows: 31.3 us, 35.7 with two waves to a row block, 44 with four; 75 pairs:
// 29.8, 32.6, 39.8; 8 pairs of 8192 rows over 8000 keys, D 128: 278, 301, 298); below that
// two waves share a row block, or four where keys are many (12 pairs of 4096 rows: 51 us,
// 60 with two, 81 with shared tiles; 24 pairs of 2048 rows without a mask: 52, 50, 61; 16
// pairs of 3108 rows over 6001 keys, D 128: 205, 224, 212).
// Splits: a second launch and the states' traffic cost 2 us and more, and 4 us of the
// caller's time, so short caches are not split (96 pairs, 1024 keys: 8.4 us, 9.4 in four; 12
// pairs, 7.6 and 7.8, of 1500 keys 9.5 and 8.3; 8 of 1024, D 128, 9.7 and 8.7).  Longer ones
// are, into at most one workgroup a CU (8 pairs of 16000 keys, D 128: 13.3 us in 256
// workgroups, 17 in 320 or 512; 24 of 60000: 65 in 192, 87 in 264) and 64 splits (one pair
// of 100000 keys: 21 us, 25 in 256), but where the pairs alone take more than half of the
// CUs into about 512 (160 pairs of 10000 to 20000 keys: 114 us, 130 whole; 272 of 4000 to
// 12000: 108, 117).
Walk walk_for(int64_t pairs, int rows, int keys, int dim) {
  const int64_t tiles = ceil_div(keys, kTile), twos = pairs * ceil_div(rows, 32), plenty = dim == 64 ? 1024 : 512;
  Walk w{1, 4, 1};
  if (rows > 16 && (twos >= plenty || tiles >= 128 || (twos >= 128 && twos * tiles > 4096))) w.blocks = 2;
  if (w.blocks == 2 && twos >= plenty) {
    w.waves = twos >= 2048 ? kShared : twos >= 1024 && tiles < 32 ? 2 : 4;
    return w;
  }
  const int64_t wgs = pairs * ceil_div(rows, 16 * w.blocks);
  if (tiles > (dim == 64 ? 24 : 16))
    w.splits = int(wgs > 128 && tiles >= 64 ? ceil_div(512, wgs) : std::max<int64_t>(1, std::min<int64_t>({256 / wgs, tiles / 4, 64})));
  return w;
}
// A prefix: two blocks by the work alone (its keys are re-read from the L2 by all its row
// blocks: 64 requests of 4 rows, 8 heads of 128, 4000 keys 23.5 us against 24.7, 256
// requests over 2000 42 against 52; 8 requests over 9000 18.1 against 15.7, 400 requests of
// 12 heads of 64 over 1000 39 against 34).  Its states are joined with the requests' own in
// any case, so splitting it costs less: into about 192 workgroups, 256 from 8192 keys on (64
// requests of 4 rows, 8 heads, 16001 keys: 63 us in 128 workgroups, 42 in 256, 44 in 512).
Walk prefix_walk_for(int heads, int64_t rows, int keys) {
  const int64_t tiles = ceil_div(keys, kTile);
  Walk w{rows > 16 && heads * ceil_div(rows, 32) * tiles >= 3000 ? 2 : 1, 4, 1};
  const int64_t wgs = heads * ceil_div(rows, 16 * w.blocks);
  w.splits = int(std::max<int64_t>(1, std::min(ceil_div(tiles >= 128 ? 256 : 192, wgs), tiles / 4)));
  return w;
}

// Whether every request walks the prefix in front of its own keys by itself: one launch in
// place of two, no workspace and no states, where that is little work.  By itself against
// shared, us: 12 heads of 64, prefix 700, 1 / 8 / 32 / 64 requests 7.1 / 7.3 / 10.0 / 13.1 and
// 8.5 / 8.7 / 9.5 / 9.8 (but for 32 the second launch's 4 us of the caller's time are saved);
// prefix 960, 32 requests 11.6 and 9.1; 1500, 4 requests 10.8 and 8.4; 8 heads of 128, 700,
// 64 requests 14.4 and 16.2, 200, 10.1 and 13.5.
bool prefix_inline(int64_t pairs, int rows, int keys, int prefix, int dim) {
  const int64_t tiles = ceil_div(keys, kTile) + ceil_div(prefix, kTile);
  return rows <= 16 && tiles <= 16 && pairs * tiles <= (dim == 64 ? 5000 : 6500);
}

AttnPlan plan_of(const KvAttnArgs& a, Walk& own, Walk& prefix) {
  AttnPlan p{};
  p.a = a;
  p.scale = float(1.4426950408889634 / __builtin_sqrt(double(a.cache.head_dim)));
  const int group = a.heads / a.cache.kv_heads, rows = group * a.q_len;
  const int64_t pairs = int64_t(a.batch) * a.cache.kv_heads;
  p.group = divisor(group);
  p.rows = divisor(rows);
  p.heads = divisor(a.cache.kv_heads);
  p.pairs = divisor(uint32_t(pairs));
  p.all_rows = pairs * rows;
  own = walk_for(pairs, rows, a.max_kv, a.cache.head_dim);
  prefix = Walk{0, 4, 0};
  if (a.prefix_len > 0 && prefix_inline(pairs, rows, a.max_kv, a.prefix_len, a.cache.head_dim)) {
    own = Walk{1, 4, 1};
    prefix.blocks = kInline;
  } else if (a.prefix_len > 0) {
    const int64_t all = int64_t(a.batch) * rows;
    prefix = prefix_walk_for(a.cache.kv_heads, all, a.prefix_len);
    own.waves = 4;
    const int64_t blocks = ceil_div(all, 16 * prefix.blocks);
    p.prefix_block_div = divisor(uint32_t(blocks));
    p.prefix_wgs = a.cache.kv_heads * blocks * prefix.splits;
  }
  const int64_t blocks = ceil_div(rows, 16 * own.blocks * (own.waves == kShared ? 4 : 1));
  p.row_block_div = divisor(uint32_t(blocks));
  p.own_wgs = pairs * blocks * own.splits;
  p.splits = own.splits;
  p.prefix_splits = prefix.splits;
  p.parts = p.splits + p.prefix_splits > 1;
  return p;
}

template <int D, int QB, int PB, int KW>
hipError_t launch(const AttnPlan& p, hipStream_t stream) {
  constexpr int bytes =
      KW == kShared ? int(sizeof(Tiles<D>)) : int(std::max(sizeof(Merge<D, QB, (KW > 0 ? KW : 1)>), PB > 0 ? sizeof(Merge<D, (PB > 0 ? PB : 1), (KW > 0 ? KW : 1)>) : size_t(0)));
  if constexpr (bytes > 64 * 1024) {  // (two blocks of 128-dim rows)
    static LdsLimit limit;
    const hipError_t e = limit.raise(reinterpret_cast<const void*>(&kv_attention_kernel<D, QB, PB, KW>), bytes);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((kv_attention_kernel<D, QB, PB, KW>), dim3(unsigned(p.prefix_wgs + p.own_wgs)), dim3(KW == kShared ? 256 : 64 * KW), bytes,
                     stream, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !p.parts) return e;
  if (p.splits + p.prefix_splits > 16)
    hipLaunchKernelGGL((kv_attention_join_kernel<D, 4>), dim3(unsigned(p.all_rows)), dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((kv_attention_join_kernel<D, 1>), dim3(unsigned(ceil_div(p.all_rows, 4))), dim3(256), 0, stream, p);
  return hipGetLastError();
}

template <int D>
hipError_t launch_walk(const AttnPlan& p, const Walk& own, const Walk& prefix, hipStream_t stream) {
  if (own.waves == kShared) return launch<D, 2, 0, kShared>(p, stream);
  if (own.waves == 2) return launch<D, 2, 0, 2>(p, stream);
  if (own.blocks == 1) {
    if (prefix.blocks == kInline) return launch<D, 1, kInline, 4>(p, stream);
    if (prefix.blocks == 0) return launch<D, 1, 0, 4>(p, stream);
    return prefix.blocks == 1 ? launch<D, 1, 1, 4>(p, stream) : launch<D, 1, 2, 4>(p, stream);
  }
  if (prefix.blocks == 0) return launch<D, 2, 0, 4>(p, stream);
  return prefix.blocks == 1 ? launch<D, 2, 1, 4>(p, stream) : launch<D, 2, 2, 4>(p, stream);
}

}  // namespace

int64_t kv_attention_workspace(const KvAttnArgs& a) {
  Walk own, prefix;
  const AttnPlan p = plan_of(a, own, prefix);
  return p.parts ? int64_t(p.splits + p.prefix_splits) * p.all_rows * (a.cache.head_dim + 2) * 4 : 0;
}

hipError_t kv_attention(const KvAttnArgs& a, hipStream_t stream) {
  Walk own, prefix;
  const AttnPlan p = plan_of(a, own, prefix);
  return a.cache.head_dim == 64 ? launch_walk<64>(p, own, prefix, stream) : launch_walk<128>(p, own, prefix, stream);
}

}  // namespace tia
