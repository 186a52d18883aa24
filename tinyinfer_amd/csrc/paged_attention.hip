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
// they count as 0 in the product and a second product of ones, over the keys that a row
// sees, says which sums must be NaN all the same.
#include <algorithm>
#include <type_traits>

#include "divisor.hpp"
#include "lds_limit.hpp"
#include "paged_cache.hpp"

namespace tia {
namespace {

constexpr int kTile = 64;   // keys per wave and step
constexpr float kNegInf = -__builtin_huge_valf();
// The reference of a row's exponents: 6 below its largest x when set, raised when one is
// 14 above it.  Weights then lie around 2^6 and below 2^14: rounded to fp16, whose smallest
// normal number is 2^-14, a weight 2^-20 times the heaviest still keeps 11 bits.
constexpr float kBelow = 6.f, kRaise = 14.f;

struct AttnPlan {
  PagedAttnArgs a;
  float scale;             // D^-1/2 log2 e
  int page_shift;          // log2(page_size / 32)
  Divisor group, rows;     // query heads per key head; rows of one request and key head
  Divisor heads, pairs;    // key heads; (request, key head) pairs
  Divisor row_block_div;   // row blocks of a pair
  int splits;              // of a request's keys
  int64_t workgroups;
  int64_t all_rows;        // batch * heads * q_len
};

typedef unsigned short u16x8_t __attribute__((ext_vector_type(8)));

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

// Waves' states as they meet in LDS: of lane (j, g)'s dims, number v of 4 and b of D / 16
// lie next to each other in b.
template <int D, int QB, int KW>
struct Merge {
  float4_t acc[KW][QB][4][D / 64][64];
  float m[KW][QB][16], l[KW][QB][16];
};

// A tile's operands as the waves of a workgroup share them, in the order in which a
// lane reads them: 16 bytes per lane, one conflict-free kilobyte per operand.
template <int D>
struct Tiles {
  half8_t k[2][4][D / 32][64], v[2][2][D / 16][64];
};

// KW waves share a row block, each with its own tiles; kShared: 4 waves have a row block
// each (`rb` counts those groups) and share every tile, each bringing a quarter of it into
// LDS while the tile before is worked on.
constexpr int kShared = 0;
template <int D, int QB, int KW>
__device__ __forceinline__ void attend(const AttnPlan& p, uint8_t* lds, int b, int head, int rb, int split) {
  const PagedAttnArgs& a = p.a;
  const int lane = int(threadIdx.x & 63), wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
  const int j = lane & 15, g = lane >> 4;
  constexpr bool SHARED = KW == kShared;
  constexpr int ROWS = 16 * QB, GROUP = SHARED ? 4 * ROWS : ROWS, STEP = SHARED ? 1 : KW, PER = D / 16;
  const int group0 = rb * GROUP, r0 = SHARED ? group0 + wave * ROWS : group0, row_count = int(p.rows.d);

  const int64_t held = int64_t(a.pages.width) * a.cache.page_size;
  const int kv = int(min(int64_t(max(a.kv_lengths[b], 0)), held));

  // This lane's rows: block u, column j.
  const int ql = a.q_lengths ? min(max(a.q_lengths[b], 0), a.q_len) : a.q_len;
  const int64_t off = a.offsets ? int64_t(a.offsets[b]) : int64_t(kv) - ql;
  const auto seen = [&](int qi) { return int(max(a.causal ? min(int64_t(kv), off + qi + 1) : int64_t(kv), int64_t(0))); };
  int row_id[QB];  // in q's order, -1 past the last row
  int end[QB];     // keys [0, end) are visible
#pragma unroll
  for (int u = 0; u < QB; ++u) {
    const int r = r0 + 16 * u + j, rc = min(r, row_count - 1);
    const int qi = div_by(rc, p.group), hg = rc - qi * int(p.group.d);
    row_id[u] = r < row_count ? (b * a.heads + head * int(p.group.d) + hg) * a.q_len + qi : -1;
    end[u] = r < row_count && qi < ql ? seen(qi) : 0;
  }
  // Keys that some row of the wave sees, and keys that every row of it with a query sees
  // (a row without one may compute anything: it is cleared at the end); keys that some
  // row of the workgroup sees.
  const auto last_of = [&](int from, int rows) {
    const int q_last = min(div_by(min(from + rows, row_count) - 1, p.group), ql - 1);
    return from >= row_count || q_last < div_by(from, p.group) ? 0 : seen(q_last);
  };
  const int last = last_of(r0, ROWS), first = last == 0 ? 0 : seen(div_by(r0, p.group));
  const int group_last = SHARED ? last_of(group0, GROUP) : last, group_first = seen(div_by(group0, p.group));
  const int tiles = (group_last + kTile - 1) / kTile, per = (tiles + p.splits - 1) / p.splits;
  const int t_end = min(tiles, (split + 1) * per);
  int t = split * per + (SHARED ? 0 : wave);

  // Pages of the halves of this wave's tiles from `t0` on, tile t0 + STEP i in lane i.
  const int32_t* table = a.pages.table + int64_t(b) * a.pages.width;
  int ids[2], ids_from = t;
  const auto look_up = [&](int t0) {
    ids_from = t0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int entry = (2 * (t0 + STEP * lane) + h) >> p.page_shift;
      const int id = entry < a.pages.width ? table[entry] : -1;
      ids[h] = id < a.cache.page_count ? id : -1;
    }
  };
  const auto page_of = [&](int tt, int h) { return __builtin_amdgcn_readlane(ids[h], (tt - ids_from) / STEP & 63); };
  // Tokens 64 tt + 32 h .. + 31 of the head: K (V is `to_v` behind).
  const int64_t head_size = paged_head_size(a.cache), to_v = int64_t(a.cache.page_size) * D;
  const auto half_on = [&](int page, int half) {
    return a.cache.pages + (int64_t(page) * a.cache.kv_heads + head) * head_size + (half & ((1 << p.page_shift) - 1)) * (32 * D);
  };
  const auto half_at = [&](int tt, int h) { return half_on(max(page_of(tt, h), 0), 2 * tt + h); };

  // One block of rows (single tokens): memory has no use for the keys again, and a second
  // product with what the weights' rounding to fp16 leaves out costs nothing that shows,
  // so the result is as near as fp32 weights would bring it.  Two blocks (prompts) take
  // the rounded weights alone: a third less matrix work.
  constexpr bool NT = QB == 1, FINE = QB == 1;
  // Two blocks of 128 dims leave no registers to load ahead into.
  constexpr bool AHEAD = QB == 1 || D == 64;
  half8_t kr[SHARED ? 1 : 4][D / 32], vr[SHARED ? 1 : PER][2];
  auto& shared = *reinterpret_cast<Tiles<D>*>(lds);
  const auto load_k = [&](int tt) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint16_t* at = half_at(tt, h);
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int c = 0; c < D / 32; ++c) kr[2 * h + kb][c] = load16<NT>(at + 16 * kb * D + 512 * c + uint32_t(8 * lane));
    }
  };
  const auto load_v = [&](int tt) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint16_t* at = half_at(tt, h) + to_v;
#pragma unroll
      for (int d = 0; d < PER; ++d) vr[d][h] = load16<NT>(at + 512 * d + uint32_t(8 * lane));
    }
  };
  // This wave's quarter of a tile into LDS: 16 keys, and half the dims of a half's values.
  const auto share = [&](int tt, int buf) {
    const uint16_t* at = half_at(tt, wave >> 1) + 8 * lane;
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
      __builtin_amdgcn_global_load_lds((global_ptr)(at + (wave & 1) * 16 * D + 512 * c), (lds_ptr)&shared.k[buf][wave][c][0], 16, 0, 0);
#pragma unroll
    for (int d = 0; d < PER / 2; ++d)
      __builtin_amdgcn_global_load_lds((global_ptr)(at + to_v + ((wave & 1) * (PER / 2) + d) * 512),
                                       (lds_ptr)&shared.v[buf][wave >> 1][(wave & 1) * (PER / 2) + d][0], 16, 0, 0);
  };
  if (t < t_end) {
    look_up(t);
    if constexpr (SHARED) share(t, 0);
    else if (AHEAD) load_k(t);
  }

  half8_t qf[QB][D / 32];
  // A row's sum starts at NaN if its query has an infinity or NaN: its scores are infinite, of
  // either sign, or NaN (and all of -inf would pass for a row without a key).
  float l[QB], m[QB];
  unsigned spoilt[QB];  // bit 4 d + e: the sum acc[u][d][e] is over an infinity or NaN that is not in it
  float4_t acc[QB][PER];
#pragma unroll
  for (int u = 0; u < QB; ++u) {
    u16x8_t top = {};
    const uint16_t* qp = a.q + int64_t(max(row_id[u], 0)) * D + 8 * g;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      half8_t x;
      __builtin_memcpy(&x, qp + 32 * c, 16);
      top = top_bits(top, x);
      qf[u][c] = end[u] > 0 ? x : half8_t{};
    }
    l[u] = __ballot(any_not_finite(top)) >> j & 0x0001000100010001u ? __builtin_nanf("") : 0.f;
    m[u] = kNegInf;
    spoilt[u] = 0;
#pragma unroll
    for (int d = 0; d < PER; ++d) acc[u][d] = float4_t{0.f, 0.f, 0.f, 0.f};
  }

  const auto value = [&](int buf, int d, int h) { return SHARED ? shared.v[buf][h][d][lane] : vr[SHARED ? 0 : d][h]; };
  // Key 16 kb + v of this lane, of the tile from key0 on, is visible to row (u, j) iff it is
  // below its half's limit.
  const auto sees = [&](int u, int key0, bool held0, bool held1, int kb, int v) {
    return 16 * kb + v < ((kb < 2 ? held0 : held1) ? end[u] - key0 - 4 * g : 0);
  };
  // A tile of which a row may not see everything: whether it has an infinity or NaN, the sums
  // that must be NaN for one that their row sees, and a value with a finite number in its place.
  const auto any_odd = [&](int buf) {
    u16x8_t top = {};
#pragma unroll
    for (int d = 0; d < PER; ++d) top = top_bits(top_bits(top, value(buf, d, 0)), value(buf, d, 1));
    return __ballot(any_not_finite(top)) != 0;
  };
  const auto spoil = [&](int t, int buf, bool held0, bool held1) {
    half8_t ones[QB][2];
#pragma unroll
    for (int u = 0; u < QB; ++u)
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int v = 0; v < 4; ++v) ones[u][kb >> 1][4 * (kb & 1) + v] = sees(u, t * kTile, held0, held1, kb, v) ? f16(1.f) : f16(0.f);
    // (Rolled, and the values read once more: this is rare, and registers are not.)
#pragma unroll 1
    for (int d = 0; d < PER; ++d) {
      float4_t hits[QB];
#pragma unroll
      for (int u = 0; u < QB; ++u) hits[u] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        half8_t x, bad;
        if constexpr (SHARED) x = shared.v[buf][h][d][lane];
        else x = load16<false>(half_on((h ? held1 : held0) ? table[(2 * t + h) >> p.page_shift] : 0, 2 * t + h) + to_v + 512 * d + uint32_t(8 * lane));
#pragma unroll
        for (int e = 0; e < 8; ++e) bad[e] = (__builtin_bit_cast(u16x8_t, x)[e] & 0x7fff) >= 0x7c00 ? f16(1.f) : f16(0.f);
#pragma unroll
        for (int u = 0; u < QB; ++u) hits[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bad, ones[u][h], hits[u], 0, 0, 0);
      }
#pragma unroll
      for (int u = 0; u < QB; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) spoilt[u] |= hits[u][e] > 0.f ? 1u << (4 * d + e) : 0u;
    }
  };
  const auto finite = [](half8_t x) {
    const f16 most = f16(65504.f);
    const half8_t high = {most, most, most, most, most, most, most, most};
    return __builtin_elementwise_max(__builtin_elementwise_min(x, high), -high);
  };

  const auto tile = [&](int t, int buf, bool held0, bool held1, auto after_scores) {
    const int key0 = t * kTile;
    const bool full = key0 + kTile <= first && held0 && held1;
    float4_t sc[QB][4];
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
#pragma unroll
      for (int u = 0; u < QB; ++u) sc[u][kb] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        const half8_t kf = SHARED ? shared.k[buf][kb][c][lane] : kr[SHARED ? 0 : kb][c];
#pragma unroll
        for (int u = 0; u < QB; ++u) sc[u][kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[u][c], sc[u][kb], 0, 0, 0);
      }
    }
    after_scores();
    half8_t pp[QB][2], rest[2];
    const auto visible = [&](int u, int kb, int v) { return sees(u, key0, held0, held1, kb, v); };
#pragma unroll
    for (int u = 0; u < QB; ++u) {
      if (!full) {
#pragma unroll
        for (int kb = 0; kb < 4; ++kb)
#pragma unroll
          for (int v = 0; v < 4; ++v) sc[u][kb][v] = visible(u, kb, v) ? sc[u][kb][v] : kNegInf;
      }
      float high = kNegInf;
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int v = 0; v < 4; ++v) high = fmaxf(high, sc[u][kb][v]);
      high *= p.scale;
      if (__ballot(high > m[u] + kRaise)) {
        high = fmaxf(high, __shfl_xor(high, 16, 64));
        high = fmaxf(high, __shfl_xor(high, 32, 64));
        const float nm = high > m[u] + kRaise ? high - kBelow : m[u];
        const float f = m[u] == kNegInf ? 0.f : __builtin_amdgcn_exp2f(m[u] - nm);
        l[u] *= f;
#pragma unroll
        for (int d = 0; d < PER; ++d) acc[u][d] *= f;
        m[u] = nm;
      }
      const float ref = m[u] == kNegInf ? 0.f : -m[u];  // -inf while every key so far is masked
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float w = __builtin_amdgcn_exp2f(fmaf(sc[u][kb][v], p.scale, ref));
          l[u] += w;
          pp[u][kb >> 1][4 * (kb & 1) + v] = f16(w);
          if constexpr (FINE) rest[kb >> 1][4 * (kb & 1) + v] = f16(w - float(f16(w)));
        }
    }
    if constexpr (!SHARED) {
      if (!full && any_odd(0)) {
        spoil(t, 0, held0, held1);
#pragma unroll
        for (int d = 0; d < PER; ++d)
#pragma unroll
          for (int h = 0; h < 2; ++h) vr[d][h] = finite(vr[d][h]);
      }
    }
#pragma unroll
    for (int d = 0; d < PER; ++d)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const half8_t vf = value(buf, d, h);
#pragma unroll
        for (int u = 0; u < QB; ++u) acc[u][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pp[u][h], acc[u][d], 0, 0, 0);
        if constexpr (FINE) acc[0][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, rest[h], acc[0][d], 0, 0, 0);
      }
  };
  // (The pages of tile t are at hand; those of t + STEP afterwards.)
  const auto next_pages = [&](int tt) {
    if (tt - ids_from >= 64 * STEP) look_up(tt);
  };
  if constexpr (SHARED) {
    for (int buf = 0; t < t_end; ++t, buf ^= 1) {
      const bool held0 = page_of(t, 0) >= 0, held1 = page_of(t, 1) >= 0;
      __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's quarter has landed
      lds_barrier();                        // everyone's has, and nobody reads the other buffer any more
      if (t + 1 < t_end) {
        next_pages(t + 1);
        share(t + 1, buf ^ 1);
      }
      // (The same for all waves: what they find lies in LDS.)
      if (((t + 1) * kTile > group_first || !held0 || !held1) && any_odd(buf)) {
        spoil(t, buf, held0, held1);
        lds_barrier();
#pragma unroll
        for (int d = 0; d < PER / 2; ++d) {
          half8_t& x = shared.v[buf][wave >> 1][(wave & 1) * (PER / 2) + d][lane];
          x = finite(x);
        }
        lds_barrier();
      }
      if (t * kTile < last) tile(t, buf, held0, held1, [] {});
    }
  } else {
    for (; t < t_end; t += KW) {
      const bool held0 = page_of(t, 0) >= 0, held1 = page_of(t, 1) >= 0;
      if (!AHEAD) load_k(t);
      else load_v(t);
      __builtin_amdgcn_sched_barrier(0);
      tile(t, 0, held0, held1, [&] {
        __builtin_amdgcn_sched_barrier(0);
        if (!AHEAD) load_v(t);
        if (t + KW < t_end) {
          next_pages(t + KW);
          if (AHEAD) load_k(t + KW);
        }
        __builtin_amdgcn_sched_barrier(0);
      });
    }
  }

#pragma unroll
  for (int u = 0; u < QB; ++u) {
    l[u] += __shfl_xor(l[u], 16, 64);
    l[u] += __shfl_xor(l[u], 32, 64);
    if (end[u] == 0) l[u] = 0.f;
    if (__ballot(spoilt[u] != 0)) {
#pragma unroll
      for (int d = 0; d < PER; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[u][d][e] = spoilt[u] >> (4 * d + e) & 1 ? __builtin_nanf("") : acc[u][d][e];
    }
  }
  // Dims PER (4 g + v) + 4 c .. + 3 of row (u, j), of `total` weight at exponent reference `top`.
  const auto put = [&](int u, int v, int c, float4_t o, float total) {
    if (row_id[u] < 0) return;
    const int dim = PER * (4 * g + v) + 4 * c;
    if (p.splits > 1) {
      const int64_t at = int64_t(split) * p.all_rows + row_id[u];
      if (total != 0.f) *reinterpret_cast<float4_t*>(a.workspace + at * D + dim) = o;
      return;
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    const half4_t y = output_of(o, total, inv);
    __builtin_memcpy(a.out + int64_t(row_id[u]) * D + dim, &y, 8);
  };
  const auto put_weight = [&](int u, float top, float total) {
    if (p.splits == 1 || g != 0 || row_id[u] < 0) return;
    float* ml = a.workspace + p.splits * p.all_rows * D + 2 * (int64_t(split) * p.all_rows + row_id[u]);
    ml[0] = top;
    ml[1] = total;
  };
  const auto piece = [&](int u, int v, int c) {
    return float4_t{acc[u][4 * c][v], acc[u][4 * c + 1][v], acc[u][4 * c + 2][v], acc[u][4 * c + 3][v]};
  };
  if constexpr (SHARED) {
#pragma unroll
    for (int u = 0; u < QB; ++u) {
#pragma unroll
      for (int v = 0; v < 4; ++v)
#pragma unroll
        for (int c = 0; c < D / 64; ++c) put(u, v, c, piece(u, v, c), l[u]);
      put_weight(u, m[u], l[u]);
    }
  } else {
    // The waves' states meet in LDS; wave w joins every KW-th v.
    auto& mg = *reinterpret_cast<Merge<D, QB, KW>*>(lds);
#pragma unroll
    for (int u = 0; u < QB; ++u) {
#pragma unroll
      for (int v = 0; v < 4; ++v)
#pragma unroll
        for (int c = 0; c < D / 64; ++c) mg.acc[wave][u][v][c][lane] = piece(u, v, c);
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
      for (int v0 = 0; v0 < 4; v0 += KW)
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int w = 0; w < KW; ++w) {
            const float4_t x = mg.acc[w][u][v0 + wave][c][lane];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = empty[w] ? o[e] : fmaf(x[e], f[w], o[e]);
          }
          put(u, v0 + wave, c, o, total);
        }
      if (wave == 0) put_weight(u, top, total);
    }
  }
}

constexpr int waves_for(int dim, int qb) { return dim == 64 && qb == 1 ? 3 : 2; }

template <int D, int QB, int KW>
__global__ __launch_bounds__(KW == kShared ? 256 : 64 * KW, waves_for(D, QB)) void paged_attention_kernel(AttnPlan p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  // The last row blocks of all (request, key head) pairs first: under the causal mask
  // they are the longest.
  const int id = int(blockIdx.x), block = div_by(id, p.pairs), at = id - block * int(p.pairs.d), b = div_by(at, p.heads);
  const int split = div_by(block, p.row_block_div), blocks = int(p.row_block_div.d);
  attend<D, QB, KW>(p, lds, b, at - b * int(p.heads.d), blocks - 1 - (block - split * blocks), split);
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

// How a call is walked: `blocks` row blocks of 16 per wave, `waves` waves to a row block
// or kShared, `splits` workgroups to its keys.
struct Walk {
  int blocks, waves, splits;
};
Walk walk_for(int64_t pairs, int rows, int keys, int dim) {
  const int64_t tiles = ceil_div(keys, kTile), twos = pairs * ceil_div(rows, 32), plenty = dim == 64 ? 1024 : 512;
  Walk w{1, 4, 1};
  if (rows > 16 && (twos >= plenty || tiles >= 128 || (twos >= 128 && twos * tiles > 4096))) w.blocks = 2;
  if (w.blocks == 2 && twos >= plenty) {
    w.waves = kShared;
    return w;
  }
  const int64_t wgs = pairs * ceil_div(rows, 16 * w.blocks);
  if (tiles > (dim == 64 ? 24 : 16))
    w.splits = int(wgs > 128 && tiles >= 64 ? ceil_div(512, wgs) : std::max<int64_t>(1, std::min<int64_t>({256 / wgs, tiles / 4, 64})));
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
  w = walk_for(pairs, rows, a.max_kv, a.cache.head_dim);
  const int64_t blocks = ceil_div(rows, 16 * w.blocks * (w.waves == kShared ? 4 : 1));
  p.row_block_div = divisor(uint32_t(blocks));
  p.workgroups = pairs * blocks * w.splits;
  p.splits = w.splits;
  return p;
}

template <int D, int QB, int KW>
hipError_t launch(const AttnPlan& p, hipStream_t stream) {
  constexpr int bytes = KW == kShared ? int(sizeof(Tiles<D>)) : int(sizeof(Merge<D, QB, (KW > 0 ? KW : 1)>));
  if constexpr (bytes > 64 * 1024) {  // (two blocks of 128-dim rows)
    static LdsLimit limit;
    const hipError_t e = limit.raise(reinterpret_cast<const void*>(&paged_attention_kernel<D, QB, KW>), bytes);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((paged_attention_kernel<D, QB, KW>), dim3(unsigned(p.workgroups)), dim3(KW == kShared ? 256 : 64 * KW), bytes, stream, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.splits == 1) return e;
  if (p.splits > 16)
    hipLaunchKernelGGL((paged_attention_join_kernel<D, 4>), dim3(unsigned(p.all_rows)), dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((paged_attention_join_kernel<D, 1>), dim3(unsigned(ceil_div(p.all_rows, 4))), dim3(256), 0, stream, p);
  return hipGetLastError();
}

template <int D>
hipError_t launch_walk(const AttnPlan& p, const Walk& w, hipStream_t stream) {
  if (w.waves == kShared) return launch<D, 2, kShared>(p, stream);
  return w.blocks == 1 ? launch<D, 1, 4>(p, stream) : launch<D, 2, 4>(p, stream);
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
