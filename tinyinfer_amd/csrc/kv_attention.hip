// Attention over the int8 KV cache for gfx950: single tokens, prompts, and a
// prefix that a batch shares, by one kernel.
//
//   o[r] = sum_j p_rj V_j / sum_j p_rj,  p_rj = 2^(x_rj - m_r),
//   x_rj = (q_r . c_j) * ks_j * D^-1/2 * log2 e,  V_j = vs_j * d_j
// with c, d the whole numbers that the cache holds (exact in fp16) and ks, vs the
// fp32 scales of token j: a key's scale is applied to its score, a value's to its
// probability, so neither c nor d is rounded.
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
// A workgroup's 4 waves take every fourth tile of 64 keys of one row block and
// merge their states (m, l, O) through LDS.  With few row blocks the keys are cut
// into splits as well, each split's state goes to the caller's workspace and a
// second kernel joins them.  A prefix is one such set of splits, its row blocks
// running over the whole batch: its keys are read once for all requests.
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"
#include "lds_limit.hpp"

namespace tia {
namespace {

constexpr int kTile = 64;   // keys per wave and step
constexpr int kWaves = 4;
constexpr float kNegInf = -__builtin_huge_valf();
// The reference of a row's exponents: 6 below its largest score when set, raised
// when a score is 14 above it.  Probabilities then lie around 2^6 and below 2^14:
// rounded to fp16, whose smallest normal number is 2^-14, a key 2^-20 times as
// heavy as the heaviest still keeps 11 bits.
constexpr float kBelow = 6.f, kRaise = 14.f;

struct AttnPlan {
  KvAttnArgs a;
  float scale;                   // D^-1/2 log2 e
  int group, rows;               // query heads per key head; rows of one request and key head
  int row_blocks, splits;        // of the requests' own keys
  int prefix_blocks, prefix_splits;
  int64_t own_wgs, prefix_wgs;
  int64_t all_rows;              // batch * heads * q_len
  bool parts;                    // states to the workspace, joined by the second kernel
};

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

// x times the value that lane N of this lane's row of 16 holds (the broadcast is an
// operand modifier of the multiplication).
template <int N>
__device__ __forceinline__ float mul_row_lane(float x, float of) {
  const float y = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, of), 0x150 + N, 0xF, 0xF, true));
  return x * y;
}
// x[kb][v] times lane 4 kb + v's value.
__device__ __forceinline__ void mul_row(float4_t (&x)[4], float of) {
#define TIA_MUL(kb, v) x[kb][v] = mul_row_lane<4 * kb + v>(x[kb][v], of);
#define TIA_MUL4(kb) TIA_MUL(kb, 0) TIA_MUL(kb, 1) TIA_MUL(kb, 2) TIA_MUL(kb, 3)
  TIA_MUL4(0) TIA_MUL4(1) TIA_MUL4(2) TIA_MUL4(3)
#undef TIA_MUL4
#undef TIA_MUL
}

template <int D, int QB>
struct Merge {
  float4_t acc[kWaves][QB * D / 16][64];
  float m[kWaves][QB][16], l[kWaves][QB][16];
};

// Row block `rb` of one set of keys.  PREFIX: rows run over the batch, key head
// `head`, the keys are the prefix's; else over request b's.
template <int D, int QB, bool PREFIX>
__device__ void attend(const AttnPlan& p, uint8_t* lds, int b0, int head, int rb, int split, int splits, int state) {
  const KvAttnArgs& a = p.a;
  const int lane = int(threadIdx.x & 63), wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
  const int j = lane & 15, g = lane >> 4;
  constexpr int ROWS = 16 * QB;
  const int64_t r0 = int64_t(rb) * ROWS;
  const int64_t row_count = PREFIX ? int64_t(a.batch) * p.rows : p.rows;

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
  int64_t row_id[QB];  // in q's order, -1 past the last row
  int end[QB];         // keys [0, end) are visible
#pragma unroll
  for (int u = 0; u < QB; ++u) {
    const int64_t r = r0 + 16 * u + j;
    const int b = PREFIX ? int(min(r, row_count - 1) / p.rows) : b0;
    const int rr = int(min(r, row_count - 1) - (PREFIX ? int64_t(b) * p.rows : 0));
    const int qi = rr / p.group, hg = rr - qi * p.group;
    row_id[u] = r < row_count ? (int64_t(b) * a.heads + int64_t(head) * p.group + hg) * a.q_len + qi : -1;
    const int ql = a.q_lengths ? min(max(a.q_lengths[b], 0), a.q_len) : a.q_len;
    int64_t e = kv;
    if (!PREFIX && a.causal) e = min(e, (a.offsets ? int64_t(a.offsets[b]) : int64_t(kv) - ql) + qi + 1);
    end[u] = r < row_count && qi < ql ? int(max(e, int64_t(0))) : 0;
  }
  // Keys that some row of the block sees, and keys that every row with a query
  // sees (a row without one may compute anything: it is cleared at the end).
  int last, first;
  if constexpr (PREFIX) {
    last = first = kv;
  } else {
    const int ql = a.q_lengths ? min(max(a.q_lengths[b0], 0), a.q_len) : a.q_len;
    const int q_first = int(r0 / p.group), q_last = min(int((min(r0 + ROWS, row_count) - 1) / p.group), ql - 1);
    const int64_t off = a.offsets ? int64_t(a.offsets[b0]) : int64_t(kv) - ql;
    const auto seen = [&](int qi) { return int(max(a.causal ? min(int64_t(kv), off + qi + 1) : int64_t(kv), int64_t(0))); };
    last = q_last < q_first ? 0 : seen(q_last);
    first = q_last < q_first ? 0 : seen(q_first);
  }
  const int tiles = (last + kTile - 1) / kTile, per = (tiles + splits - 1) / splits;
  const int t_end = min(tiles, (split + 1) * per);
  int t = split * per + wave;

  const int64_t base = (int64_t(slot) * a.cache.kv_heads + head) * a.cache.capacity;
  const uint8_t* kp = a.cache.k + base * D + j * D + 16 * g;
  const uint8_t* vp = a.cache.v + base * D + lane * 16;
  // Lane (j, g) holds the scales of the tile's key 16 (j / 4) + 4 g + j % 4: of row g's
  // 16 scores of a tile, number 4 kb + v in order, lane 4 kb + v has the scale.
  const int my_key = 16 * (j >> 2) + 4 * g + (j & 3);
  const float* ksp = a.cache.k_scales + base + my_key;
  const float* vsp = a.cache.v_scales + base + my_key;
  u32x4_t kr[4][D / 64], vr[D / 16];
  float ksr = 0.f, vsr = 0.f;
  auto load_k = [&](int tt) {
    const uint8_t* at = kp + int64_t(tt) * (kTile * D);
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int c = 0; c < D / 64; ++c) kr[kb][c] = *reinterpret_cast<const u32x4_t*>(at + 16 * kb * D + 64 * c);
    ksr = ksp[int64_t(tt) * kTile];
  };
  auto load_v = [&](int tt) {
    const uint8_t* at = vp + int64_t(tt) * (kTile * D);
#pragma unroll
    for (int d = 0; d < D / 16; ++d) vr[d] = *reinterpret_cast<const u32x4_t*>(at + 1024 * d);
    vsr = vsp[int64_t(tt) * kTile];
  };
  if (t < t_end) {
    load_k(t);
    load_v(t);
  }

  // Step (c, s) of a dot product takes dims 64 c + 16 g + 8 s .. + 7 from lane (., g).
  half8_t qf[QB][D / 32];
#pragma unroll
  for (int u = 0; u < QB; ++u) {
    const uint16_t* qp = a.q + max(row_id[u], int64_t(0)) * D + 16 * g;
#pragma unroll
    for (int c = 0; c < D / 64; ++c)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        half8_t x;
        __builtin_memcpy(&x, qp + 64 * c + 8 * s, 16);
        qf[u][2 * c + s] = end[u] > 0 ? x : half8_t{};
      }
  }

  float m[QB], l[QB];
  float4_t acc[QB][D / 16];
#pragma unroll
  for (int u = 0; u < QB; ++u) {
    m[u] = kNegInf;
    l[u] = 0.f;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) acc[u][d] = float4_t{0.f, 0.f, 0.f, 0.f};
  }
  // O is kept in units of `unit`, a power of two not below any value scale seen:
  // the weight p * vs / unit that is rounded to fp16 is then at most p.
  float unit = 0.f, inv_unit = 1.f;

  // One tile; MORE: this wave has a next one, whose loads are issued as the registers fall free.
  auto step = [&](auto more_c, int tt) {
    constexpr bool MORE = decltype(more_c)::value;
    const bool full = (tt + 1) * kTile <= first;
    float4_t sc[QB][4];
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
#pragma unroll
      for (int u = 0; u < QB; ++u) sc[u][kb] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < D / 64; ++c)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const half8_t kf = widen8(kr[kb][c][2 * s], kr[kb][c][2 * s + 1]);
#pragma unroll
          for (int u = 0; u < QB; ++u)
            sc[u][kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[u][2 * c + s], sc[u][kb], 0, 0, 0);
        }
      __builtin_amdgcn_sched_barrier(0);
    }
    const float ck = ksr * p.scale;
    // (Past the last key any row sees, scales may be anything.)
    const float vs = tt * kTile + my_key < last ? vsr : 0.f;
    if constexpr (MORE) load_k(tt + kWaves);
    if (__ballot(vs > unit)) {
      const float top = wave_max(vs);
      const float raised = __builtin_amdgcn_ldexpf(1.f, __builtin_amdgcn_frexp_expf(top));  // > top
      const float f = unit / raised;
      unit = raised;
      inv_unit = 1.f / raised;
#pragma unroll
      for (int u = 0; u < QB; ++u)
#pragma unroll
        for (int d = 0; d < D / 16; ++d) acc[u][d] *= f;
    }
    const float wv = vs * inv_unit;
    half8_t pp[QB][2];
#pragma unroll
    for (int u = 0; u < QB; ++u) {
      mul_row(sc[u], ck);
      const int lim = end[u] - tt * kTile - 4 * g;  // key 16 kb + v of this lane is visible iff < lim
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
      if (__ballot(high > m[u] + kRaise)) {
        high = fmaxf(high, __shfl_xor(high, 16, 64));
        high = fmaxf(high, __shfl_xor(high, 32, 64));
        const float nm = high > m[u] + kRaise ? high - kBelow : m[u];
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
      mul_row(sc[u], wv);
      if (!full) mask(0.f);  // (0 times a scale that is not finite)
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int v = 0; v < 4; ++v)
          pp[u][kb >> 1][4 * (kb & 1) + v] = f16(sc[u][kb][v]);
    }
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const half8_t vf = widen8(vr[d][2 * c], vr[d][2 * c + 1]);
#pragma unroll
        for (int u = 0; u < QB; ++u) acc[u][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pp[u][c], acc[u][d], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (MORE) load_v(tt + kWaves);
  };
  for (; t + kWaves < t_end; t += kWaves) step(std::true_type{}, t);
  if (t < t_end) step(std::false_type{}, t);

  // The waves' states meet in LDS; wave w joins every fourth (block, 16 dims).
  auto& mg = *reinterpret_cast<Merge<D, QB>*>(lds);
#pragma unroll
  for (int u = 0; u < QB; ++u) {
    l[u] += __shfl_xor(l[u], 16, 64);
    l[u] += __shfl_xor(l[u], 32, 64);
    if (end[u] == 0) l[u] = 0.f;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) mg.acc[wave][u * (D / 16) + d][lane] = acc[u][d] * unit;
    if (g == 0) {
      mg.m[wave][u][j] = m[u];
      mg.l[wave][u][j] = l[u];
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < QB; ++u) {
    float top = kNegInf, total = 0.f, f[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = mg.l[w][u][j] == 0.f ? top : fmaxf(top, mg.m[w][u][j]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float lw = mg.l[w][u][j];
      f[w] = lw == 0.f ? 0.f : __builtin_amdgcn_exp2f(mg.m[w][u][j] - top);
      total += lw * f[w];
    }
    if (row_id[u] < 0) continue;
    const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
    for (int d0 = 0; d0 < D / 16; d0 += kWaves) {
      const int d = d0 + wave;
      float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float4_t x = mg.acc[w][u * (D / 16) + d][lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = f[w] == 0.f ? o[e] : fmaf(x[e], f[w], o[e]);
      }
      if (p.parts) {
        const int64_t at = int64_t(state) * p.all_rows + row_id[u];
        if (total != 0.f) *reinterpret_cast<float4_t*>(a.workspace + at * D + 16 * d + 4 * g) = o;
      } else {
        half4_t y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = f16r(total == 0.f ? 0.f : o[e] * inv);
        __builtin_memcpy(a.out + row_id[u] * D + 16 * d + 4 * g, &y, 8);
      }
    }
    if (p.parts && wave == 0 && g == 0) {
      const int64_t states = int64_t(p.splits + p.prefix_splits) * p.all_rows;
      float* ml = a.workspace + states * D + 2 * (int64_t(state) * p.all_rows + row_id[u]);
      ml[0] = top;
      ml[1] = total;
    }
  }
}

// Waves per SIMD that the registers are budgeted for.
constexpr int waves_for(int dim, int qb) { return dim == 64 ? (qb == 1 ? 4 : qb == 2 ? 3 : 2) : (qb == 1 ? 3 : 2); }

template <int D, int QB, int PB>
__global__ __launch_bounds__(64 * kWaves, waves_for(D, QB > PB ? QB : PB)) void kv_attention_kernel(AttnPlan p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  int64_t id = blockIdx.x;
  const int heads = p.a.cache.kv_heads;
  if constexpr (PB > 0) {
    if (id < p.prefix_wgs) {
      const int head = int(id % heads);
      id /= heads;
      attend<D, PB, true>(p, lds, 0, head, int(id % p.prefix_blocks), int(id / p.prefix_blocks), p.prefix_splits,
                          p.splits + int(id / p.prefix_blocks));
      return;
    }
    id -= p.prefix_wgs;
  }
  const int64_t bh = int64_t(p.a.batch) * heads;
  const int at = int(id % bh);
  const int rest = int(id / bh);
  attend<D, QB, false>(p, lds, at / heads, at % heads, p.row_blocks - 1 - rest % p.row_blocks, rest / p.row_blocks,
                       p.splits, rest / p.row_blocks);
}

// One wave per row joins its splits' states.
template <int D>
__global__ __launch_bounds__(256) void kv_attention_join_kernel(AttnPlan p) {
  constexpr int LPR = D / 4, PARTS = 64 / LPR;
  const int lane = int(threadIdx.x & 63), part = lane / LPR, at = 4 * (lane % LPR);
  const int64_t row = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= p.all_rows) return;
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
  for (int s = part; s < states; s += PARTS) {
    const float* x = ml + 2 * (s * p.all_rows + row);
    const float lw = x[1];
    if (lw == 0.f) continue;
    const float f = __builtin_amdgcn_exp2f(x[0] - top);
    const float4_t y = *reinterpret_cast<const float4_t*>(p.a.workspace + (s * p.all_rows + row) * D + at);
    total = fmaf(lw, f, total);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf(y[e], f, o[e]);
  }
#pragma unroll
  for (int x = LPR; x < 64; x <<= 1) {
    total += __shfl_xor(total, x, 64);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], x, 64);
  }
  if (part != 0) return;
  const float inv = total == 0.f ? 0.f : 1.f / total;
  half4_t y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = f16r(total == 0.f ? 0.f : o[e] * inv);
  __builtin_memcpy(p.a.out + row * D + at, &y, 8);
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// 16-row blocks per wave: as many as the rows fill, up to what the registers hold.
int blocks_for(int64_t rows, int dim) { return rows <= 16 ? 1 : rows <= 32 || dim == 128 ? 2 : 4; }

constexpr int64_t kWantedWgs = 1024;

int splits_for(int64_t wgs, int keys) {
  const int64_t tiles = ceil_div(keys, kTile);
  return int(std::max<int64_t>(1, std::min(ceil_div(kWantedWgs, wgs), tiles / kWaves)));
}

AttnPlan plan_of(const KvAttnArgs& a, int& qb, int& pb) {
  AttnPlan p{};
  p.a = a;
  const int dim = a.cache.head_dim;
  p.scale = float(1.4426950408889634 / __builtin_sqrt(double(dim)));
  p.group = a.heads / a.cache.kv_heads;
  p.rows = p.group * a.q_len;
  p.all_rows = int64_t(a.batch) * a.heads * a.q_len;
  qb = blocks_for(p.rows, dim);
  p.row_blocks = int(ceil_div(p.rows, 16 * qb));
  p.own_wgs = int64_t(a.batch) * a.cache.kv_heads * p.row_blocks;
  p.splits = splits_for(p.own_wgs, a.max_kv);
  p.own_wgs *= p.splits;
  pb = 0;
  if (a.prefix_len > 0) {
    pb = blocks_for(int64_t(a.batch) * p.rows, dim);
    p.prefix_blocks = int(ceil_div(int64_t(a.batch) * p.rows, 16 * pb));
    p.prefix_wgs = int64_t(a.cache.kv_heads) * p.prefix_blocks;
    p.prefix_splits = splits_for(p.prefix_wgs, a.prefix_len);
    p.prefix_wgs *= p.prefix_splits;
  }
  p.parts = p.splits + p.prefix_splits > 1;
  return p;
}

template <int D, int QB, int PB>
hipError_t launch(const AttnPlan& p, hipStream_t stream) {
  constexpr int bytes = int(std::max(sizeof(Merge<D, QB>), PB > 0 ? sizeof(Merge<D, (PB > 0 ? PB : 1)>) : size_t(0)));
  static LdsLimit limit;
  if (bytes > 64 * 1024) {
    const hipError_t e = limit.raise(reinterpret_cast<const void*>(&kv_attention_kernel<D, QB, PB>), bytes);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((kv_attention_kernel<D, QB, PB>), dim3(unsigned(p.prefix_wgs + p.own_wgs)), dim3(64 * kWaves), bytes,
                     stream, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !p.parts) return e;
  hipLaunchKernelGGL((kv_attention_join_kernel<D>), dim3(unsigned(ceil_div(p.all_rows, 4))), dim3(256), 0, stream, p);
  return hipGetLastError();
}

template <int D, int QB>
hipError_t launch_prefix(const AttnPlan& p, int pb, hipStream_t stream) {
  if (pb == 0) return launch<D, QB, 0>(p, stream);
  if (pb == 1) return launch<D, QB, 1>(p, stream);
  if constexpr (D == 64)
    if (pb == 4) return launch<D, QB, 4>(p, stream);
  return launch<D, QB, 2>(p, stream);
}

template <int D>
hipError_t launch_blocks(const AttnPlan& p, int qb, int pb, hipStream_t stream) {
  if (qb == 1) return launch_prefix<D, 1>(p, pb, stream);
  if constexpr (D == 64)
    if (qb == 4) return launch_prefix<D, 4>(p, pb, stream);
  return launch_prefix<D, 2>(p, pb, stream);
}

}  // namespace

int64_t kv_attention_workspace(const KvAttnArgs& a) {
  int qb, pb;
  const AttnPlan p = plan_of(a, qb, pb);
  return p.parts ? int64_t(p.splits + p.prefix_splits) * p.all_rows * (a.cache.head_dim + 2) * 4 : 0;
}

hipError_t kv_attention(const KvAttnArgs& a, hipStream_t stream) {
  int qb, pb;
  const AttnPlan p = plan_of(a, qb, pb);
  return a.cache.head_dim == 64 ? launch_blocks<64>(p, qb, pb, stream) : launch_blocks<128>(p, qb, pb, stream);
}

}  // namespace tia
