// The int8 KV cache: rows quantised as they are written, and read back as fp16.
//
// A row x of D fp16 values (one token, one head) is held as D bytes c + 128 and
// one fp32 scale s:
//   s = fp32_rn(max|x| / 127), so 0 for a row of zeros (a scale that no other row's
//       weight is rounded against), NaN for a row with an infinity or NaN, so that what
//       reads it answers NaN instead of a number the row does not stand for (the bytes
//       of both are those of c = 0);
//   c = the whole number nearest x / s, ties to even, |c| <= 127.
// The quotient is decided exactly: t = x * rcp(s) is off by less than 2^-15, so
// rint(t) is right unless t lies that near half way between whole numbers; then q =
// rint(t) is at most one off, and x - q s is an fp32 number (a multiple of s's last
// place, at most about s), so one fma gives it without rounding and comparing it with
// s / 2 settles the last step.
//
// Layout (T = capacity, a multiple of 64), made for the attention kernel's
// matrix operands so that it loads 16 bytes per lane and moves nothing between
// lanes:
//   K  [slot][head][T / 16][D / 64][16 tokens][64 dims]
//   V  [slot][head][T / 64][D / 16][64 lanes][16 bytes]: byte i of lane l of
//      record d of a block of 64 tokens is token 16 (i / 4) + 4 (l / 16) + i % 4,
//      dim 16 d + l % 16
//   scales [slot][head][T], K's and V's apart.
// The stored byte is c + 128: 0x6400 | byte is then the fp16 number 1152 + c.
//
// Both directions are bound by memory where there is much of it: 8 prompts of up to 1000
// rows, 25 heads of 64, are quantised in 17 us (up to 51 MB in, 27 out), 65536 rows of 8
// heads of 128 read back in 74 us (403 MB, 5.4 TB/s); single tokens by the launch (32
// requests of 12 heads: 4.3 us, 4.2 back).
#include "common.hpp"
#include "kernels.hpp"

namespace tia {
namespace {

typedef unsigned short u16x8_t __attribute__((ext_vector_type(8)));

// 16 bytes at any even address (the device allows unaligned vector accesses).
__device__ __forceinline__ u16x8_t load_row8(const uint16_t* p) {
  u16x8_t r;
  __builtin_memcpy(&r, p, 16);
  return r;
}
__device__ __forceinline__ void store_row8(uint16_t* p, u16x8_t v) { __builtin_memcpy(p, &v, 16); }

// Largest |x| bits of a row whose pieces of 8 lie in LPR neighbouring lanes.
template <int LPR>
__device__ __forceinline__ unsigned row_top(u16x8_t x) {
  unsigned top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, unsigned(x[e]) & 0x7fffu);
#pragma unroll
  for (int o = 1; o < LPR; o <<= 1) top = max(top, unsigned(__shfl_xor(int(top), o, kWave)));
  return top;
}

struct RowScale {
  float s, inv;  // inv 0 for a row of zeros or with a non-finite value: every byte 128
};
__device__ __forceinline__ RowScale row_scale(unsigned top) {
  if (top >= 0x7c00u) return {__builtin_nanf(""), 0.f};
  if (top == 0) return {0.f, 0.f};
  const float s = h2f(uint16_t(top)) / 127.f;
  return {s, __builtin_amdgcn_rcpf(s)};
}

__device__ __forceinline__ float nearest(float x, RowScale r) {
  float q = rintf(x * r.inv);
  const float rest = 2.f * fmaf(-q, r.s, x);
  const bool odd = int(q) & 1;
  if (rest > r.s || (rest == r.s && odd)) q += 1.f;
  else if (rest < -r.s || (rest == -r.s && odd)) q -= 1.f;
  return q;
}
// The bytes of 8 values.
__device__ __forceinline__ uint64_t quantise(u16x8_t bits, RowScale r) {
  float q[8], close = 1.f;  // close: the least distance from half way
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float t = h2f(bits[e]) * r.inv;
    q[e] = rintf(t);
    close = fminf(close, fabsf(fabsf(t - q[e]) - 0.5f));
  }
  if (r.inv == 0.f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = 0.f;
  } else if (close < 0x1p-14f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = nearest(h2f(bits[e]), r);
  }
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e >> 2] = __builtin_amdgcn_cvt_pk_u8_f32(q[e] + 128.f, e & 3, w[e >> 2]);
  return uint64_t(w[1]) << 32 | w[0];
}

// Offsets of (token, dim) from the start of a slot's head.
__device__ __forceinline__ int64_t k_byte(int64_t t, int dim, int D) {
  return (t >> 4) * 16 * D + (dim >> 6) * 1024 + (t & 15) * 64 + (dim & 63);
}
__device__ __forceinline__ int64_t v_byte(int64_t t, int dim, int D) {
  const int r = int(t & 63);
  return (t >> 6) * 64 * D + (dim >> 4) * 1024 + ((dim & 15) + 16 * ((r >> 2) & 3)) * 16 + 4 * (r >> 4) + (r & 3);
}

// Whether a later request of the call writes token t of `slot` too: its row is
// then the one that stays, as if the requests were written one after another.
__device__ bool written_later(const KvAppendArgs& a, int b, int64_t t) {
  const int slot = a.slots[b];
  for (int o = b + 1; o < a.batch; ++o) {
    if (a.slots[o] != slot) continue;
    const int64_t n = a.lengths ? min(max(a.lengths[o], 0), a.rows) : a.rows;
    if (t >= a.positions[o] && t < int64_t(a.positions[o]) + n) return true;
  }
  return false;
}
// Whether any later request shares the slot (called by whole waves).
__device__ __forceinline__ bool slot_shared(const KvAppendArgs& a, int b, int slot) {
  for (int o = b + 1; o < a.batch; o += kWave) {
    const int at = o + int(threadIdx.x & 63);
    if (__ballot(at < a.batch && a.slots[at] == slot)) return true;
  }
  return false;
}

// A few rows per request (single tokens): D / 8 lanes per row, V's bytes stored
// one by one (they lie in other records).  One wave per 512 / D rows of a request.
template <int D>
__global__ __launch_bounds__(64) void append_rows_kernel(KvAppendArgs a) {
  constexpr int LPR = D / 8, RPW = 64 / LPR;
  const int b = int(blockIdx.y), lane = int(threadIdx.x), seg = lane % LPR;
  const int64_t row = int64_t(blockIdx.x) * RPW + lane / LPR;  // head * rows + i
  const int64_t count = int64_t(a.cache.kv_heads) * a.rows;
  const int64_t src = (int64_t(b) * count + min(row, count - 1)) * D + 8 * seg;
  const u16x8_t k = load_row8(a.k + src), v = load_row8(a.v + src);
  const int slot = a.slots[b], n = a.lengths ? a.lengths[b] : a.rows;
  const int head = int(row / a.rows), i = int(row - int64_t(head) * a.rows);
  const int64_t t = int64_t(a.positions[b]) + i;
  if (slot < 0 || slot >= a.cache.slots) return;
  bool live = row < count && i < n && t >= 0 && t < a.cache.capacity;
  if (slot_shared(a, b, slot)) live = live && !written_later(a, b, t);
  const unsigned ktop = row_top<LPR>(k), vtop = row_top<LPR>(v);
  if (!live) return;
  const RowScale kr = row_scale(ktop), vr = row_scale(vtop);
  const int64_t at = (int64_t(slot) * a.cache.kv_heads + head) * a.cache.capacity;
  const uint64_t kq = quantise(k, kr), vq = quantise(v, vr);
  uint8_t* vd = a.cache.v + at * D;
#pragma unroll
  for (int e = 0; e < 8; ++e) vd[v_byte(t, 8 * seg + e, D)] = uint8_t(vq >> (8 * e));
  *reinterpret_cast<uint64_t*>(a.cache.k + at * D + k_byte(t, 8 * seg, D)) = kq;
  if (seg == 0) {
    a.cache.k_scales[at + t] = kr.s;
    a.cache.v_scales[at + t] = vr.s;
  }
}

// Prompts: a workgroup takes the rows of one request and head that fall into one
// block of 64 tokens; V's bytes pass through LDS into whole 16-byte pieces of the
// block's records (pieces that hold other tokens too are stored byte by byte).
template <int D>
__global__ __launch_bounds__(256) void append_block_kernel(KvAppendArgs a) {
  constexpr int LPR = D / 8, RPP = 256 / LPR;
  __shared__ uint8_t vt[64][D + 4];
  __shared__ uint8_t lives[64];
  const int head = int(blockIdx.y), b = int(blockIdx.z), tid = int(threadIdx.x), seg = tid % LPR;
  const int slot = a.slots[b];
  const int n = a.lengths ? min(a.lengths[b], a.rows) : a.rows;
  const int64_t pos = a.positions[b];
  if (slot < 0 || slot >= a.cache.slots || n <= 0) return;
  const int64_t t0 = ((pos >> 6) + blockIdx.x) << 6;
  if (t0 < 0 || t0 >= a.cache.capacity || t0 >= pos + n) return;
  const bool shared = slot_shared(a, b, slot);
  const int64_t at = (int64_t(slot) * a.cache.kv_heads + head) * a.cache.capacity;
#pragma unroll
  for (int p = 0; p < 64 / RPP; ++p) {
    const int r = p * RPP + tid / LPR;
    const int64_t t = t0 + r, i = t - pos;
    bool live = i >= 0 && i < n;
    if (shared) live = live && !written_later(a, b, t);
    const int64_t src = ((int64_t(b) * a.cache.kv_heads + head) * a.rows + min(max(i, int64_t(0)), int64_t(n - 1))) * D + 8 * seg;
    const u16x8_t k = load_row8(a.k + src), v = load_row8(a.v + src);
    const RowScale kr = row_scale(row_top<LPR>(k)), vr = row_scale(row_top<LPR>(v));
    const uint64_t kq = quantise(k, kr), vq = quantise(v, vr);
    *reinterpret_cast<uint32_t*>(&vt[r][8 * seg]) = uint32_t(vq);
    *reinterpret_cast<uint32_t*>(&vt[r][8 * seg + 4]) = uint32_t(vq >> 32);
    if (seg == 0) lives[r] = live;
    if (live) {
      *reinterpret_cast<uint64_t*>(a.cache.k + at * D + k_byte(t, 8 * seg, D)) = kq;
      if (seg == 0) {
        a.cache.k_scales[at + t] = kr.s;
        a.cache.v_scales[at + t] = vr.s;
      }
    }
  }
  __syncthreads();
  uint8_t* vd = a.cache.v + (at + t0) * D;
#pragma unroll
  for (int piece = tid; piece < 4 * D; piece += 256) {
    const int d = 16 * (piece >> 6) + (piece & 15), g = (piece >> 4) & 3;
    uint32_t w[4];
    bool all = true;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      w[c] = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[c] |= uint32_t(vt[16 * c + 4 * g + i][d]) << (8 * i);
        all = all && lives[16 * c + 4 * g + i];
      }
    }
    if (all) {
      *reinterpret_cast<u32x4_t*>(vd + 16 * piece) = u32x4_t{w[0], w[1], w[2], w[3]};
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (lives[16 * c + 4 * g + i]) vd[16 * piece + 4 * c + i] = uint8_t(w[c] >> (8 * i));
    }
  }
}

// (+ 0: a byte that was never written, -128, times its scale of 0 is -0.)
__device__ __forceinline__ uint16_t value_of(unsigned byte, float s) { return f2h(float(int(byte) - 128) * s + 0.f); }

// Rows [0, rows) of every request: token positions[b] + i, zeros where i is past
// lengths[b] or the token is outside the cache.  A workgroup takes one request's,
// one head's rows of one block of 64 tokens.
template <int D>
__global__ __launch_bounds__(256) void read_kernel(KvReadArgs a) {
  constexpr int LPR = D / 8, RPP = 256 / LPR;
  __shared__ uint8_t vt[64][D + 4];
  const int head = int(blockIdx.y), b = int(blockIdx.z), tid = int(threadIdx.x), seg = tid % LPR;
  const int slot = a.slots[b];
  const int64_t pos = a.positions[b];
  const int64_t t0 = ((pos >> 6) + blockIdx.x) << 6;
  if (t0 >= pos + a.rows) return;
  const bool held = slot >= 0 && slot < a.cache.slots && t0 >= 0 && t0 < a.cache.capacity;
  const int n = held ? max(min(a.lengths ? a.lengths[b] : a.rows, a.rows), 0) : 0;
  const int64_t at = (int64_t(slot) * a.cache.kv_heads + head) * a.cache.capacity;
  if (n > 0 && t0 < pos + n) {  // (t0 may lie in front of pos: n = 0 alone does not say that)
    const uint8_t* vd = a.cache.v + (at + t0) * D;
#pragma unroll
    for (int piece = tid; piece < 4 * D; piece += 256) {
      const int d = 16 * (piece >> 6) + (piece & 15), g = (piece >> 4) & 3;
      const u32x4_t w = *reinterpret_cast<const u32x4_t*>(vd + 16 * piece);
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) vt[16 * c + 4 * g + i][d] = uint8_t(w[c] >> (8 * i));
    }
  }
  __syncthreads();
#pragma unroll
  for (int p = 0; p < 64 / RPP; ++p) {
    const int r = p * RPP + tid / LPR;
    const int64_t t = t0 + r, i = t - pos;
    if (i < 0 || i >= a.rows) continue;
    u16x8_t k = {}, v = {};
    if (i < n) {
      const uint64_t kq = *reinterpret_cast<const uint64_t*>(a.cache.k + at * D + k_byte(t, 8 * seg, D));
      const float ks = a.cache.k_scales[at + t], vs = a.cache.v_scales[at + t];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        k[e] = value_of(unsigned(kq >> (8 * e)) & 255u, ks);
        v[e] = value_of(vt[r][8 * seg + e], vs);
      }
    }
    const int64_t dst = ((int64_t(b) * a.cache.kv_heads + head) * a.rows + i) * D + 8 * seg;
    store_row8(a.k + dst, k);
    store_row8(a.v + dst, v);
  }
}

// Blocks of 64 tokens that `rows` rows from any position on can touch.
unsigned blocks_of(int rows) { return unsigned((int64_t(rows) + 62) / 64 + 1); }

}  // namespace

hipError_t kv_append_i8(const KvAppendArgs& a, hipStream_t stream) {
  const KvI8& c = a.cache;
  if (a.rows <= kKvAppendRowsMax) {
    const int per = 512 / c.head_dim;
    const dim3 grid(unsigned((int64_t(c.kv_heads) * a.rows + per - 1) / per), unsigned(a.batch));
    if (c.head_dim == 64) hipLaunchKernelGGL((append_rows_kernel<64>), grid, dim3(64), 0, stream, a);
    else hipLaunchKernelGGL((append_rows_kernel<128>), grid, dim3(64), 0, stream, a);
  } else {
    const dim3 grid(blocks_of(a.rows), unsigned(c.kv_heads), unsigned(a.batch));
    if (c.head_dim == 64) hipLaunchKernelGGL((append_block_kernel<64>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((append_block_kernel<128>), grid, dim3(256), 0, stream, a);
  }
  return hipGetLastError();
}

hipError_t kv_read_i8(const KvReadArgs& a, hipStream_t stream) {
  const KvI8& c = a.cache;
  const dim3 grid(blocks_of(a.rows), unsigned(c.kv_heads), unsigned(a.batch));
  if (c.head_dim == 64) hipLaunchKernelGGL((read_kernel<64>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((read_kernel<128>), grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace tia
