// One token per row of logits from a given random number, with temperature,
// top-k, top-p and min-p.
//
// Order of a row's tokens: logit descending, index ascending.  w = exp((logit -
// max) / T).  Kept are the first k tokens; of these the shortest run from the
// front whose mass reaches top_p of theirs; of these the tokens with w >= min_p;
// the first token always.  The answer is the first token whose cumulative mass
// exceeds u times the mass of the kept ones.
//
// All three filters keep a run from the front, so nothing is sorted: a histogram
// of (count, mass) over the distance from the maximum finds the bin in which a
// count or a mass is reached, and only that bin's tokens are ordered.  Masses are
// whole numbers of 2^-44 of the heaviest token's, computed from 64-bit
// exponentials: their sums are the same in any order, so an answer depends on
// its row alone, and cumulative masses are right to about 1e-12, so a token is
// the one that 64-bit arithmetic gives.  A token lighter than 2^-45 counts as 0.
//
// One workgroup per row: its passes after the first read the row from cache.
#include "common.hpp"
#include "kernels.hpp"

namespace tia {
namespace {

constexpr int kThreads = 1024, kBins = 2048, kList = 512;
constexpr double kUnit = 17592186044416.0;  // 2^44
constexpr double kPerNat = 64.0;            // bins per unit of (max - logit) / T
constexpr float kNegInf = -__builtin_huge_valf();
constexpr int kNoToken = 0x7fffffff;

typedef unsigned long long u64;

struct Bins {
  u64 mass[kBins];      // then: mass in front of the bin
  unsigned count[kBins];  // then: tokens in front of the bin
};
struct SampleLds {
  Bins all, sub;
  u64 key[kList], w[kList];
  u64 wave_mass[kThreads / 64];
  unsigned wave_count[kThreads / 64];
  float wave_max[kThreads / 64];
  int wave_at[kThreads / 64];
  u64 total_mass, low, high, answer_key, answer_mass;
  unsigned total_count, list_count;
  int bin;
};

// 64-bit key whose ascending order is the row's: value descending, then index.
__device__ __forceinline__ u64 order_key(float x, int i) {
  const unsigned b = __builtin_bit_cast(unsigned, x + 0.f);  // -0 orders as 0
  const unsigned up = b & 0x80000000u ? ~b : b | 0x80000000u;
  return u64(~up) << 32 | unsigned(i);
}

template <typename T>
struct Row {
  const T* p;
  int n;
  // f(value, index) for every token of the row.
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    constexpr int W = 16 / sizeof(T);
    for (int i = int(threadIdx.x) * W; i < n; i += kThreads * W) {
      if (i + W <= n) {
        T x[W];
        __builtin_memcpy(x, p + i, 16);
#pragma unroll
        for (int e = 0; e < W; ++e) f(float(x[e]), i + e);
      } else {
        for (int e = i; e < n; ++e) f(float(p[e]), e);
      }
    }
  }
};

struct Scale {
  double top, per;  // max, 1 / T
  __device__ __forceinline__ double distance(float x) const { return (top - double(x)) * per; }
};
// Bin of a distance; kBins where its token weighs nothing.
__device__ __forceinline__ int bin_of(double d) {
  const double at = d * kPerNat;
  return at < double(kBins) ? int(at) : kBins;  // (NaN: kBins)
}
__device__ __forceinline__ u64 mass_of(double e) { return u64(e * kUnit + 0.5); }

// Exclusive sums over the bins, totals in total_mass and total_count.
__device__ void scan(SampleLds& s, Bins& b) {
  const int t = int(threadIdx.x), lane = t & 63, wave = t >> 6;
  __syncthreads();
  u64 m = b.mass[2 * t] + b.mass[2 * t + 1];
  unsigned c = b.count[2 * t] + b.count[2 * t + 1];
  u64 mi = m;
  unsigned ci = c;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 mu = __shfl_up(mi, o, 64);
    const unsigned cu = __shfl_up(ci, o, 64);
    if (lane >= o) {
      mi += mu;
      ci += cu;
    }
  }
  if (lane == 63) {
    s.wave_mass[wave] = mi;
    s.wave_count[wave] = ci;
  }
  __syncthreads();
  u64 mb = 0;
  unsigned cb = 0;
  for (int w = 0; w < wave; ++w) {
    mb += s.wave_mass[w];
    cb += s.wave_count[w];
  }
  const u64 m0 = b.mass[2 * t];
  const unsigned c0 = b.count[2 * t];
  b.mass[2 * t] = mb + mi - m;
  b.mass[2 * t + 1] = mb + mi - m + m0;
  b.count[2 * t] = cb + ci - c;
  b.count[2 * t + 1] = cb + ci - c + c0;
  if (t == kThreads - 1) {
    s.total_mass = mb + mi;
    s.total_count = cb + ci;
  }
  __syncthreads();
}

// What a position is asked by: the first token whose count or mass, with all in
// front of it, reaches `goal` (goal >= 1, and at most the total).
struct Goal {
  bool by_count;
  u64 goal;
};
struct Place {
  u64 mass;        // of the tokens up to this one
  unsigned count;  // of the same
  u64 key;
};

__device__ __forceinline__ void clear(Bins& b) {
  for (int i = int(threadIdx.x); i < kBins; i += kThreads) {
    b.mass[i] = 0;
    b.count[i] = 0;
  }
}

// The last bin in front of which the goal is not yet reached, in s.bin.
__device__ void find_bin(SampleLds& s, const Bins& b, const Goal& g, u64 mass0, unsigned count0, u64 mass_all,
                         unsigned count_all) {
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = 2 * int(threadIdx.x) + e;
    const u64 before = g.by_count ? count0 + u64(b.count[i]) : mass0 + b.mass[i];
    const u64 after = i + 1 < kBins ? (g.by_count ? count0 + u64(b.count[i + 1]) : mass0 + b.mass[i + 1])
                                    : (g.by_count ? count0 + u64(count_all) : mass0 + mass_all);
    if (before < g.goal && g.goal <= after) s.bin = i;
  }
  __syncthreads();
}

template <typename T>
__device__ Place locate(SampleLds& s, const Row<T>& row, const Scale& sc, const Goal& g, u64 mass_all, unsigned count_all) {
  find_bin(s, s.all, g, 0, 0, mass_all, count_all);
  const int bin = s.bin;
  u64 mass0 = s.all.mass[bin];
  unsigned count0 = s.all.count[bin];
  unsigned n = (bin + 1 < kBins ? s.all.count[bin + 1] : count_all) - count0;
  u64 low = 0, high = ~u64(0);
  if (n > kList) {
    // A crowded bin: its keys' range, cut into kBins runs of equal width until
    // one run's tokens fit the list.  (Keys are distinct, so this ends.)
    if (threadIdx.x == 0) {
      s.low = ~u64(0);
      s.high = 0;
    }
    __syncthreads();
    u64 lo = ~u64(0), hi = 0;
    row.each([&](float x, int i) {
      if (bin_of(sc.distance(x)) != bin) return;
      const u64 k = order_key(x, i);
      lo = min(lo, k);
      hi = max(hi, k);
    });
    atomicMin(&s.low, lo);
    atomicMax(&s.high, hi);
    __syncthreads();
    low = s.low;
    high = s.high;
    while (n > kList) {
      int shift = 0;
      while (((high - low) >> shift) >= kBins) ++shift;
      __syncthreads();
      clear(s.sub);
      __syncthreads();
      row.each([&](float x, int i) {
        const double d = sc.distance(x);
        if (bin_of(d) != bin) return;
        const u64 k = order_key(x, i);
        if (k < low || k > high) return;
        const int at = int((k - low) >> shift);
        atomicAdd(&s.sub.mass[at], mass_of(exp(-d)));
        atomicAdd(&s.sub.count[at], 1u);
      });
      scan(s, s.sub);
      const u64 m_all = s.total_mass;
      const unsigned c_all = s.total_count;
      find_bin(s, s.sub, g, mass0, count0, m_all, c_all);
      const int at = s.bin;
      n = (at + 1 < kBins ? s.sub.count[at + 1] : c_all) - s.sub.count[at];
      mass0 += s.sub.mass[at];
      count0 += s.sub.count[at];
      low += u64(at) << shift;
      high = min(high, low + ((u64(1) << shift) - 1));
      __syncthreads();
    }
  }
  // The list: every token of the run, each ranked by all the others.
  if (threadIdx.x == 0) s.list_count = 0;
  __syncthreads();
  row.each([&](float x, int i) {
    const double d = sc.distance(x);
    if (bin_of(d) != bin) return;
    const u64 k = order_key(x, i);
    if (k < low || k > high) return;
    const unsigned at = atomicAdd(&s.list_count, 1u);
    if (at < kList) {
      s.key[at] = k;
      s.w[at] = mass_of(exp(-d));
    }
  });
  __syncthreads();
  const unsigned t = threadIdx.x;
  if (t < min(n, unsigned(kList))) {
    const u64 k = s.key[t], w = s.w[t];
    u64 before = mass0;
    unsigned rank = count0;
    for (unsigned o = 0; o < n; ++o)
      if (s.key[o] < k) {
        before += s.w[o];
        ++rank;
      }
    const u64 b = g.by_count ? rank : before, a = g.by_count ? rank + 1 : before + w;
    if (b < g.goal && g.goal <= a) {
      s.answer_key = k;
      s.answer_mass = before + w;
      s.total_count = rank + 1;
    }
  }
  __syncthreads();
  const Place got{s.answer_mass, s.total_count, s.answer_key};
  __syncthreads();
  return got;
}

// floor(f * m) for 0 <= f < 1, exact: f is a 24-bit number times a power of two.
__device__ __forceinline__ u64 part_of(float f, u64 m, bool& whole) {
  // f * 2^64 as a whole number (what lies below 2^-64 counts as 0).
  const u64 fx = f > 0.f ? u64(ldexp(double(f), 64)) : 0;
  whole = fx * m == 0;
  return __umul64hi(fx, m);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs a) {
  __shared__ SampleLds s;
  const int b = int(blockIdx.x), t = int(threadIdx.x);
  const Row<T> row{static_cast<const T*>(a.logits) + int64_t(b) * a.vocab, a.vocab};
  const float temp = a.temperature ? a.temperature[b] : a.temperature_all;
  const int top_k = a.top_k ? a.top_k[b] : a.top_k_all;
  const float top_p = a.top_p ? a.top_p[b] : a.top_p_all, min_p = a.min_p ? a.min_p[b] : a.min_p_all;
  float u = a.uniforms[b];
  u = u > 0.f ? fminf(u, 0.99999994f) : 0.f;

  clear(s.all);
  float bv = kNegInf;
  int bi = kNoToken;
  row.each([&](float x, int i) {
    if (x > bv) {
      bv = x;
      bi = i;
    }
  });
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float ov = __shfl_xor(bv, o, 64);
    const int oi = __shfl_xor(bi, o, 64);
    amax_merge(bv, bi, ov, oi);
  }
  if ((t & 63) == 0) {
    s.wave_max[t >> 6] = bv;
    s.wave_at[t >> 6] = bi;
  }
  __syncthreads();
  for (int w = 0; w < kThreads / 64; ++w) amax_merge(bv, bi, s.wave_max[w], s.wave_at[w]);
  if (bi == kNoToken || !(temp > 0.f) || bv == -kNegInf) {
    // No token above -inf, or the greedy one.
    if (t == 0) {
      a.tokens[b] = bi;
      a.probs[b] = bi == kNoToken ? 0.f : 1.f;
    }
    return;
  }
  const Scale sc{double(bv), 1.0 / double(temp)};
  u64 min_mass = 0;
  unsigned min_count = 0;
  const bool use_min = min_p > 0.f;
  row.each([&](float x, int) {
    const double d = sc.distance(x);
    const int at = bin_of(d);
    if (at >= kBins) return;
    const double e = exp(-d);
    const u64 w = mass_of(e);
    atomicAdd(&s.all.mass[at], w);
    atomicAdd(&s.all.count[at], 1u);
    if (use_min && e >= double(min_p)) {
      min_mass += w;
      ++min_count;
    }
  });
  scan(s, s.all);
  const u64 mass_all = s.total_mass;
  const unsigned count_all = s.total_count;

  // The kept run: its length and mass.
  u64 kept = mass_all, k_mass = mass_all;
  unsigned length = count_all;
  if (top_k > 0 && unsigned(top_k) < count_all) {
    const Place p = locate(s, row, sc, Goal{true, u64(top_k)}, mass_all, count_all);
    kept = k_mass = p.mass;
    length = p.count;
  }
  if (top_p < 1.f) {
    // The last token kept is the first with cumulative mass >= top_p * k_mass.
    bool whole;
    u64 goal = part_of(top_p, k_mass, whole);
    goal = max(whole ? goal : goal + 1, u64(1));
    const Place p = locate(s, row, sc, Goal{false, goal}, mass_all, count_all);
    kept = p.mass;
    length = p.count;
  }
  if (use_min) {
    __syncthreads();
    if (t == 0) {
      s.total_mass = 0;
      s.total_count = 0;
    }
    __syncthreads();
    atomicAdd(&s.total_mass, min_mass);
    atomicAdd(&s.total_count, min_count);
    __syncthreads();
    const unsigned n = s.total_count;
    const u64 m = s.total_mass;
    __syncthreads();
    if (n < length) {
      kept = n == 0 ? mass_of(1.0) : m;  // min_p above 1: the first token
    }
  }
  bool whole;
  const Place p = locate(s, row, sc, Goal{false, part_of(u, kept, whole) + 1}, mass_all, count_all);
  if (t == 0) {
    const int token = int(p.key & 0xffffffffu);
    a.tokens[b] = token;
    a.probs[b] = float(exp(-sc.distance(float(row.p[token]))) * kUnit / double(kept));
  }
}

}  // namespace

hipError_t sample(const SampleArgs& a, hipStream_t stream) {
  const dim3 grid(unsigned(a.batch)), block(kThreads);
  if (a.f32) hipLaunchKernelGGL((sample_kernel<float>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((sample_kernel<f16>), grid, block, 0, stream, a);
  return hipGetLastError();
}

}  // namespace tia
