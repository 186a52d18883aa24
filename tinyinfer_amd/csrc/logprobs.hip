// Log probabilities of given tokens, a row's entropy and its likeliest tokens.
//
//   m = max x,  Z = sum e^(x - m),  log p(t) = x_t - m - log Z,
//   H = -sum p log p = log Z - (sum e^(x - m) (x - m)) / Z
//
// One workgroup per row reads it once.  A thread keeps the largest x it has met, how many
// times, the sum of e^(x - m) over the others and sum e^(x - m) (x - m): a likely token's
// log probability, log1p of a small sum, and a sure row's entropy keep their digits, and a
// larger maximum rescales three numbers.  Tokens are ordered by logit, ties by index.  The
// alternatives come from a list of the tokens at or above a bar that `top` tokens reach for
// certain: of the threads' largest first tokens, the least one that is among the r largest of
// its wave, where r times the waves are `top` or more.  Where the list does not hold them
// (many equal logits, rising ones) the range of the tokens above the bar is cut into runs
// and read again until it does.
//
// NaN logits count as -inf.  A row with a +inf has all its probability on the first one, a
// row without a logit above -inf none anywhere: log probabilities of -inf, entropy 0.
#include "common.hpp"
#include "kernels.hpp"

namespace tia {
namespace {

typedef unsigned long long u64;
constexpr int kNoToken = 0x7fffffff;
constexpr float kNegInf = -__builtin_huge_valf(), kLog2e = 1.4426950408889634f;
constexpr int kList = 1024, kRuns = 2048;

// 64-bit key whose descending order is the row's: value, then the lower index.  Never 0.
__device__ __forceinline__ u64 key_of(float x, int i) {
  const unsigned b = __builtin_bit_cast(unsigned, x + 0.f);  // -0 orders as 0
  const unsigned up = b & 0x80000000u ? ~b : b | 0x80000000u;
  return u64(up) << 32 | unsigned(~i);
}
__device__ __forceinline__ float value_of(u64 key) {
  const unsigned up = unsigned(key >> 32);
  return __builtin_bit_cast(float, up & 0x80000000u ? up & 0x7fffffffu : ~up);
}
__device__ __forceinline__ int index_of(u64 key) { return int(~unsigned(key)); }

__device__ __forceinline__ u64 wave_max_key(u64 v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const u64 w = __shfl_xor(v, o, 64);
    v = v > w ? v : w;
  }
  return v;
}

// What a thread knows of the tokens it has met: their maximum m, how many there are of it,
// and over the others rest = sum e^(x - m), spread = sum e^(x - m) (x - m).
struct Stats {
  float m, count, rest, spread;
  // To a maximum of at least this one's.  (Differences end at -200, where e^ is 0.)
  __device__ __forceinline__ void raise(float to) {
    const float d = fmaxf(m - to, -200.f), f = m == to ? 1.f : __builtin_amdgcn_exp2f(d * kLog2e);
    spread = m == to ? spread : f * fmaf(d, rest + count, spread);
    rest = m == to ? rest : f * (rest + count);
    count = m == to ? count : 0.f;
    m = to;
  }
  __device__ __forceinline__ void join(Stats o) {
    const float to = fmaxf(m, o.m);
    raise(to);
    o.raise(to);
    count += o.count;
    rest += o.rest;
    spread += o.spread;
  }
  __device__ __forceinline__ Stats from(int lane) const {
    return {__shfl_xor(m, lane, 64), __shfl_xor(count, lane, 64), __shfl_xor(rest, lane, 64), __shfl_xor(spread, lane, 64)};
  }
  template <int N>
  __device__ __forceinline__ void add(const float (&x)[N]) {
    float high = kNegInf;
#pragma unroll
    for (int i = 0; i < N; ++i) high = fmaxf(high, x[i]);  // (NaN loses)
    const bool equal = __ballot(high >= m);
    raise(fmaxf(m, high));
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float d = fmaxf(x[i] - m, -200.f);  // (NaN and -inf too: e^-200 is 0)
      float e = __builtin_amdgcn_exp2f(d * kLog2e);
      spread = fmaf(d, e, spread);
      if (equal) {
        count += x[i] == m ? 1.f : 0.f;
        e = x[i] == m ? 0.f : e;
      }
      rest += e;
    }
  }
};

template <typename T>
struct Vec {
  static constexpr int W = 16 / int(sizeof(T));
  typedef T type __attribute__((ext_vector_type(W)));
};

template <typename T, int THREADS>
struct Lds {
  u64 list[kList];
  u64 bar[THREADS / 64];
  Stats stats[THREADS / 64];
  unsigned run[kRuns];
  unsigned count, pick, above;
  u64 low, high;
};

// The row as threads see it: token `head` on starts a 16-byte boundary, vector v of it is
// tokens head + W v ..; the few in front and behind are one token each of the first threads.
template <typename T, int THREADS>
struct Row {
  static constexpr int W = Vec<T>::W, A = 4;  // vectors of a thread at a time
  const T* p;
  int n, head, vectors;
  __device__ __forceinline__ Row(const T* row, int length) : p(row), n(length) {
    head = min(n, int(-(reinterpret_cast<uintptr_t>(row) / sizeof(T))) & (W - 1));
    vectors = (n - head) / W;
  }
  __device__ __forceinline__ int rounds() const { return (vectors + A * THREADS - 1) / (A * THREADS); }
  // This thread's token in front of or behind the vectors, or -1.
  __device__ __forceinline__ int edge() const {
    const int t = int(threadIdx.x), at = t < head ? t : t + vectors * W;
    return at < n && (t < head || t < n - vectors * W) ? at : -1;
  }
  __device__ __forceinline__ void load(typename Vec<T>::type (&x)[A], int round) const {
#pragma unroll
    for (int c = 0; c < A; ++c) {
      const int v = (round * A + c) * THREADS + int(threadIdx.x);
      x[c] = *reinterpret_cast<const typename Vec<T>::type*>(p + head + min(v, vectors - 1) * W);
    }
  }
  __device__ __forceinline__ int token(int round, int c) const { return head + ((round * A + c) * THREADS + int(threadIdx.x)) * W; }
  // f(value, index) for every token.
  template <typename F>
  __device__ void each(F f) const {
    const int e = edge();
    if (e >= 0) f(float(p[e]), e);
    for (int r = 0; r < rounds(); ++r) {
      typename Vec<T>::type x[A];
      load(x, r);
#pragma unroll
      for (int c = 0; c < A; ++c)
#pragma unroll
        for (int i = 0; i < W; ++i)
          if (token(r, c) + i < head + vectors * W) f(float(x[c][i]), token(r, c) + i);
    }
  }
};

// The list again, for a row whose tokens at or above `bar` (keys) are more than it holds: the
// range of their keys is cut into kRuns runs, and the one in which the `top`-th lies is cut
// again, until it and the runs above fit.  (Keys are distinct, so this ends.)
template <typename T, int THREADS>
__device__ __noinline__ void refill(Lds<T, THREADS>& s, const Row<T, THREADS>& row, u64 bar, unsigned top) {
  u64 low = ~u64(0), high = 0;
  if (threadIdx.x == 0) {
    s.low = low;
    s.high = high;
  }
  __syncthreads();
  row.each([&](float x, int i) {
    if (!(x > kNegInf)) return;
    const u64 k = key_of(x, i);
    if (k < bar) return;
    low = min(low, k);
    high = max(high, k);
  });
  atomicMin(&s.low, low);
  atomicMax(&s.high, high);
  __syncthreads();
  low = s.low;
  high = s.high;
  unsigned front = 0;  // tokens above `high`: fewer than top
  while (true) {
    const u64 width = (high - low) / kRuns + 1;
    for (int i = int(threadIdx.x); i < kRuns; i += THREADS) s.run[i] = 0;
    __syncthreads();
    row.each([&](float x, int i) {
      if (!(x > kNegInf)) return;
      const u64 k = key_of(x, i);
      if (k >= low && k <= high) atomicAdd(&s.run[(high - k) / width], 1u);
    });
    __syncthreads();
    if (threadIdx.x == 0) {
      unsigned sum = front;
      int r = 0;
      while (r < kRuns - 1 && sum + s.run[r] < top) sum += s.run[r++];
      s.pick = unsigned(r);
      s.above = sum;
    }
    __syncthreads();
    const unsigned pick = s.pick, above = s.above, in = s.run[pick];
    const u64 from = high - u64(pick) * width, to = from - low < width ? low : from - width + 1;
    __syncthreads();
    if (above + in <= kList || width == 1) {
      low = to;
      break;
    }
    front = above;
    high = from;
    low = to;
  }
  if (threadIdx.x == 0) s.count = 0;
  __syncthreads();
  row.each([&](float x, int i) {
    if (!(x > kNegInf)) return;
    const u64 k = key_of(x, i);
    if (k < low) return;
    const unsigned at = atomicAdd(&s.count, 1u);
    if (at < kList) s.list[at] = k;
  });
  __syncthreads();
}

template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void logprobs_kernel(LogprobsArgs a) {
  constexpr int WAVES = THREADS / 64;
  using R = Row<T, THREADS>;
  __shared__ Lds<T, THREADS> s;
  const int tid = int(threadIdx.x), lane = tid & 63, wave = tid >> 6;
  const T* logits = static_cast<const T*>(a.logits) + int64_t(blockIdx.x) * a.vocab;
  const R row(logits, a.vocab);
  const int rounds = row.rounds();
  typename Vec<T>::type next[R::A];
  if (rounds > 0) row.load(next, 0);
  const int edge = row.edge();
  const float edge_x = edge >= 0 ? float(logits[edge]) : kNegInf;
  if (tid == 0) s.count = 0;
  Stats mine{kNegInf, 0.f, 0.f, 0.f};
  u64 bar = ~u64(0);
  const auto offer = [&](float x, int i) {
    if (x > kNegInf && key_of(x, i) >= bar) {
      const unsigned at = atomicAdd(&s.count, 1u);
      if (at < kList) s.list[at] = key_of(x, i);
    }
  };
  {
    const float x[1] = {edge_x};
    mine.add(x);
  }
  float bar_x = __builtin_huge_valf();  // the bar's value: no token below it counts
  for (int r = 0; r < rounds || r == 0; ++r) {
    float x[R::A * R::W];
    float high = kNegInf;
    int high_at = 0;
#pragma unroll
    for (int c = 0; c < R::A; ++c)
#pragma unroll
      for (int i = 0; i < R::W; ++i) {
        const bool is = row.token(r, c) < row.head + row.vectors * R::W;  // (a vector is whole or not there)
        x[c * R::W + i] = is ? float(next[c][i]) : kNegInf;
      }
    if (r + 1 < rounds) row.load(next, r + 1);
    mine.add(x);
    if (a.top > 0) {
      if (r == 0) {
        // The bar, from every thread's first tokens.
        high = edge_x;
        high_at = edge;
#pragma unroll
        for (int i = 0; i < R::A * R::W; ++i) {
          const int at = row.token(0, i / R::W) + i % R::W;
          const bool more = x[i] > high || (x[i] == high && at < high_at);
          high_at = more ? at : high_at;
          high = more ? x[i] : high;
        }
        u64 best = high > kNegInf ? key_of(high, high_at) : 0, bound = best;
        const int ranks = (a.top + WAVES - 1) / WAVES;
        for (int i = 0; i < ranks; ++i) {
          bound = wave_max_key(best);
          best = best == bound ? 0 : best;
        }
        if (lane == 0) s.bar[wave] = bound;
        __syncthreads();  // (and the count is 0)
        bar = s.bar[0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) bar = min(bar, s.bar[w]);
        bar_x = bar == 0 ? kNegInf : value_of(bar);
        offer(edge_x, edge);
      }
      high = kNegInf;
#pragma unroll
      for (int i = 0; i < R::A * R::W; ++i) high = fmaxf(high, x[i]);
      if (high >= bar_x) {
#pragma unroll
        for (int i = 0; i < R::A * R::W; ++i)
          if (x[i] >= bar_x) offer(x[i], row.token(r, i / R::W) + i % R::W);
      }
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mine.join(mine.from(o));
  if (lane == 0) s.stats[wave] = mine;
  __syncthreads();
  mine = s.stats[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) mine.join(s.stats[w]);

  const bool none = mine.m == kNegInf, sure = mine.m == __builtin_huge_valf();
  const float log_z = logf(mine.count) + log1pf(mine.rest / mine.count);
  int first = kNoToken;  // sure: the first +inf
  if (sure) {
    if (tid == 0) s.pick = unsigned(kNoToken);
    __syncthreads();
    row.each([&](float x, int i) {
      if (x == __builtin_huge_valf()) atomicMin(&s.pick, unsigned(i));
    });
    __syncthreads();
    first = int(s.pick);
  }
  const auto log_p = [&](float x, int i) {
    if (sure) return i == first ? 0.f : kNegInf;
    return x > kNegInf ? (x - mine.m) - log_z : kNegInf;
  };
  if (tid == 0) a.entropy[blockIdx.x] = none || sure ? 0.f : log_z - mine.spread / (mine.count + mine.rest);
  for (int i = tid; i < a.given; i += THREADS) {
    const int64_t at = int64_t(blockIdx.x) * a.given + i;
    const int token = a.tokens[at];
    a.logprobs[at] = token >= 0 && token < a.vocab ? log_p(float(logits[token]), token) : kNegInf;
  }
  if (a.top == 0) return;
  if (s.count > kList) refill(s, row, bar, unsigned(a.top));
  const unsigned n = min(s.count, unsigned(kList));
  const int64_t out = int64_t(blockIdx.x) * a.top;
  for (unsigned i = unsigned(tid); i < n; i += THREADS) {
    const u64 k = s.list[i];
    unsigned before = 0;
    for (unsigned o = 0; o < n; ++o) before += s.list[o] > k;
    if (before < unsigned(a.top)) {
      a.top_tokens[out + before] = index_of(k);
      a.top_logprobs[out + before] = log_p(value_of(k), index_of(k));
    }
  }
  for (unsigned i = n + unsigned(tid); i < unsigned(a.top); i += THREADS) {
    a.top_tokens[out + i] = kNoToken;
    a.top_logprobs[out + i] = kNegInf;
  }
}

}  // namespace

hipError_t logprobs(const LogprobsArgs& a, hipStream_t stream) {
  if (a.f32) hipLaunchKernelGGL((logprobs_kernel<float, 1024>), dim3(unsigned(a.batch)), dim3(1024), 0, stream, a);
  else hipLaunchKernelGGL((logprobs_kernel<f16, 1024>), dim3(unsigned(a.batch)), dim3(1024), 0, stream, a);
  return hipGetLastError();
}

}  // namespace tia
