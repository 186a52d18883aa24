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
// over the distance from the maximum, 256 bins to a unit of (max - logit) / T,
// finds the bin in which a count or a mass is reached, and only the tokens of the
// few bins in question are gathered and ordered.  A token of bin b at distance
// (b + f) / 256 weighs e^(-b/256) (1 - q), q = 1 - e^(-f/256) < 1.02 * 2^-8: bins hold
// their count and the sum of q in units of 2^-34, one 64-bit LDS addition per token (a bin
// that holds the whole vocabulary fits: sample_bins.hpp), and masses are whole numbers of 2^-44: sums are the same in any order, and an
// answer depends on its row alone.  A token's mass is right to 1.4 * 2^-30 of itself (the
// fraction's 2^-23 of a bin, and fp32 roundings of q), a bin's rounded to 2^-45, and tokens
// 32 units from the maximum weigh nothing: at most V e^-32 of the likeliest one's mass is left
// out, 3.4e-9 at 2^18 tokens.  So the token is the one that 64-bit arithmetic gives but for a
// random number (or a top-p) within twice 2^-29 + V e^-32 of a border, 1.1e-8 at most; fp32
// numbers next to 1 are 6e-8 apart.
//
// One workgroup per row reads it three times (maximum, bins, gathering), the second and
// third time from cache.  (Keeping it in registers needs every pass unrolled over them: 50
// KB of code that runs once per wave, fetched from memory, took 20 us a pass; a pass over
// 201 KB in L2 reads in 1.6 us.)  Rows with a small top-k take a shorter way that
// reads them once.
//
// What bounds it.  32 rows of 50257 with top-p take 26 us: about 3 for the maximum (one CU's
// loads), 6.5 for the bins and 4 for the gathering (20 and 6 vector instructions a token), 3.5
// for the sums over the bins, 2 for the searches, 3 for ordering and answers; without data (a
// few tokens) 13 are left.  32 CUs are busy, their VALU 76 %.  (Several workgroups to a row
// would have to bring their bins together, 64 KB each; not tried.)  256 rows
// of 128257 by a top-k up to 200, top-p and min-p take 39 us, 22 of them memory; by top-p
// alone 75.
#include "common.hpp"
#include "kernels.hpp"
#include "lds_limit.hpp"
#include "sample_bins.hpp"

namespace tia {
namespace {

using namespace sample_bins;

constexpr int kThreads = 1024, kPerThread = 8, kBins = kThreads * kPerThread, kList = 512, kRuns = 2048;
// A top-k up to which a row may be sampled in one pass: half of what the list holds, so
// that a bin which ends past the k-th token still fits.
constexpr unsigned kShort = 256;
// Whether it is: ordering the k costs k^2, the longer way the row twice more.  In one pass
// against the longer way, us: 64 rows of 1000 tokens, k = 40 12.6 and 14.1, k = 256 17.1 and
// 14.2; of 10000, 13.2 and 17.2, 18.2 and 17.3; of 20000, 13.3 and 18.9, 18.2 and 19.1; 32
// rows of 50257, 14.9 and 30.8, 19.7 and 30.6.
__device__ __forceinline__ bool is_short(unsigned k, unsigned vocab) { return k <= kShort && k < vocab && k * k / 4 <= vocab; }
constexpr int kNoToken = 0x7fffffff;
constexpr float kNegInf = -__builtin_huge_valf();
// Place of a bin in LDS: a thread's kPerThread bins are followed by a gap, so that the
// threads of a wave, each at its own run, meet in no bank.
__device__ __forceinline__ constexpr unsigned slot(unsigned bin) { return bin + (bin >> 3); }

struct SampleLds {
  union {
    u64 bin[slot(kBins)];   // while the row is counted
    u64 mass[slot(kBins)];  // then: the mass in front of each bin
  };
  unsigned count[slot(kBins)];  // tokens in front of each bin
  u64 runs[kRuns];
  u64 key[kList];         // the gathered tokens,
  unsigned at[kList], q[kList];  // their bins and losses
  unsigned wanted[kBins / 32];   // a bit per bin whose tokens are gathered
  u64 wave_mass[kThreads / 64];
  unsigned wave_count[kThreads / 64], run_count[kBins / 1024];
  float wave_max[kThreads / 64];
  int wave_at[kThreads / 64];
  u64 low, high, answer_key, answer_mass;
  unsigned answer_count, list_count, claims[3];  // (a claim per goal of a row: top-k, top-p, the random number)
};

// 64-bit key whose ascending order is the row's: value descending, then index.
__device__ __forceinline__ u64 order_key(float x, int i) {
  const unsigned b = __builtin_bit_cast(unsigned, x + 0.f);  // -0 orders as 0
  const unsigned up = b & 0x80000000u ? ~b : b | 0x80000000u;
  return u64(~up) << 32 | unsigned(i);
}

__device__ __forceinline__ float value_of(u64 key) {
  const unsigned up = ~unsigned(key >> 32);
  return __builtin_bit_cast(float, up & 0x80000000u ? up & 0x7fffffffu : ~up);
}

// A row: its 16-byte vectors on 16-byte boundaries of memory, and the few tokens in
// front of the first and behind the last of them.
template <typename T>
struct Row {
  static constexpr int W = 16 / int(sizeof(T));
  typedef T vec __attribute__((ext_vector_type(W)));
  const T* p;
  int n, head, vectors;  // tokens; those in front of the first vector

  __device__ __forceinline__ Row(const T* row, int length) : p(row), n(length) {
    head = min(n, int(-(reinterpret_cast<uintptr_t>(row) / sizeof(T))) & (W - 1));
    vectors = (n - head) / W;
  }
  // The vectors at, at + kThreads, ... (the last one's values past it).
  template <int A>
  __device__ __forceinline__ void load(vec (&x)[A], int at) const {
#pragma unroll
    for (int c = 0; c < A; ++c) x[c] = *reinterpret_cast<const vec*>(p + head + min(at + c * kThreads, vectors - 1) * W);
  }
  template <typename F>
  __device__ __forceinline__ void edges(F f) const {
    const int t = int(threadIdx.x), at = t < head ? t : t + vectors * W;
    if (at < n && (t < head || t < n - vectors * W)) f(float(p[at]), at);
  }
  // f(value, index) for every token, the next vectors on their way while A are worked on.
  template <int A, typename F>
  __device__ __forceinline__ void each(F f) const {
    edges(f);
    int at = int(threadIdx.x);
    if (at >= vectors) return;
    vec x[A];
    load(x, at);
    while (at < vectors) {
      vec next[A];
      load(next, at + A * kThreads);
#pragma unroll
      for (int c = 0; c < A; ++c) {
        if (at + c * kThreads >= vectors) break;
#pragma unroll
        for (int e = 0; e < W; ++e) f(float(x[c][e]), head + (at + c * kThreads) * W + e);
      }
#pragma unroll
      for (int c = 0; c < A; ++c) x[c] = next[c];
      at += A * kThreads;
    }
  }
  // f(value, index) for the few tokens that `rare` holds for.
  template <typename P, typename F>
  __device__ __forceinline__ void pick(P rare, F f) const {
    constexpr int A = 32 / W;
    edges([&](float x, int i) {
      if (rare(x)) f(x, i);
    });
    for (int at = int(threadIdx.x); at < vectors; at += A * kThreads) {
      vec x[A];
      load(x, at);
      unsigned hits = 0;
#pragma unroll
      for (int c = 0; c < A; ++c)
#pragma unroll
        for (int e = 0; e < W; ++e) hits |= unsigned(rare(float(x[c][e]))) << (c * W + e);
#pragma unroll
      for (int c = 1; c < A; ++c)
        if (at + c * kThreads >= vectors) hits &= (1u << (c * W)) - 1;
      while (hits) {
        const int k = __builtin_ctz(hits), i = head + (at + k / W * kThreads) * W + k % W;
        hits &= hits - 1;
        f(float(p[i]), i);
      }
    }
  }
  // f(value, index) for every token of the few vectors that hold one which is `rare`: for a
  // test of several instructions, of which a vector's masks are joined by the scalar unit (32
  // rows of 128257 with top-p and min-p: 46 us, 54 by pick; but top-k 256 21.9, 20.4 by pick).
  template <typename P, typename F>
  __device__ __forceinline__ void pick_vectors(P rare, F f) const {
    constexpr int A = 32 / W;
    edges(f);
    for (int at = int(threadIdx.x); at < vectors; at += A * kThreads) {
      vec x[A];
      load(x, at);
      unsigned hits = 0;
#pragma unroll
      for (int c = 0; c < A; ++c) {
        bool any = false;
#pragma unroll
        for (int e = 0; e < W; ++e) any |= rare(float(x[c][e]));
        hits |= unsigned(any) << c;
      }
      while (hits) {
        const int c = __builtin_ctz(hits), v = at + c * kThreads;
        hits &= hits - 1;
        if (v >= vectors) break;
        const vec y = *reinterpret_cast<const vec*>(p + head + v * W);
#pragma unroll
        for (int e = 0; e < W; ++e) f(float(y[e]), head + v * W + e);
      }
    }
  }
  // A vector per thread, spread evenly over a row of more, and of the edges a token; -inf
  // where there is none.
  __device__ __forceinline__ vec sample(T& edge) const {
    const int t = int(threadIdx.x), i = t < head ? t : t + vectors * W;
    edge = t < head || t < n - vectors * W ? p[i] : T(kNegInf);
    const int at = vectors <= kThreads ? t : int(unsigned(vectors) * u64(t) / kThreads);
    if (at < vectors) return *reinterpret_cast<const vec*>(p + head + at * W);
    return vec(T(kNegInf));
  }
};

// Distances from the maximum in bins, in fp32 with what its roundings leave out: D =
// max - logit is a sum of two fp32 numbers exactly, 256 / T of two to 2^-48.  The
// rounded distance, monotone in the logit, gives the bin (of tokens in order the bins
// are in order); its fraction, taken with the rest, is right to about 2^-23 of a bin.
struct Scale {
  float top, per, per_rest;  // max; 256 / T
  double temp;
  __device__ __forceinline__ Scale(float max, float t) : top(max), temp(t) {
    const double p = kPerUnit / temp;
    per = float(fmin(p, 3e38));  // (T below 1e-36: every smaller logit is past the last bin)
    per_rest = float(p - double(per));
    if (!(fabsf(per_rest) < 1e30f)) per_rest = 0.f;
  }
  // Not below kBins for -inf, neither below nor above for NaN.
  __device__ __forceinline__ float distance(float x) const { return (top - x) * per; }
  // The part of the distance behind its bin's near edge: in [-kFraction, 1 + kFraction].
  __device__ __forceinline__ float fraction(float x) const {
    const float d = top - x, back = d - top, rest = (top - (d - back)) - (x + back);
    return fmaf(d, per, -floorf(d * per)) + fmaf(d, per_rest, rest * per);
  }
  __device__ __noinline__ double weight_of(float x) const { return exp((double(x) - double(top)) / temp); }
};
// e^(-i/256)
__device__ __forceinline__ double step(int i) {
  constexpr double k[kPerThread] = {1.0, 0.9961013694701175, 0.9922179382602435, 0.9883496471138451,
                                    0.9844964370054085, 0.9806582491395386, 0.976835024950062, 0.9730267060991332};
  double x = k[0];
#pragma unroll
  for (int e = 1; e < kPerThread; ++e) x = i == e ? k[e] : x;
  return x;
}
__device__ __noinline__ double run_edge(unsigned run) { return exp((double(run) * -kPerThread + double(kSlack)) / kPerUnit); }
// Mass of a weight in a bin whose edge is e = run_edge * step.
__device__ __forceinline__ u64 mass_of(u64 weight, double e) { return u64(fma(double(weight), e * kMass, 0.5)); }

// Turns the counted bins into what stands in front of each; all threads return the totals.
__device__ void scan(SampleLds& s, u64& mass_all, unsigned& count_all) {
  const int t = int(threadIdx.x), lane = t & 63, wave = t >> 6;
  __syncthreads();
  const double edge = run_edge(unsigned(t));
  u64 m[kPerThread], mi = 0;
  unsigned c[kPerThread], ci = 0;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const u64 b = s.bin[slot(kPerThread * t + i)];
    m[i] = mi;
    c[i] = ci;
    mi += mass_of(weight_of(b), edge * step(i));
    ci += count_of(b);
  }
  const u64 mine = mi;
  const unsigned many = ci;
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
  u64 front = mi - mine;
  unsigned before = ci - many;
  mass_all = 0;
  count_all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    front += w < wave ? s.wave_mass[w] : 0;
    before += w < wave ? s.wave_count[w] : 0;
    mass_all += s.wave_mass[w];
    count_all += s.wave_count[w];
  }
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    s.mass[slot(kPerThread * t + i)] = front + m[i];
    s.count[slot(kPerThread * t + i)] = before + c[i];
  }
  __syncthreads();
}

// What a position is asked by: the first token whose count or mass, with all in
// front of it, reaches `goal` (goal >= 1, and at most the total), which is the last one
// that begins in front of it.
struct Goal {
  bool by_count;
  u64 goal;
};
struct Place {
  u64 mass;        // of the tokens up to this one
  unsigned count;  // of the same
  u64 key;
};

// floor(f m) for 0 <= f < 1 exactly (bits of f below 2^-64 count as 0); whole: f m is a whole number.
__device__ __forceinline__ u64 part_of(float f, u64 m, bool& whole) {
  const u64 fx = f > 0.f ? u64(ldexp(double(f), 64)) : 0;
  whole = fx * m == 0;
  return __umul64hi(fx, m);
}
// Goal of the first token with cumulative mass >= top_p m, and of the first above u m.
__device__ __forceinline__ Goal goal_p(float top_p, u64 m) {
  bool whole;
  const u64 g = part_of(top_p, m, whole), up = whole ? g : g + 1;
  return Goal{false, up > 0 ? up : 1};
}
__device__ __forceinline__ Goal goal_u(float u, u64 m) {
  bool whole;
  return Goal{false, part_of(u, m, whole) + 1};
}

// The bin in which the goal is reached: the last one that begins in front of it.  Every
// wave searches for itself: its lanes look at 64 bins in even steps, then at the 128 of
// one step.
__device__ __forceinline__ unsigned find_bin(const SampleLds& s, const Goal& g) {
  const unsigned lane = threadIdx.x & 63;
  const auto in_front = [&](unsigned bin) { return __ballot((g.by_count ? u64(s.count[slot(bin)]) : s.mass[slot(bin)]) < g.goal); };
  static_assert(kBins == 64 * 128, "two steps of the search");
  const unsigned run = 128 * (__popcll(in_front(128 * lane)) - 1);  // (bin 0 always is)
  return run + __popcll(in_front(run + lane)) + __popcll(in_front(run + 64 + lane)) - 1;
}

__device__ __forceinline__ bool is_wanted(const SampleLds& s, unsigned bin) { return s.wanted[bin >> 5] >> (bin & 31) & 1; }
__device__ __forceinline__ void take(SampleLds& s, u64 key, unsigned bin, float fraction) {
  const unsigned i = atomicAdd(&s.list_count, 1u);
  if (i < kList) {
    s.key[i] = key;
    s.at[i] = bin;
    s.q[i] = loss(fraction);
  }
}

// A gathered token's place in the row's order, one per thread.
struct Gathered {
  u64 key = 0, before = 0, after = 0;  // mass in front of the token, and with it
  unsigned rank = 0, bin = ~0u;
  // weight0, count0: what stands in front of the list within its (single) bin.  Several
  // threads to a token, each comparing it with a part of the others.
  __device__ __forceinline__ void order(SampleLds& s, u64 weight0, unsigned count0) {
    const unsigned n = min(s.list_count, unsigned(kList)), t = threadIdx.x;
    unsigned wide = 64;
    while (wide < n) wide *= 2;
    const unsigned mine = t & (wide - 1), part = t / wide, parts = kThreads / wide, chunk = (n + parts - 1) / parts;
    if (t < n) s.runs[t] = 0;
    __syncthreads();
    if (mine < n) {
      const u64 own = s.key[mine];
      const unsigned of = s.at[mine], end = min(n, (part + 1) * chunk);
      u64 front = 0;  // as a bin: count and sum of losses
#pragma unroll 4
      for (unsigned o = part * chunk; o < end; ++o)
        front += (s.at[o] == of) & (s.key[o] < own) ? (u64(1) << kCountShift) + s.q[o] : 0;
      if (front) atomicAdd(&s.runs[mine], front);
    }
    __syncthreads();
    bin = ~0u;
    if (t >= n) return;
    key = s.key[t];
    bin = s.at[t];
    const u64 front = weight0 + weight_of(s.runs[t]);
    rank = s.count[slot(bin)] + count0 + count_of(s.runs[t]);
    const double e = run_edge(bin / kPerThread) * step(int(bin % kPerThread));
    before = s.mass[slot(bin)] + mass_of(front, e);
    after = s.mass[slot(bin)] + mass_of(front + kOne - s.q[t], e);
  }
  // Goal number `which` of the row (its claim is still 0).  Without any token gathered from
  // the bin the row's first one stands for all.
  __device__ __forceinline__ Place resolve(SampleLds& s, unsigned of, const Goal& g, int which) const {
    const unsigned claim = bin == of ? claim_of(g.by_count ? rank : before, g.goal, rank, threadIdx.x) : 0;
    if (claim) atomicMax(&s.claims[which], claim);
    __syncthreads();  // (the answer in front of this one has been read)
    const unsigned best = s.claims[which];
    if (threadIdx.x == claimant(best)) {
      s.answer_key = best ? key : 0;
      s.answer_mass = best ? after : s.mass[slot(of)] + 1;
      s.answer_count = best ? rank + 1 : s.count[slot(of)] + 1;
    }
    __syncthreads();
    return Place{s.answer_mass, s.answer_count, s.answer_key};
  }
};

// Gathers the tokens of `bin`, or where they are too many those of a run of it in which
// the goal is reached.
template <typename T>
__device__ __noinline__ Gathered gather(SampleLds& s, const Row<T>& row, const Scale& sc, const Goal& g, unsigned bin,
                                        unsigned count_all) {
  u64 low = 0, high = ~u64(0), weight0 = 0;
  unsigned count0 = 0, n = (bin + 1 < kBins ? s.count[slot(bin + 1)] : count_all) - s.count[slot(bin)];
  const auto in_bin = [&](float x) {
    const float d = sc.distance(x);
    return d >= float(bin) && d < float(bin + 1);
  };
  __syncthreads();
  if (n > kList) {
    // A crowded bin: its keys' range, cut into runs of equal width until one run's
    // tokens fit the list.  (Keys are distinct, so this ends.)
    if (threadIdx.x == 0) {
      s.low = ~u64(0);
      s.high = 0;
    }
    __syncthreads();
    u64 lo = ~u64(0), hi = 0;
    row.template each<2>([&](float x, int i) {
      if (!in_bin(x)) return;
      const u64 k = order_key(x, i);
      lo = min(lo, k);
      hi = max(hi, k);
    });
    atomicMin(&s.low, lo);
    atomicMax(&s.high, hi);
    __syncthreads();
    low = s.low;
    high = s.high;
    const double e = run_edge(bin / kPerThread) * step(int(bin % kPerThread));
    while (n > kList) {
      int shift = 0;
      while (((high - low) >> shift) >= kRuns) ++shift;
      __syncthreads();
      for (int i = int(threadIdx.x); i < kRuns; i += kThreads) s.runs[i] = 0;
      __syncthreads();
      row.template each<2>([&](float x, int i) {
        if (!in_bin(x)) return;
        const u64 k = order_key(x, i);
        if (k >= low && k <= high) atomicAdd(&s.runs[(k - low) >> shift], packed(sc.fraction(x)));
      });
      __syncthreads();
      // (Rare enough that every thread walks the runs by itself.)
      int at = 0;
      for (; at < kRuns - 1; ++at) {
        const u64 b = s.runs[at], w = weight0 + weight_of(b);
        const unsigned c = count0 + count_of(b);
        if (g.goal <= (g.by_count ? u64(s.count[slot(bin)] + c) : s.mass[slot(bin)] + mass_of(w, e))) break;
        weight0 = w;
        count0 = c;
      }
      n = count_of(s.runs[at]);
      low += u64(at) << shift;
      high = min(high, low + ((u64(1) << shift) - 1));
    }
  }
  __syncthreads();
  if (threadIdx.x < kBins / 32) s.wanted[threadIdx.x] = 0;
  if (threadIdx.x == 0) s.list_count = 0;
  __syncthreads();
  // The whole bin is at hand for the next goal, a run of it is not.
  if (threadIdx.x == 0 && weight0 == 0 && high == ~u64(0)) s.wanted[bin >> 5] = 1u << (bin & 31);
  row.pick(in_bin, [&](float x, int i) {
    const u64 k = order_key(x, i);
    if (k >= low && k <= high) take(s, k, bin, sc.fraction(x));
  });
  __syncthreads();
  Gathered mine;
  mine.order(s, weight0, count0);
  return mine;
}

template <typename T>
__device__ __forceinline__ Place locate(SampleLds& s, const Row<T>& row, const Scale& sc, Gathered& mine, const Goal& g,
                                        unsigned count_all, int which) {
  const unsigned bin = find_bin(s, g);
  if (!is_wanted(s, bin)) mine = gather(s, row, sc, g, bin, count_all);
  return mine.resolve(s, bin, g, which);
}


// The bin of the token with `goal` - 1 others in front of it, from the counts per bin;
// before: the tokens in front of the bin.  kBins if there are fewer.  A wave sums 1024 bins,
// 16 to a lane; every wave then looks into the thousand in question and into one lane's.
__device__ __forceinline__ unsigned bin_of_rank(SampleLds& s, unsigned goal, unsigned& before) {
  const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const auto sum_of = [&](unsigned run) {
    unsigned sum = 0;
#pragma unroll
    for (unsigned i = 0; i < 16; ++i) sum += s.count[slot(run + 16 * lane + i)];
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const unsigned up = __shfl_up(sum, o, 64);
      sum += lane >= unsigned(o) ? up : 0;
    }
    return sum;
  };
  if (wave < kBins / 1024) {
    const unsigned sum = sum_of(1024 * wave);
    if (lane == 63) s.run_count[wave] = sum;
  }
  __syncthreads();
  before = 0;
  unsigned run = 0;
  while (run < kBins / 1024 && before + s.run_count[run] < goal) before += s.run_count[run++];
  if (run == kBins / 1024) return kBins;
  run *= 1024;
  const unsigned sum = sum_of(run);
  const int over = __popcll(__ballot(before + sum < goal));
  if (over > 0) before += __shfl(sum, over - 1, 64);
  unsigned upto = s.count[slot(run + 16 * over + (lane & 15))];
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    const unsigned up = __shfl_up(upto, o, 16);
    upto += (lane & 15) >= unsigned(o) ? up : 0;
  }
  const int bin = __popcll(__ballot(lane < 16 && before + upto < goal));
  if (bin > 0) before += __shfl(upto, bin - 1, 64);
  return run + 16 * over + bin;
}

__device__ __forceinline__ float block_top(SampleLds& s, float top) {
  top = wave_max(top);
  if ((threadIdx.x & 63) == 0) s.wave_max[threadIdx.x >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) top = fmaxf(top, s.wave_max[w]);
  return top;
}

// A top-k that is_short, in one pass over the row: a sample of it says which logits are
// likely to be among four times as many as may be kept, the tokens with those are gathered,
// and everything else is read off the list: the maximum, the bin of the last token that may
// be kept, the order up to that bin and the cumulative masses.  False, nothing written: too
// few tokens were found, or more than the lists hold.
template <typename T>
__device__ __forceinline__ bool sample_short(SampleLds& s, const Row<T>& row, float temp, unsigned most, float top_p,
                                             float min_p, float u, int32_t* token, float* prob) {
  const unsigned t = threadIdx.x, lane = t & 63;
  const auto clear = [&] {
    for (unsigned i = t; i < slot(kBins); i += kThreads) s.count[i] = 0;
    if (t == 0) s.list_count = 0;
  };
  clear();
  float top = kNegInf;
  T edge;
  const auto sampled = row.sample(edge);
  top = fmaxf(top, float(edge));
#pragma unroll
  for (int e = 0; e < Row<T>::W; ++e) top = fmaxf(top, float(sampled[e]));
  top = block_top(s, top);
  if (top == kNegInf || top == -kNegInf) return false;
  const Scale about(top, temp);
  const auto counts = [&](float x) {
    const float d = about.distance(x);
    if (d < float(kBins)) atomicAdd(&s.count[slot(unsigned(d))], 1u);
  };
  counts(float(edge));
#pragma unroll
  for (int e = 0; e < Row<T>::W; ++e) counts(float(sampled[e]));
  __syncthreads();
  unsigned before;
  const unsigned enough = row.vectors <= kThreads ? most : 4 * most * Row<T>::W * kThreads / unsigned(row.n) + 8;
  const float least = top - float(min(bin_of_rank(s, enough, before) + 1, unsigned(kBins))) / about.per;
  __syncthreads();
  clear();
  __syncthreads();
  row.pick([&](float x) { return x >= least; },
           [&](float x, int i) {
             const unsigned at = atomicAdd(&s.list_count, 1u);
             if (at < kBins) s.bin[at] = order_key(x, i);
           });
  __syncthreads();
  const unsigned found = s.list_count;
  if (found < most || found > kBins) return false;
  for (unsigned i = t; i < found; i += kThreads) top = fmaxf(top, value_of(s.bin[i]));
  top = block_top(s, top);
  if (top == -kNegInf) return false;
  const Scale sc(top, temp);
  unsigned counted = 0;
  for (unsigned i = t; i < found; i += kThreads) {
    const float d = sc.distance(value_of(s.bin[i]));
    if (d < float(kBins)) {
      atomicAdd(&s.count[slot(unsigned(d))], 1u);
      ++counted;
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) counted += __shfl_xor(counted, o, 64);
  if (lane == 0) s.wave_count[t >> 6] = counted;
  __syncthreads();
  counted = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) counted += s.wave_count[w];
  most = min(most, counted);
  const unsigned last = bin_of_rank(s, most, before);
  const unsigned n = before + s.count[slot(last)];
  if (n > kList) return false;
  __syncthreads();
  if (t == 0) s.list_count = 0;
  __syncthreads();
  for (unsigned i = t; i < found; i += kThreads) {
    const u64 key = s.bin[i];
    if (sc.distance(value_of(key)) < float(last + 1)) s.key[atomicAdd(&s.list_count, 1u)] = key;
  }
  __syncthreads();
  // Ranks: `parts` threads to a token, each comparing it with a part of the others.
  unsigned wide = 64;
  while (wide < n) wide *= 2;
  const unsigned mine = t & (wide - 1), part = t / wide, parts = kThreads / wide, chunk = (n + parts - 1) / parts;
  if (t < n) s.q[t] = 0;
  __syncthreads();
  const u64 key = s.key[min(mine, n - 1)];
  {
    unsigned ahead = 0;
    const unsigned end = min(n, (part + 1) * chunk);
#pragma unroll 4
    for (unsigned o = part * chunk; o < end; ++o) ahead += s.key[o] < key;
    if (mine < n) atomicAdd(&s.q[mine], ahead);
  }
  __syncthreads();
  // Masses in the row's order, in units of 2^-44 of the heaviest token's, and their sums.
  constexpr double unit = 17592186044416.0;
  double weight = 0;
  unsigned rank = ~0u;
  if (t < n) {  // (mine = t)
    rank = s.q[t];
    weight = sc.weight_of(value_of(key));
    s.runs[rank] = u64(fma(weight, unit, 0.5));
  }
  __syncthreads();
  u64 sum = t < n ? s.runs[t] : 0;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 up = __shfl_up(sum, o, 64);
    sum += lane >= unsigned(o) ? up : 0;
  }
  if (lane == 63) s.wave_mass[t >> 6] = sum;
  __syncthreads();
#pragma unroll
  for (unsigned w = 0; w < kList / 64; ++w) sum += w < t >> 6 ? s.wave_mass[w] : 0;
  if (t < n) s.runs[t] = sum;
  unsigned kept = most;
  if (min_p > 0.f) {
    const unsigned heavy = __syncthreads_count(t < n && weight >= double(min_p));
    kept = min(kept, max(heavy, 1u));
  } else {
    __syncthreads();
  }
  if (top_p < 1.f) {
    const u64 goal = goal_p(top_p, s.runs[most - 1]).goal;
    kept = min(kept, 1u + unsigned(__syncthreads_count(t < n && s.runs[t] < goal)));
  }
  const u64 mass = s.runs[kept - 1], goal = goal_u(u, mass).goal;
  if (rank < n && s.runs[rank] >= goal && (rank == 0 || s.runs[rank - 1] < goal)) {
    *token = int(key & 0xffffffffu);
    *prob = float(weight * unit / double(mass));
  }
  return true;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  SampleLds& s = *reinterpret_cast<SampleLds*>(lds);
  const int b = int(blockIdx.x), t = int(threadIdx.x);
  Row<T> row(static_cast<const T*>(a.logits) + int64_t(b) * a.vocab, a.vocab);
  const float temp = a.temperature ? a.temperature[b] : a.temperature_all;
  const int top_k = a.top_k ? a.top_k[b] : a.top_k_all;
  const float top_p = a.top_p ? a.top_p[b] : a.top_p_all, min_p = a.min_p ? a.min_p[b] : a.min_p_all;
  float u = a.uniforms[b];
  u = u > 0.f ? fminf(u, 0.99999994f) : 0.f;

  const unsigned most = top_k > 0 && top_k < a.vocab ? unsigned(top_k) : unsigned(a.vocab);
  if (is_short(most, unsigned(a.vocab)) && temp > 0.f && sample_short(s, row, temp, most, top_p, min_p, u, a.tokens + b, a.probs + b)) return;

  float top = kNegInf;
  row.template each<4>([&](float x, int) { top = fmaxf(top, x); });
  __syncthreads();
  top = block_top(s, top);
  if (top == kNegInf || !(temp > 0.f) || top == -kNegInf) {
    // No token above -inf, or the likeliest one.
    int at = kNoToken;
    if (top != kNegInf) row.template each<2>([&](float x, int i) { at = x == top ? min(at, i) : at; });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) at = min(at, __shfl_xor(at, o, 64));
    if ((t & 63) == 0) s.wave_at[t >> 6] = at;
    __syncthreads();
    if (t == 0) {
      for (int w = 1; w < kThreads / 64; ++w) at = min(at, s.wave_at[w]);
      a.tokens[b] = at;
      a.probs[b] = at == kNoToken ? 0.f : 1.f;
    }
    return;
  }
  const Scale sc(top, temp);
  for (unsigned i = unsigned(t); i < slot(kBins); i += kThreads) s.bin[i] = 0;
  if (t < kBins / 32) s.wanted[t] = 0;
  if (t < 3) s.claims[t] = 0;
  if (t == 0) s.list_count = 0;
  __syncthreads();
  row.template each<4>([&](float x, int) {
    const float d = sc.distance(x);
    if (d < float(kBins)) atomicAdd(&s.bin[slot(unsigned(d))], packed(sc.fraction(x)));
  });
  u64 mass_all;
  unsigned count_all;
  scan(s, mass_all, count_all);

  const bool use_k = top_k > 0 && unsigned(top_k) < count_all, use_p = top_p < 1.f, use_m = min_p > 0.f;
  // The bin of the logit whose weight is min_p: all tokens in front of it are heavier.
  unsigned far = 0;
  if (use_m) {
    const float d = sc.distance(float(double(top) + sc.temp * log(fmin(double(min_p), 1.0))));
    far = unsigned(fminf(fmaxf(d, 0.f), float(kBins - 1)));
  }

  // The bins in question, from masses known to a bin: their tokens are gathered in one pass.
  {
    const auto behind = [&](unsigned bin) { return bin + 1 < kBins ? s.mass[slot(bin + 1)] : mass_all; };
    constexpr int kRanges = 4;
    unsigned from[kRanges] = {1, 1, 1, 1}, to[kRanges] = {0, 0, 0, 0};
    u64 low = mass_all, high = mass_all;  // the kept mass lies between
    if (use_k) {
      from[0] = to[0] = find_bin(s, Goal{true, u64(top_k)});
      low = s.mass[slot(to[0])];
      high = behind(to[0]);
    }
    if (use_p) {
      from[1] = find_bin(s, goal_p(top_p, max(low, u64(1))));
      to[1] = low == high ? from[1] : find_bin(s, goal_p(top_p, high));
      low = s.mass[slot(from[1])];
      high = behind(to[1]);
    }
    if (use_m) {
      from[2] = to[2] = far;
      low = min(low, s.mass[slot(far)]);
      high = min(high, behind(far));
    }
    from[3] = find_bin(s, goal_u(u, max(low, u64(1))));
    to[3] = find_bin(s, goal_u(u, max(high, u64(1))));
    unsigned tokens = 0;
#pragma unroll
    for (int r = 0; r < kRanges; ++r) {
      if (from[r] > to[r]) continue;
      tokens += (to[r] + 1 < kBins ? s.count[slot(to[r] + 1)] : count_all) - s.count[slot(from[r])];
    }
    if (tokens <= kList) {  // (bins in two ranges count twice)
      if (t < kBins / 32) {
        unsigned bits = 0;
#pragma unroll
        for (int r = 0; r < kRanges; ++r) {
          const int first = int(from[r]) - 32 * t, end = int(to[r]) - 32 * t;  // bits first .. end of this word
          if (from[r] <= to[r] && first < 32 && end >= 0)
            bits |= (~0u << max(first, 0)) & (~0u >> (31 - min(end, 31)));
        }
        s.wanted[t] = bits;
      }
      __syncthreads();
      const auto act = [&](float x, int i) {
        const float d = sc.distance(x);
        bool in = false;
#pragma unroll
        for (int r = 0; r < kRanges; ++r) in |= d >= float(from[r]) && d < float(to[r] + 1);
        if (in) take(s, order_key(x, i), unsigned(d), sc.fraction(x));
      };
      // The ranges in logits, |x - mid| <= half, wider by more than all roundings on the way
      // (each within 2^-24 of |top| or far_, eight in sum).
      float mid[kRanges], half[kRanges];
#pragma unroll
      for (int r = 0; r < kRanges; ++r) {
        const float near = float(from[r]) / sc.per, far_ = float(to[r] + 1) / sc.per;
        mid[r] = top - 0.5f * (near + far_);
        half[r] = 0.5f * (far_ - near) + 0x1p-20f * (fabsf(top) + far_);
        if (!(half[r] < 1e38f) || !(fabsf(mid[r]) < 1e38f)) mid[r] = 0.f, half[r] = -kNegInf;
        if (from[r] > to[r]) half[r] = -1.f;
      }
      const auto near_range = [&](float x, int r) { return fabsf(x - mid[r]) <= half[r]; };
      if (!use_k && !use_m)
        row.pick_vectors([&](float x) { return near_range(x, 1) | near_range(x, 3); }, act);
      else
        row.pick_vectors([&](float x) { return near_range(x, 0) | near_range(x, 1) | near_range(x, 2) | near_range(x, 3); }, act);
      __syncthreads();
    }
  }
  Gathered mine;
  mine.order(s, 0, 0);

  // The kept run: its length and mass.
  u64 kept = mass_all;
  unsigned length = count_all;
  if (use_k) {
    const Place p = locate(s, row, sc, mine, Goal{true, u64(top_k)}, count_all, 0);
    kept = p.mass;
    length = p.count;
  }
  if (use_p) {
    const Place p = locate(s, row, sc, mine, goal_p(top_p, kept), count_all, 1);
    kept = p.mass;
    length = p.count;
  }
  if (use_m) {
    // The tokens of bin `far` with w >= min_p stand in front of its others.
    __syncthreads();
    if (t == 0) s.low = 0;
    __syncthreads();
    u64 heavy = 0;
    if (is_wanted(s, far)) {
      const float x = value_of(mine.key);
      if (mine.bin == far && sc.weight_of(x) >= double(min_p)) heavy = packed(sc.fraction(x));
    } else {
      row.template each<2>([&](float x, int) {
        const float d = sc.distance(x);
        if (d >= float(far) && d < float(far + 1) && sc.weight_of(x) >= double(min_p)) heavy += packed(sc.fraction(x));
      });
    }
    if (heavy) atomicAdd(&s.low, heavy);
    __syncthreads();
    const unsigned n = s.count[slot(far)] + count_of(s.low);
    const u64 m = s.mass[slot(far)] + mass_of(weight_of(s.low), run_edge(far / kPerThread) * step(int(far % kPerThread)));
    __syncthreads();
    if (n < length) kept = n == 0 ? mass_of(kOne - loss(0.f), run_edge(0)) : m;  // (n = 0: min_p above 1)
  }
  const Place p = locate(s, row, sc, mine, goal_u(u, kept), count_all, 2);
  if (t == 0) {
    const int token = int(p.key & 0xffffffffu);
    a.tokens[b] = token;
    a.probs[b] = float(sc.weight_of(float(row.p[token])) * (double(kOne) * kMass) / double(kept));
  }
}

}  // namespace

hipError_t sample(const SampleArgs& a, hipStream_t stream) {
  const dim3 grid(unsigned(a.batch)), block(kThreads);
  static LdsLimit limits[2];
  const void* kernel = a.f32 ? reinterpret_cast<const void*>(&sample_kernel<float>) : reinterpret_cast<const void*>(&sample_kernel<f16>);
  const hipError_t e = limits[a.f32].raise(kernel, int(sizeof(SampleLds)));
  if (e != hipSuccess) return e;
  if (a.f32) hipLaunchKernelGGL((sample_kernel<float>), grid, block, sizeof(SampleLds), stream, a);
  else hipLaunchKernelGGL((sample_kernel<f16>), grid, block, sizeof(SampleLds), stream, a);
  return hipGetLastError();
}

}  // namespace tia
