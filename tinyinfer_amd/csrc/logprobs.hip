// Log probabilities of given tokens, a row's entropy and its likeliest tokens.
//
//   m = max x,  Z = sum e^(x - m),  log p(t) = x_t - m - log Z,
//   H = -sum p log p = log Z - (sum e^(x - m) (x - m)) / Z
//
// A workgroup, or several, read a row once.  A wave keeps the largest x it has met and how many
// logits equal it, its lanes the sum of e^(x - m) over the others and sum e^(x - m) (x - m): a
// likely token's log probability, log1p of a small sum, and a sure row's entropy keep their
// digits, and a larger maximum rescales three numbers.
//
// Alternatives, by logit, ties by index.  A thread takes 32 tokens a round; the largest of them
// stands for this piece.  Every wave gives the largest few of its first pieces, and the
// `top`-th of all these is a bar that `top` tokens reach for certain; pieces that reach it are
// listed.  The `top`-th of the list is a second bar, so only the pieces at or above that one,
// `top` and ties, are looked at again.  Where a list does not hold them (many equal logits,
// rising ones) the range of the tokens at or above the bar is cut into runs and read again until
// it does.
//
// What bounds it: memory for hundreds of rows (768 rows of 128257 in fp32, 5 alternatives: 68.4 us, 5.8
// TB/s; of 50257 in fp16 26.2, tokens in place of bytes: fp32 30.9), for a few the chain of latencies (32 rows of 50257 in fp16, 20 alternatives: 14.0 us; about 2.5
// of them launch, 1 the first loads, 2 the bar, 1 a round of the row, 1 sums, 3 the list, 2 joining the
// parts, 1 their order; one row of fp32, 5 alternatives 9.6, none 6.8).  Whole rows take 16.6, and what
// one CU fetches, about 9 bytes a cycle, bounds them: loads two to four rounds ahead, or a quarter
// fewer vector instructions, change nothing.  512 threads: with 256 the 32 rows take 23.1 us.
//
// NaN logits count as -inf.  A row with a +inf has all its probability on the first one, a
// row without a logit above -inf none anywhere: log probabilities of -inf, entropy 0.
#include "common.hpp"
#include "kernels.hpp"
#include "queue_scratch.hpp"

namespace tia {
namespace {

typedef unsigned long long u64;
constexpr int kNoToken = 0x7fffffff;
constexpr float kNegInf = -__builtin_huge_valf(), kLog2e = 1.4426950408889634f;
constexpr int kThreads = 512, kList = 1024, kRuns = 2048, kFirsts = 128;

// A row split over workgroups: each leaves its waves' sums, how many alternatives it has and
// these (or their first `top`), and the last one to arrive joins them.
constexpr int kParts = 16, kPartKeys = 64, kPartCount = 32, kPartList = 36, kPartFloats = 168;
constexpr int kSplitWorkgroups = 256, kSplitRows = kSplitWorkgroups / 2;
static_assert(kParts * kPartKeys == kList && kPartKeys >= kLogprobsTopMax, "a list holds all parts'");
TIA_QUEUE_POOL(lp_pool, kSplitWorkgroups * kPartFloats, kSplitRows)

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

// The largest x of a wave, in every lane, and the sum, by operand modifiers: no trip through LDS.
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp(float old, float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, old), __builtin_bit_cast(int, x), CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ float last_lane(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}
__device__ __forceinline__ float max_of_wave(float x) {
  x = fmaxf(x, dpp<0x111, 0xF>(kNegInf, x));  // 1, 2, 4, 8 lanes back within rows of 16
  x = fmaxf(x, dpp<0x112, 0xF>(kNegInf, x));
  x = fmaxf(x, dpp<0x114, 0xF>(kNegInf, x));
  x = fmaxf(x, dpp<0x118, 0xF>(kNegInf, x));
  x = fmaxf(x, dpp<0x142, 0xA>(kNegInf, x));  // rows 0 and 2's last lane to rows 1 and 3
  x = fmaxf(x, dpp<0x143, 0xC>(kNegInf, x));  // row 1's to rows 2 and 3
  return last_lane(x);
}
__device__ __forceinline__ float sum_of_wave(float x) {
  x += dpp<0x111, 0xF>(0.f, x);
  x += dpp<0x112, 0xF>(0.f, x);
  x += dpp<0x114, 0xF>(0.f, x);
  x += dpp<0x118, 0xF>(0.f, x);
  x += dpp<0x142, 0xA>(0.f, x);
  x += dpp<0x143, 0xC>(0.f, x);
  return last_lane(x);
}

// What a wave knows of the logits it has met: their maximum m and how many equal it (the
// same in all lanes), and per lane over the others rest = sum e^(x - m), spread = sum
// e^(x - m) (x - m).
struct Stats {
  float m, count, rest, spread;
  // To a maximum of at least this one; `counted` of the count are this lane's to carry over.
  // (Differences end at -200, where e^ is 0.)
  __device__ __forceinline__ void raise(float to, float counted) {
    if (m == to) return;
    const float d = fmaxf(m - to, -200.f), f = __builtin_amdgcn_exp2f(d * kLog2e);
    spread = f * fmaf(d, rest + counted, spread);
    rest = f * (rest + counted);
    count = 0.f;
    m = to;
  }
  // x, and their maximum (called by whole waves).
  template <int N>
  __device__ __forceinline__ void add(float (&x)[N], float high) {
    if (__ballot(high > m)) raise(max_of_wave(fmaxf(high, m)), (threadIdx.x & 63) == 0 ? count : 0.f);
    if (__ballot(high == m)) {
      int equal = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        equal += __popcll(__ballot(x[i] == m));
        x[i] = x[i] == m ? kNegInf : x[i];
      }
      count += float(equal);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float d = fmaxf(x[i] - m, -200.f);  // (NaN and -inf too: e^-200 is 0)
      const float e = __builtin_amdgcn_exp2f(d * kLog2e);
      spread = fmaf(d, e, spread);
      rest += e;
    }
  }
};

template <typename T>
struct Vec {
  static constexpr int W = 16 / int(sizeof(T));
  typedef T type __attribute__((ext_vector_type(W)));
  typedef type loose __attribute__((aligned(sizeof(T))));  // (the device allows unaligned vector accesses)
};

template <typename T, int THREADS, int ENTRIES>
struct Lds {
  u64 keys[2][kList];  // two lists, one the other's order
  float firsts[kFirsts];  // the waves' largest first logits
  Stats stats[ENTRIES];
  union {
    unsigned run[kRuns];
    unsigned rank[kList];
  };
  unsigned count, found, pick, above;
  u64 low, high;
};

// The row as threads see it: vector v is tokens W v .., wherever in memory the row starts
// (so an answer does not depend on that), the few behind the last one are one token each of
// the first threads.  A thread takes N tokens, A vectors, a round.
template <typename T, int THREADS, int TOKENS, bool PART>
struct Row {
  static constexpr int W = Vec<T>::W, N = TOKENS, A = N / W;
  const T* p;
  int n, vectors, from = 0, to = 0;
  __device__ __forceinline__ Row(const T* row, int length) : p(row), n(length), vectors(length / W) {}
  __device__ __forceinline__ int rounds() const { return (vectors + A * THREADS - 1) / (A * THREADS); }
  // A part's rounds; the last part has the edge.
  __device__ __forceinline__ void take(int part, int per) {
    from = part * per;
    to = min(from + per, rounds());
  }
  __device__ __forceinline__ int first() const { return PART ? from : 0; }
  __device__ __forceinline__ int last() const { return PART ? to : rounds(); }
  // This thread's token behind the vectors, or -1.
  __device__ __forceinline__ int edge() const {
    const int at = vectors * W + int(threadIdx.x);
    return at < n && last() == rounds() ? at : -1;
  }
  __device__ __forceinline__ int vector(int round, int c) const { return (round * A + c) * THREADS + int(threadIdx.x); }
  __device__ __forceinline__ int token(int round, int i) const { return vector(round, i / W) * W + i % W; }
  // Token i (0 .. N - 1) of a piece, numbered by round and thread (behind the last round: the
  // threads' edges), or -1.
  __device__ __forceinline__ int token_of(int piece, int i) const {
    const int round = piece / THREADS, t = piece % THREADS, v = (round * A + i / W) * THREADS + t;
    if (round == rounds()) return i == 0 ? vectors * W + t : -1;
    return v < vectors ? v * W + i % W : -1;
  }
  __device__ __forceinline__ void load(typename Vec<T>::type (&x)[A], int round) const {
#pragma unroll
    for (int c = 0; c < A; ++c)
      x[c] = __builtin_nontemporal_load(reinterpret_cast<const typename Vec<T>::loose*>(p + min(vector(round, c), vectors - 1) * W));
  }
  // A round's values; -inf past the last vector.
  __device__ __forceinline__ void values(float (&x)[N], const typename Vec<T>::type (&v)[A], int round) const {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = float(v[i / W][i % W]);
    if ((round + 1) * A * THREADS > vectors) {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = vector(round, i / W) < vectors ? x[i] : kNegInf;
    }
  }
  // f(value, index) for every token.
  template <typename F>
  __device__ void each(F f) const {
    const int e = edge();
    if (e >= 0) f(float(p[e]), e);
    for (int r = first(); r < last(); ++r) {
      typename Vec<T>::type x[A];
      load(x, r);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (vector(r, i / W) < vectors) f(float(x[i / W][i % W]), token(r, i));
    }
  }
};

// The list again, for a row of which it does not hold all tokens at or above `bar`: the
// range of their keys is cut into kRuns runs, and the one in which the `top`-th lies is cut
// again, until it and the runs above fit.  (Keys are distinct, so this ends.)
template <typename T, int THREADS, int N, bool PART, int E>
__device__ __forceinline__ void refill(Lds<T, THREADS, E>& s, const Row<T, THREADS, N, PART>& row, int to_list, float bar, unsigned top) {
  u64 low = ~u64(0), high = 0;
  if (threadIdx.x == 0) {
    s.low = low;
    s.high = high;
  }
  __syncthreads();
  row.each([&](float x, int i) {
    if (!(x >= bar)) return;
    const u64 k = key_of(x, i);
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
      if (!(x >= bar)) return;
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
  if (threadIdx.x == 0) s.found = 0;
  __syncthreads();
  row.each([&](float x, int i) {
    if (!(x >= bar)) return;
    const u64 k = key_of(x, i);
    if (k < low) return;
    const unsigned at = atomicAdd(&s.found, 1u);
    if (at < kList) s.keys[to_list][at] = k;
  });
  __syncthreads();
}

// The top-th largest of many >= top numbers, 64 H at most, by every wave for itself.
template <int H>
__device__ __forceinline__ float nth_of(const float* numbers, int many, int top) {
  const int lane = int(threadIdx.x & 63);
  float mine[H], least = kNegInf;
  int above[H];
#pragma unroll
  for (int h = 0; h < H; ++h) {
    mine[h] = lane + 64 * h < many ? numbers[lane + 64 * h] : kNegInf;
    above[h] = 0;
  }
#pragma unroll
  for (int from = 0; from < H; ++from)
#pragma unroll 8
    for (int i = 0; i < min(many - 64 * from, 64); ++i) {
      const float other = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, mine[from]), i));
#pragma unroll
      for (int h = 0; h < H; ++h) above[h] += other > mine[h];
    }
#pragma unroll
  for (int h = 0; h < H; ++h) least = fmaxf(least, lane + 64 * h < many && above[h] < top ? -mine[h] : kNegInf);
  return -max_of_wave(least);
}

// List `from`'s n keys in their order, into the other one; several threads to a key, each comparing it with a part
// of the others.
template <typename T, int THREADS, int E>
__device__ __forceinline__ void sort_list(Lds<T, THREADS, E>& s, int from, unsigned n) {
  const u64* list = s.keys[from];
  const unsigned tid = threadIdx.x;
  unsigned wide = 64;
  while (wide < n) wide *= 2;
  for (unsigned i = tid; i < n; i += THREADS) s.rank[i] = 0;
  __syncthreads();
  const unsigned parts = max(unsigned(THREADS) / wide, 1u), part = tid / wide, chunk = (n + parts - 1) / parts;
  for (unsigned i = tid & (wide - 1); i < n; i += THREADS) {
    const u64 k = list[i];
    const unsigned end = min(n, (part + 1) * chunk);
    unsigned before = 0;
#pragma unroll 8
    for (unsigned o = part * chunk; o < end; ++o) before += list[o] > k;
    if (before) atomicAdd(&s.rank[i], before);
  }
  __syncthreads();
  for (unsigned i = tid; i < n; i += THREADS) s.keys[1 - from][s.rank[i]] = list[i];
  __syncthreads();
}

// One workgroup per row, or `parts` of them with `per` rounds each.
template <typename T, int N, bool SPLIT>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(LogprobsArgs a, int parts, int per) {
  constexpr int THREADS = kThreads, WAVES = THREADS / 64;
  using R = Row<T, THREADS, N, SPLIT>;
  __shared__ Lds<T, THREADS, SPLIT ? kParts * WAVES : WAVES> s;
  const int tid = int(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int line = int(SPLIT ? blockIdx.y : blockIdx.x), part = SPLIT ? int(blockIdx.x) : 0;
  const T* logits = static_cast<const T*>(a.logits) + int64_t(line) * a.vocab;
  R row(logits, a.vocab);
  if constexpr (SPLIT) row.take(part, per);
  const int first_round = row.first(), rounds = row.last(), edge = row.edge();
  typename Vec<T>::type next[R::A];
  if (rounds > first_round) row.load(next, first_round);
  const float edge_x = edge >= 0 ? float(logits[edge]) : kNegInf;
  float x[R::N];
#pragma unroll
  for (int i = 0; i < R::N; ++i) x[i] = kNegInf;
  if (rounds > first_round) row.values(x, next, first_round);
  if (rounds > first_round + 1) row.load(next, first_round + 1);
  const auto largest = [&] {
    float high = x[0];
#pragma unroll
    for (int i = 1; i < R::N; ++i) high = fmaxf(high, x[i]);  // (NaN loses)
    return fmaxf(high, kNegInf);
  };
  float high = largest();

  // The bar: `top` tokens at least are not below it.
  float bar = __builtin_huge_valf();
  if (a.top > 0) {
    if (tid == 0) s.count = s.found = 0;
    // Waves with vectors, how many logits each gives, and all of them.
    const int active = min(max((row.vectors - first_round * R::A * THREADS + 63) / 64, 1), WAVES), each = min((a.top + active - 1) / active + 1, kFirsts / active);
    const int many = each * active;
    if (wave < active) {
      float left = fmaxf(high, edge_x);
      for (int i = 0; i < each; ++i) {
        const float best = max_of_wave(left);
        const u64 who = __ballot(left == best);
        if (lane == 0) s.firsts[each * wave + i] = best;
        if (lane == __builtin_ctzll(who)) left = kNegInf;
      }
    }
    __syncthreads();
    // The least of those with fewer than `top` above them.
    if (many < a.top) {
      bar = kNegInf;
    } else if (many <= 64) {
      bar = nth_of<1>(s.firsts, many, a.top);
    } else {
      bar = nth_of<2>(s.firsts, many, a.top);
    }
    bar = fmaxf(bar, -3.402823466e38f);  // (a logit of -inf is none)
  }
  const auto offer = [&](float v, int piece) {
    const unsigned at = atomicAdd(&s.count, 1u);
    if (at < kList) s.keys[0][at] = key_of(v, piece);
  };

  Stats stats{kNegInf, 0.f, 0.f, 0.f};
  if (high >= bar) offer(high, first_round * THREADS + tid);
  stats.add(x, high);
  for (int r = first_round + 1; r < rounds; ++r) {
    row.values(x, next, r);
    if (r + 1 < rounds) row.load(next, r + 1);
    high = largest();
    if (high >= bar) offer(high, r * THREADS + tid);
    stats.add(x, high);
  }
  if (wave == 0) {  // (the first threads have them)
    float e[1] = {edge_x};
    stats.add(e, fmaxf(edge_x, kNegInf));
    if (edge_x >= bar) offer(edge_x, row.rounds() * THREADS + tid);
  }
  stats.rest = sum_of_wave(stats.rest);
  stats.spread = sum_of_wave(stats.spread);
  if (lane == 0) s.stats[wave] = stats;
  __syncthreads();
  // The pieces' tokens at or above the bar, in the list that it returns.  (The list again is called
  // from one place and compiled into it: a call would give every thread a stack, 11 % of the
  // time of many rows.)
  const auto list = [&] {
    int at_list = 0;
    bool again = s.count > kList;
    if (!again) {
      // (Few pieces are looked at in one go.)
      constexpr unsigned AT_ONCE = THREADS / N, DEEP = 4;
      const unsigned pieces = s.count;
      at_list = 1;
      if (pieces > DEEP * AT_ONCE) {
        sort_list(s, 0, pieces);
        at_list = 0;
        if (pieces >= unsigned(a.top)) bar = value_of(s.keys[1][a.top - 1]);
      }
      const u64* list = s.keys[1 - at_list];
      for (unsigned e = unsigned(tid) / N; e < pieces; e += DEEP * AT_ONCE) {
        int token[DEEP];
        float v[DEEP];
#pragma unroll
        for (unsigned c = 0; c < DEEP; ++c) {
          const u64 k = list[min(e + c * AT_ONCE, pieces - 1)];
          token[c] = e + c * AT_ONCE < pieces && value_of(k) >= bar ? row.token_of(index_of(k), tid % N) : -1;
        }
        if (__ballot(token[0] >= 0) == 0) break;  // (none from here on: they are in order, or this is the only go)
#pragma unroll
        for (unsigned c = 0; c < DEEP; ++c) v[c] = token[c] >= 0 ? float(logits[token[c]]) : kNegInf;
#pragma unroll
        for (unsigned c = 0; c < DEEP; ++c)
          if (v[c] >= bar) {
            const unsigned at = atomicAdd(&s.found, 1u);
            if (at < kList) s.keys[at_list][at] = key_of(v[c], token[c]);
          }
      }
      __syncthreads();
      again = s.found > kList;
    }
    if (__builtin_expect(again, 0)) refill(s, row, at_list, bar, unsigned(a.top));
    return at_list;
  };
  int at_list = 0;
  if constexpr (SPLIT) {
    unsigned found = 0;
    if (a.top > 0) {
      at_list = list();
      found = s.found;
      if (found > kPartKeys) {
        sort_list(s, at_list, found);
        at_list = 1 - at_list;
        found = unsigned(a.top);
      }
    }
    const int slot = queue_slot_resolve(lp_pool_keys, lane < kQueueSlots ? lp_pool_keys[lane] : 0ull);
    float* const pool = lp_pool_data[slot];
    const auto rsrc = agent_rsrc(pool, uint32_t(sizeof(lp_pool_data[0])));
    float* const mine = pool + (line * parts + part) * kPartFloats;
    const auto keys_of = [](float* at) { return reinterpret_cast<u64*>(at + kPartList); };
    if (tid < WAVES) {
      const Stats& w = s.stats[tid];
      st_agent4(rsrc, uint32_t(((line * parts + part) * kPartFloats + 4 * tid) * 4), f32x4_t{w.m, w.count, w.rest, w.spread});
    }
    if (tid == 0) st_agent(mine + kPartCount, __builtin_bit_cast(float, found));
    if (unsigned(tid) < found)
      __hip_atomic_store(keys_of(mine) + tid, s.keys[at_list][tid], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    unsigned* const counter = lp_pool_ctr[slot] + line * kCounterStride;
    if (!wg_arrive_last(counter, parts)) return;
    depart(counter);
    float* const all = pool + line * parts * kPartFloats;
    if (tid < parts * WAVES) {
      const f32x4_t w = ld_agent4(rsrc, uint32_t(((line * parts + tid / WAVES) * kPartFloats + 4 * (tid % WAVES)) * 4));
      s.stats[tid] = Stats{w[0], w[1], w[2], w[3]};
    }
    if (tid == 0) s.found = 0;
    u64 keys[kList / THREADS];
    bool held[kList / THREADS];
#pragma unroll
    for (int i = 0; i < kList / THREADS; ++i) {
      const int at = i * THREADS + tid, from = min(at / kPartKeys, parts - 1);
      float* const theirs = all + from * kPartFloats;
      keys[i] = __hip_atomic_load(keys_of(theirs) + at % kPartKeys, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      held[i] = at / kPartKeys < parts && unsigned(at % kPartKeys) < __builtin_bit_cast(unsigned, ld_agent(theirs + kPartCount));
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kList / THREADS; ++i)
      if (held[i]) s.keys[0][atomicAdd(&s.found, 1u)] = keys[i];
    at_list = 0;
  }
  // (Every LANES lanes have all of the waves' sums.)
  constexpr int ENTRIES = SPLIT ? kParts * WAVES : WAVES, LANES = SPLIT ? 64 : WAVES;
  float m = kNegInf, count = 0.f, rest = 0.f, spread = 0.f;
  if constexpr (SPLIT) {
    const int entries = parts * WAVES;
    Stats w[ENTRIES / LANES];
#pragma unroll
    for (int h = 0; h < ENTRIES / LANES; ++h) {
      w[h] = lane + LANES * h < entries ? s.stats[lane + LANES * h] : Stats{kNegInf, 0.f, 0.f, 0.f};
      m = fmaxf(m, w[h].m);
    }
    m = max_of_wave(m);
#pragma unroll
    for (int h = 0; h < ENTRIES / LANES; ++h) {
      w[h].raise(m, w[h].count);
      count += w[h].count, rest += w[h].rest, spread += w[h].spread;
    }
  } else {
#pragma unroll
    for (int w = 0; w < WAVES; ++w) m = fmaxf(m, s.stats[w].m);
    stats = s.stats[lane % WAVES];
    stats.raise(m, stats.count);
    count = stats.count, rest = stats.rest, spread = stats.spread;
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    count += __shfl_xor(count, o, 64);
    rest += __shfl_xor(rest, o, 64);
    spread += __shfl_xor(spread, o, 64);
  }

  const bool none = m == kNegInf, sure = m == __builtin_huge_valf();
  const float log_z = logf(count) + log1pf(rest / count);
  int first = kNoToken;  // sure: the first +inf
  if (sure) {
    if (tid == 0) s.pick = unsigned(kNoToken);
    __syncthreads();
    for (int i = tid; i < a.vocab; i += THREADS)
      if (float(logits[i]) == __builtin_huge_valf()) {
        atomicMin(&s.pick, unsigned(i));
        break;
      }
    __syncthreads();
    first = int(s.pick);
  }
  const auto log_p = [&](float v, int i) {
    if (sure) return i == first ? 0.f : kNegInf;
    return v > kNegInf ? (v - m) - log_z : kNegInf;
  };
  if (tid == 0) a.entropy[line] = none || sure ? 0.f : log_z - spread / (count + rest);
  for (int i = tid; i < a.given; i += THREADS) {
    const int64_t at = int64_t(line) * a.given + i;
    const int token = a.tokens[at];
    a.logprobs[at] = token >= 0 && token < a.vocab ? log_p(float(logits[token]), token) : kNegInf;
  }
  if (a.top == 0) return;
  if constexpr (!SPLIT) at_list = list();
  if constexpr (SPLIT) __syncthreads();
  const unsigned n = s.found;
  sort_list(s, at_list, n);
  const int64_t out = int64_t(line) * a.top;
  for (unsigned i = unsigned(tid); i < unsigned(a.top); i += THREADS) {
    const u64 k = i < n ? s.keys[1 - at_list][i] : 0;
    a.top_tokens[out + i] = i < n ? index_of(k) : kNoToken;
    a.top_logprobs[out + i] = i < n ? log_p(value_of(k), index_of(k)) : kNegInf;
  }
}

// Tokens of a thread's piece: 16, or 32 from here on, fewer pieces to list and more registers.  us,
// with 16 and 32: one row of 50257 in fp32, 5 alternatives 9.6 and 10.4, 768 of them 31.9 and 38.1; 768
// whole rows of 128257 84 and 80, with 64 alternatives 466 (the list overflows) and 127.
constexpr int kWideVocab = 65536;
static_assert((1 << 18) <= kParts * 32 * kThreads && kWideVocab <= kParts * 16 * kThreads, "rounds of the longest rows");

// Rows that leave CUs idle are split over as many workgroups as there are CUs, with as few rounds each
// as that allows: a CU fetches 9 bytes a cycle, and bringing the parts together costs about 2 us.
// us, split against whole: fp32, 50257 tokens, 5 alternatives, 1 / 32 / 64 rows 9.6 / 10.7 / 12.5 and 12.0 /
// 14.0 / 14.4; 128257 tokens, 1 / 32 / 128 rows (of two parts) 11.5 / 12.9 / 22.2 and 20.1 / 22.4 / 23.8; 30000
// tokens (4 rounds), 1 / 64 rows 9.8 / 10.7 and 10.4 / 11.8.  Not below 4 rounds (20000 tokens, 1 / 32
// rows 9.8 / 10.5 and 9.1 / 10.6), nor in two parts below 8 (50257, 128 rows 14.9 and 14.5) but for many
// alternatives (64: 25.8 and 35.0).  These are ordered by every part: two rounds at least (64 of 50257,
// 32 rows 19.8, with one 23.0, whole 33.7).
template <typename T, int N>
void launch(const LogprobsArgs& a, hipStream_t stream) {
  constexpr int W = Vec<T>::W, ROUND = N / W * kThreads;
  const int rounds = (a.vocab / W + ROUND - 1) / ROUND;
  int per = a.top > kPartKeys / 2 ? 2 : 1;
  while (per < rounds && int64_t(a.batch) * ((rounds + per - 1) / per) > kSplitWorkgroups) ++per;
  const int parts = (rounds + per - 1) / per;
  if (rounds >= 4 && parts >= 2 && (parts > 2 || rounds >= 8 || a.top > kPartKeys / 2))
    hipLaunchKernelGGL((logprobs_kernel<T, N, true>), dim3(unsigned(parts), unsigned(a.batch)), dim3(kThreads), 0, stream, a, parts, per);
  else
    hipLaunchKernelGGL((logprobs_kernel<T, N, false>), dim3(unsigned(a.batch)), dim3(kThreads), 0, stream, a, 1, 0);
}

}  // namespace

hipError_t logprobs(const LogprobsArgs& a, hipStream_t stream) {
  const bool wide = a.vocab > kWideVocab;
  if (a.f32) wide ? launch<float, 32>(a, stream) : launch<float, 16>(a, stream);
  else wide ? launch<f16, 32>(a, stream) : launch<f16, 16>(a, stream);
  return hipGetLastError();
}

}  // namespace tia
