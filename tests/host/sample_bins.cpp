// The sampler's packed bins on the CPU: what up to 2^18 tokens of one bin sum up to is
// their count and their weight, wherever in the bin they lie.
#include "../../tinyinfer_amd/csrc/sample_bins.hpp"

#include <cmath>
#include <cstdio>
#include <initializer_list>

using namespace tia::sample_bins;

int main() {
  const double near = std::exp(double(kSlack) / kPerUnit);  // weight of a bin's edge
  for (int step = -1; step <= 1025; ++step) {
    const float fraction = step < 0 ? -kFraction : step > 1024 ? 1.f + kFraction : float(step) / 1024.f;
    const double want = std::exp(-double(fraction) / kPerUnit);
    for (unsigned n : {1u, 511u, 131072u, 258399u, 262143u, 262144u}) {
      u64 sum = 0;
      for (unsigned i = 0; i < n; ++i) sum += packed(fraction);
      if (count_of(sum) != n) return std::printf("%u tokens at %g count as %u\n", n, fraction, count_of(sum)), 1;
      const double got = double(weight_of(sum)) / double(kOne) * near / n;
      // The loss is cut off to 2^-34 and summed in fp32 (three roundings of 2^-24 of it).
      if (std::fabs(got - want) > 0x1p-34 + 3 * 0x1p-24 * 0x1.1p-8 + 0x1p-36)
        return std::printf("%u tokens at %g weigh %.12g each, not %.12g\n", n, fraction, got, want), 1;
    }
    // One likeliest token at the bin's edge, the others behind it.
    u64 sum = packed(0.f);
    for (int i = 1; i < kVocabMax; ++i) sum += packed(fraction);
    if (count_of(sum) != unsigned(kVocabMax)) return std::printf("one and others at %g: %u\n", fraction, count_of(sum)), 1;
  }
  return 0;
}
