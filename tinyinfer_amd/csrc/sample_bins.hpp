// The whole numbers in which the sampler holds a bin of tokens: count << 45 | sum of
// losses, and what of that fits.  Host and device (constexpr).
#pragma once

namespace tia {
namespace sample_bins {

typedef unsigned long long u64;

constexpr int kVocabMax = 1 << 18;
constexpr double kPerUnit = 256.0;  // bins per unit of (max - logit) / T
constexpr int kCountShift = 45;     // a bin: count << 45 | sum of losses
constexpr u64 kOne = u64(1) << 34;  // weight of a token at its bin's near edge
constexpr double kMass = 1024.0;    // a mass: weight * e^(-b/256) * 2^10
// A token's fraction, the part of its distance behind its bin's near edge, lies in
// [-kFraction, 1 + kFraction] (its roundings: 2^-12 of the product, and 1.5 times 2^-11 of
// what the fp32 distance and scale leave out).  Losses count from kSlack in front of the
// edge on, so that none is negative.
constexpr float kFraction = 1.f / 1024 + 1.f / (1 << 20);
constexpr float kSlack = 1.f / 64;

// (1 - e^(-f/256)) 2^34 of a fraction f, to its terms of third order (the fourth is below
// 2^-36 of a weight).
constexpr unsigned loss(float fraction) {
  constexpr double h = 1.0 / kPerUnit, one = double(kOne);
  const float f = fraction + kSlack;
  return unsigned(f * (f * (f * float(one * h * h * h / 6) + float(-one * h * h / 2)) + float(one * h)));
}
constexpr u64 packed(float fraction) { return (u64(1) << kCountShift) + loss(fraction); }
constexpr unsigned count_of(u64 packed) { return unsigned(packed >> kCountShift); }
constexpr u64 weight_of(u64 packed) { return count_of(packed) * kOne - (packed & ((u64(1) << kCountShift) - 1)); }

// A whole vocabulary in one bin: its losses stay below the count (0.51 of 2^45), its count
// within 64 bits, the mass of as many tokens too.
static_assert(kFraction < kSlack, "a loss is not negative");
static_assert(u64(kVocabMax) * loss(1.f + kFraction) < u64(1) << kCountShift, "the losses of a bin reach its count");
static_assert(u64(kVocabMax) <= ~u64(0) >> kCountShift, "the count of a bin");
static_assert(double(kVocabMax) * double(kOne) * kMass < 9.2e18, "the mass of a row");

// The place a goal asks for is the last token that begins in front of it.  What a gathered
// token, number `thread` of at most 1024, of `rank` in its row's order, claims: 0 if it
// begins at the goal or behind, else the more the later it stands.  The largest claim wins,
// so there is a place wherever masses that disagree would end (a token in front of the goal
// is enough), and it is a gathered token.
constexpr unsigned claim_of(u64 begin, u64 goal, unsigned rank, unsigned thread) {
  return begin < goal ? (rank + 1) << 10 | thread : 0;
}
constexpr unsigned claimant(unsigned claim) { return claim & 1023; }
static_assert(unsigned(kVocabMax) <= ~0u >> 10, "a rank in a claim");

}  // namespace sample_bins
}  // namespace tia
