// The place of a goal among a bin's tokens on the CPU: the token that the goal falls into,
// and for a goal that their masses do not reach the last of them.
#include "../../tinyinfer_amd/csrc/sample_bins.hpp"

#include <cstdio>
#include <initializer_list>

using namespace tia::sample_bins;

int main() {
  const u64 begin[] = {100, 130, 131, 190}, end = 200;
  const auto thread = [](unsigned i) { return (7 * i + 5) % 1024; };
  for (u64 goal = 101; goal <= 260; ++goal) {
    unsigned best = 0, want = 3;
    for (unsigned i = 0; i < 3; ++i)
      if (begin[i] < goal && goal <= begin[i + 1]) want = i;
    for (unsigned i : {2u, 0u, 3u, 1u}) {
      const unsigned claim = claim_of(begin[i], goal, 70 + i, thread(i));
      if ((claim != 0) != (begin[i] < goal)) return std::printf("claim of %u at %llu\n", i, goal), 1;
      if (claim > best) best = claim;
    }
    if (!best || claimant(best) != thread(want))
      return std::printf("goal %llu (of %llu): thread %u, not %u\n", goal, end, claimant(best), thread(want)), 1;
  }
  // The last rank there is outdoes the one before it, by whichever thread.
  return claim_of(0, 1, kVocabMax - 1, 0) > claim_of(0, 1, kVocabMax - 2, 1023) ? 0 : 1;
}
