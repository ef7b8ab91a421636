// Slots of random ascending calls (csrc/attention_place.h): enough for all tiles, no more than one a token where a
// group fits a tile, and none without rows where every sequence has one token.  Prints the first violation.
#include <cstdio>
#include <random>
#include <vector>

#include "attention_place.h"

using namespace m5k::attn;

int main() {
  std::mt19937 g(2);
  const auto up_to = [&](int n) { return static_cast<int>(g() % (n + 1)); };
  for (int i = 0; i < 3000; ++i) {
    const int group = 1 + up_to(300), per = i & 1 ? 32 : 128, sequences = 1 + up_to(i % 10 ? 90 : 900);
    const bool single = i % 3 == 0;
    std::vector<int32_t> starts(sequences + 1, 0);
    for (int b = 0; b < sequences; ++b)
      starts[b + 1] = starts[b] + (single ? 1 : i % 3 == 1 ? up_to(1) : up_to(40));
    const int tokens = starts[sequences] + (i % 5 ? 0 : up_to(9));
    if (tokens == 0) continue;
    const int64_t slots = slots_before(tokens, sequences + 1, group, per);
    if (group <= per && slots > tokens) return std::printf("call %d: %lld slots\n", i, static_cast<long long>(slots));
    int64_t end = 0, tiles = 0;
    for (int b = 0; b <= sequences; ++b) {
      const int own = (tokens_of(starts.data(), b, sequences, tokens) * group + per - 1) / per;
      const int first = first_slot(starts.data(), b, tokens, group, per);
      if (first < end) return std::printf("call %d: sequence %d begins inside another\n", i, b), 1;
      end = first + own;
      tiles += own;
    }
    if (end > slots) return std::printf("call %d: %lld slots, the last tile ends at %lld\n", i,
                                        static_cast<long long>(slots), static_cast<long long>(end)), 1;
    const bool tail = starts[sequences] < tokens;  // tokens behind the last sequence share tiles, but not slots
    if (single && group <= per && !tail && tiles != slots) return std::printf("call %d: empty slots\n", i), 1;
  }
  return 0;
}
