// Every slot of random calls through csrc/attention_place.h: with starts in any order and of any value the rows that a
// tile has are rows of the call; with ascending ones every row belongs to one tile.  Prints the first violation.
#include <cstdio>
#include <random>
#include <vector>

#include "attention_place.h"

using namespace m5k::attn;

static int check(const std::vector<int32_t>& starts, int tokens, int group, int per, bool ascending) {
  const int sequences = static_cast<int>(starts.size()) - 1;
  const int slots = static_cast<int>(int64_t{tokens} * group / per) + sequences + 1;
  std::vector<int> seen(static_cast<size_t>(tokens) * group, 0);
  for (int slot = 0; slot < slots; ++slot) {
    const auto probes = [&](int lo, int left, int apart) {
      int below = 0;
      for (int lane = 0; lane < 64; ++lane)
        below += lane * apart < left && first_slot(starts.data(), lo + lane * apart, tokens, group, per) <= slot;
      return below;
    };
    const int seq = sequence_of_slot(sequences + 1, probes);
    if (seq < 0 || seq > sequences) return std::printf("slot %d: sequence %d\n", slot, seq);
    const int rows = tokens_of(starts.data(), seq, sequences, tokens) * group;
    const int tile = slot - first_slot(starts.data(), seq, tokens, group, per);
    if (!tile_has_rows(tile, rows, per)) continue;
    for (int64_t r = int64_t{tile} * per; r < int64_t{tile + 1} * per; ++r) {
      if (r >= rows) break;
      const int64_t at = int64_t{start_of(starts.data(), seq, tokens)} * group + r;  // token * group + head
      if (r < 0 || at < 0 || at >= int64_t{tokens} * group)
        return std::printf("slot %d: sequence %d of %d rows, row %lld\n", slot, seq, rows, static_cast<long long>(r));
      ++seen[at];
    }
  }
  if (ascending)
    for (size_t i = 0; i < seen.size(); ++i)
      if (seen[i] != 1) return std::printf("row %zu in %d tiles\n", i, seen[i]);
  return 0;
}

int main() {
  std::mt19937 g(1);
  const auto up_to = [&](int n) { return static_cast<int>(g() % (n + 1)); };
  if (check({0, 70, 3, 100}, 100, 8, 32, false) || check({0, 1000, 2}, 1000, 8, 128, false)) return 1;
  for (int i = 0; i < 4000; ++i) {
    const int group = 1 + up_to(15), per = i & 1 ? 32 : 128, sequences = 1 + up_to(i % 10 ? 9 : 300);
    const int tokens = 1 + up_to(i % 7 ? 200 : 2000);
    std::vector<int32_t> starts(sequences + 1, 0);
    const bool ascending = i % 4 == 0, wild = i % 4 == 1;
    int32_t at = 0;
    for (int b = 1; b <= sequences; ++b) {
      at = ascending ? at + up_to((tokens - at) / 2) : up_to(tokens);
      starts[b] = wild ? static_cast<int32_t>(g()) : at;
    }
    if (!ascending) starts[0] = wild ? static_cast<int32_t>(g()) : up_to(tokens);
    if (check(starts, tokens, group, per, ascending)) return std::printf("call %d\n", i), 1;
  }
  return 0;
}
