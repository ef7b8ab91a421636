// Where the rows of a paged attention call lie: the integer arithmetic that gives a workgroup its sequence, tile and
// tokens, apart from the kernels so that a host compiler takes it too.
//
// The packed rows (token * G + head of its group) of a sequence are cut into tiles of R.  Sequence b owns the slots
// from min(starts[b] * ceil(G / R), starts[b] * G / R + b) on: both grow by its tiles at least, so that it owns as
// many, and the first of them is known without the lengths of the sequences before it.  The first term leaves single
// tokens no slot without rows (see slots_before).  The tokens behind the last sequence are sequence number
// `sequences`, which sees nothing.
//
// Starts lie on the device and nothing checks them.  In any order and of any value they are taken as cut to [0,
// tokens]; a slot then finds some sequence, perhaps one that does not own it, and has rows only if its tile is one of
// that sequence's: every row that is read or written is a row of the call.
#pragma once

#include <stdint.h>

#ifdef __HIP__
#include <hip/hip_runtime.h>
#define M5K_PLACE __host__ __device__ __forceinline__
#else
#define M5K_PLACE inline
#endif

namespace m5k {
namespace attn {

// First token of sequence b.
M5K_PLACE int start_of(const int32_t* starts, int b, int tokens) {
  const int s = b == 0 ? 0 : starts[b];
  return s < 0 ? 0 : s > tokens ? tokens : s;
}

// Its tokens: up to the next sequence's first one.
M5K_PLACE int tokens_of(const int32_t* starts, int b, int sequences, int tokens) {
  const int n = (b == sequences ? tokens : start_of(starts, b + 1, tokens)) - start_of(starts, b, tokens);
  return n < 0 ? 0 : n;
}

// Slots of `sequences` sequences that have `tokens` tokens together.  Workgroups go to parts of the chip in turn, and
// wait for their part even while another has room: empty slots in between, of no regular distance, let some parts have
// more work than others.  (64 single tokens over 4096 keys each, 8 key heads, E4M3, groups of 8 and of 7 query heads,
// by the second term alone: 110 and 132 us.)  Equal lengths gain or stay, in 16 bits too: 56 on 8 heads of 128, 64
// sequences of 300 / 1000 / 4000 keys by the second term alone 25.5 / 69.5 / 247 us, so 19.2 / 53.7 / 188; 128 of 1000
// 116 and 102; 24 of 2000 46.8 and 47.7.  Unequal ones go either way, by which of the long ones share a compute unit:
// of 8 draws for each of 16 to 200 sequences, at random up to 8190 keys or spread over the logarithm from 32, the time
// by both terms over that by the second alone is 0.74 to 1.30 in 16 bits, 0.79 to 1.14 in E4M3, 0.74 to 1.23 in INT8;
// its mean over the draws of a kind 0.93 to 1.04, and over all of them 0.996, 0.987 and 0.991.
M5K_PLACE int64_t slots_before(int64_t tokens, int64_t sequences, int group, int rows_per_tile) {
  const int64_t each = tokens * ((group + rows_per_tile - 1) / rows_per_tile);
  const int64_t packed = tokens * group / rows_per_tile + sequences;
  return each < packed ? each : packed;
}
M5K_PLACE int first_slot(const int32_t* starts, int b, int tokens, int group, int rows_per_tile) {
  return static_cast<int>(slots_before(start_of(starts, b, tokens), b, group, rows_per_tile));
}

// The last b of [0, n) whose first slot does not lie behind a slot, 64 probes at a time: count(lo, left, apart) says
// for how many of lo, lo + apart, ... below lo + left (64 at most) that holds.  Ascending starts make those the first.
template <class Count>
M5K_PLACE int sequence_of_slot(int n, Count count) {
  int lo = 0, left = n;
  while (left > 1) {
    const int apart = (left + 63) >> 6, below = count(lo, left, apart);
    const int at = below > 1 ? (below - 1) * apart : 0;
    lo += at;
    left = left - at < apart ? left - at : apart;
  }
  return lo;
}

// Whether a sequence of `rows` rows has the tile.  A slot of descending starts can lie before its sequence's first one.
M5K_PLACE bool tile_has_rows(int tile, int rows, int rows_per_tile) {
  return tile >= 0 && tile < (rows + rows_per_tile - 1) / rows_per_tile;
}

}  // namespace attn
}  // namespace m5k
