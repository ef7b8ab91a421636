// Where the rows of a paged attention call lie: the integer arithmetic that gives a workgroup its sequence, tile and
// tokens, apart from the kernels so that a host compiler takes it too.
//
// The packed rows (token * G + head of its group) of a sequence are cut into tiles of R.  Sequence b owns the slots
// from (starts[b] * G / R) + b on: at least as many as it has tiles, and the first of them is known without the lengths
// of the sequences before it.  The tokens behind the last sequence are sequence number `sequences`, which sees nothing.
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

M5K_PLACE int first_slot(const int32_t* starts, int b, int tokens, int group, int rows_per_tile) {
  return static_cast<int>(int64_t{start_of(starts, b, tokens)} * group / rows_per_tile) + b;
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
