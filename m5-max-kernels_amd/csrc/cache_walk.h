// How many heads a workgroup of the quantised cache's writes and reads walks over, apart from the kernels so that a host
// compiler takes it too.
#pragma once

#include <stdint.h>

namespace m5k {

// As many as leave each compute unit `waves` waves' work.
inline int walk_of(int64_t workgroups, int heads, int threads, int waves) {
  const int64_t w = workgroups * heads * (threads / 64) / (int64_t{256} * waves);
  return static_cast<int>(w < 1 ? 1 : w > 8 ? 8 : w);
}

// Of an append whose workgroups have `threads` threads.  16: sines and cosines are made once a walk (4096 tokens turned,
// 32 heads of q, 8 of k and v of 128, blocks of 64, read back: 36 us; with 8 and 32 waves 36 and 50 us; single tokens
// have too few rows to walk).
inline int append_walk(int64_t tokens, int block, int kv_heads, int heads, int threads) {
  return walk_of(tokens / block, 2 * kv_heads + heads, threads, 16);
}

// Of a read, by 256 threads with 8 channels each.  16: 19569 tokens, 16 heads of 64, INT8 to FP16, with 64 waves 26.3 us
// instead of 24.5, with 128 34.5; 32769 tokens, 8 heads of 128, E4M3 to BF16, the same from 8 to 128.
inline int read_walk(int64_t tokens, int head_dim, int kv_heads) {
  return walk_of((tokens * (head_dim / 8) + 255) / 256, 2 * kv_heads, 256, 16);
}

}  // namespace m5k
