// A paged cache in 8 bits: written as it is quantised, and read back.
//
// A block of up to 128 tokens of one head shares a power of two 2^e: the least that brings the block's largest
// magnitude to Q or below (Q = 448 for E4M3, 127 for INT8).  x 2^-e is exact, so that a code, the nearest of its format
// with ties to even, depends on nothing but the value and e, and code 2^e is exact in BF16.  A power of two costs E4M3
// nothing (its relative step is the same everywhere) and INT8 up to one bit of eight.
//
// Append.  A workgroup has one block of one operand and walks over heads: 8 channels a thread and pass, all of the
// block's rows in its registers between the maximum and the codes, so that each value is read once.  Only the block
// that a sequence's first new token falls into can hold older ones; it keeps the larger exponent, and where that grows
// the old codes are rounded again under it.  Keys are turned in 64 bits: in 32, about one code in 10^6, next to a
// border, would be another one than the formula's.  The result enters FP32 rounded to odd, which a second rounding to
// fewer bits cannot tell from the 64-bit number.  Sines and cosines stand in LDS for all heads of the walk.
//
// What bounds it.  Single tokens: a chain of dependent loads (sequence, length, page, exponent) and the angles in 64
// bits: 64 tokens, 8 key heads and 56 query heads of 128 take 7.4 us by graph replay (7.9 in a kernel trace), 5.9
// without the queries, 4.7 without turning.  Chunks: 4096 tokens, 32 heads of 64, FP16 to INT8, 15.7 us in a kernel
// trace (14.8 the least), 3.2 TB/s of 4.9: a barrier a head, with one head's loads ahead of it, and two waves a SIMD,
// which wait for 65% of their cycles.
#include "attention_place.h"
#include "cache_walk.h"
#include "fast_div.h"
#include "m5k_common.h"
#include "rope_turn.h"

namespace m5k {
namespace {

constexpr int THREADS = 256;
constexpr int BLOCK_MAX = 128;  // tokens of a block
constexpr int Q_HEADS = 4;      // heads of q whose rows are under way at once
constexpr int READ_HEADS = 4;   // heads of a read

// ---- codes ----------------------------------------------------------------------------------------

// Exponent byte of a block whose largest magnitude is `top`, infinity where a value is not finite.  Q = m 2^k: the
// mantissa of `top` above m's carries into the exponent.
template <int MODE>
__device__ __forceinline__ int exponent_of(float top) {
  if (top == __builtin_inff()) return 255;
  constexpr uint32_t MANTISSA = MODE == M5K_QUANT_FP8 ? 0x600000u : 0x7E0000u;  // 1.75 2^8, 1.984375 2^6
  constexpr int K = MODE == M5K_QUANT_FP8 ? 8 : 6;
  const int e = static_cast<int>((__float_as_uint(top) + (0x7FFFFFu - MANTISSA)) >> 23) - K;
  return e < 0 ? 0 : e;
}

// 2^(127 - byte) and 2^(byte - 127).
__device__ __forceinline__ float unit_of(int byte) {
  return __uint_as_float(byte >= 254 ? 0x00400000u : static_cast<uint32_t>(254 - byte) << 23);
}
__device__ __forceinline__ float scale_of(int byte) {
  return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7FC00000u : static_cast<uint32_t>(byte) << 23);
}

// Codes of 8 values whose magnitudes are at most Q.
template <int MODE>
__device__ __forceinline__ uint2 encode8(const float (&x)[8]) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (MODE == M5K_QUANT_FP8) {
      int c = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false);
      w[i] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], c, true));
    } else {
      uint32_t t[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) t[j] = __float_as_uint(x[4 * i + j] + 0x1.8p23f);  // a whole number, ties to even
      w[i] = __builtin_amdgcn_perm(t[1], t[0], 0x0C0C0400u) | __builtin_amdgcn_perm(t[3], t[2], 0x04000C0Cu);
    }
  }
  return make_uint2(w[0], w[1]);
}

// What 4 codes stand for before their scale.
template <int MODE>
__device__ __forceinline__ void decode4(uint32_t w, float (&x)[4]) {
  if constexpr (MODE == M5K_QUANT_FP8) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
    x[0] = lo[0];
    x[1] = lo[1];
    x[2] = hi[0];
    x[3] = hi[1];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = static_cast<float>(static_cast<int>(w << (24 - 8 * j)) >> 24);
  }
}

// ---- turns ----------------------------------------------------------------------------------------

// Cosine and sine of a, times magnitude, to a few units of 64 bits' last place while a stays below 2^30: the nearest
// multiple of pi / 2 taken off in two parts, Taylor series of the rest (first terms left out below 1e-17).
__device__ __forceinline__ double2 turn64(double a, double magnitude) {
  const double q = rint(a * 0.63661977236758134308);  // 2 / pi
  double r = __builtin_fma(-q, 1.57079632679489655800, a);
  r = __builtin_fma(-q, 6.12323399573676603587e-17, r);
  const double z = r * r;
  double s = 1.0 / 355687428096000.0;
  s = __builtin_fma(z, s, -1.0 / 1307674368000.0);
  s = __builtin_fma(z, s, 1.0 / 6227020800.0);
  s = __builtin_fma(z, s, -1.0 / 39916800.0);
  s = __builtin_fma(z, s, 1.0 / 362880.0);
  s = __builtin_fma(z, s, -1.0 / 5040.0);
  s = __builtin_fma(z, s, 1.0 / 120.0);
  s = __builtin_fma(z, s, -1.0 / 6.0);
  s = __builtin_fma(r * z, s, r);
  double c = 1.0 / 20922789888000.0;
  c = __builtin_fma(z, c, -1.0 / 87178291200.0);
  c = __builtin_fma(z, c, 1.0 / 479001600.0);
  c = __builtin_fma(z, c, -1.0 / 3628800.0);
  c = __builtin_fma(z, c, 1.0 / 40320.0);
  c = __builtin_fma(z, c, -1.0 / 720.0);
  c = __builtin_fma(z, c, 1.0 / 24.0);
  c = __builtin_fma(z, c, -0.5);
  c = __builtin_fma(z, c, 1.0);
  const int quarter = static_cast<int>(static_cast<int64_t>(q) & 3);
  const double cosine = quarter & 1 ? s : c, sine = quarter & 1 ? c : s;
  return make_double2(quarter == 1 || quarter == 2 ? -cosine * magnitude : cosine * magnitude,
                      quarter >= 2 ? -sine * magnitude : sine * magnitude);
}

// FP32 rounded to odd: cut off, with the last bit set where anything was.  Infinity beyond FP32's range.
__device__ __forceinline__ float round_to_odd(double v) {
  const float f = static_cast<float>(v);
  const double back = f;
  if (!(fabs(back) < __builtin_inf()) || back == v) return f;
  const uint32_t u = __float_as_uint(f);
  return __uint_as_float((u - (fabs(back) > fabs(v) ? 1u : 0u)) | 1u);
}

// ---- append ---------------------------------------------------------------------------------------

struct Operand {
  const void* src;
  uint8_t *codes, *exps;
  int64_t src_head, src_token, page, head, slot, exp_page, exp_head;
};

// A number that the device divides by.
struct Divisor {
  uint32_t magic, shift;
  int value;
};
Divisor divisor(int value) {
  Divisor d;
  d.value = value;
  magic_of(static_cast<uint32_t>(value), d.magic, d.shift);
  return d;
}
__device__ __forceinline__ int over(int n, const Divisor& d) { return static_cast<int>(fast_div(n, d.magic, d.shift)); }

struct AppendArgs {
  Operand op[2];  // K, V
  const void* q;
  void* q_out;
  int64_t q_head, q_token;
  const int32_t *table, *starts, *context;
  const double* frequencies;
  int64_t table_width;
  int tokens, kv_heads, heads, pairs, interleaved, sequences, pages, walk, slots;
  Divisor block, page_size, groups, q_groups;
  double magnitude;
};

// First block slot of a sequence.  Its n tokens touch no more than min(n, floor(n / block) + 2) blocks, wherever the
// first one falls, and both terms of the minimum here grow by at least that much from a sequence to the next.
__host__ __device__ __forceinline__ int block_slots(int tokens, int whole_blocks, int sequences) {
  const int blocks = whole_blocks + 2 * sequences;
  return tokens < blocks ? tokens : blocks;
}
__device__ __forceinline__ int first_block_slot(const AppendArgs& a, int b) {
  const int start = attn::start_of(a.starts, b, a.tokens);
  return block_slots(start, over(start, a.block), b);
}

// Where a pair's cosine and sine stand in its row of LDS: the first of each half-layout chunk side by side, then the
// second and so on, so that the lanes of a row read neighbours.
template <int D>
__device__ __forceinline__ int turn_at(int pair) {
  return (pair & 7) * (D / 16) + (pair >> 3);
}

// Channels c0 .. c0 + 7 of a row, turned: `turns` holds the row's cosines and sines a pair.  put(i, own, other, turn,
// turns) gets each channel, its partner, and what they are multiplied by.  D / 8 neighbouring lanes, all of them
// active, have the row's chunks.
template <int DT, int D, class Turn, class F>
__device__ __forceinline__ void turned8(const void* src, int64_t row, int c0, const Turn* turns, int pairs,
                                        bool interleaved, const float (&x)[8], F put) {
  float other[8];
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 8; ++i) other[i] = x[i ^ 1];
  } else if (pairs % 8 == 0) {  // a chunk's partners are a chunk, of a lane nearby
    const int from = c0 < pairs ? c0 + pairs : c0 < 2 * pairs ? c0 - pairs : c0;
    const int lane = (threadIdx.x & 63 & ~(D / 8 - 1)) + from / 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) other[i] = __shfl(x[i], lane);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = c0 + i;
      other[i] = d < 2 * pairs ? load_elem<DT>(src, row + (d < pairs ? d + pairs : d - pairs)) : 0.0f;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = c0 + i;
    if (d >= 2 * pairs) {
      put(i, x[i], 0.0f, Turn{}, false);
    } else {
      const Turn t = turns[turn_at<D>(interleaved ? d >> 1 : d < pairs ? d : d - pairs)];
      put(i, x[i], other[i], Turn{t.x, (interleaved ? i & 1 : d >= pairs) ? t.y : -t.y}, true);
    }
  }
}

// 8 values as DT at element `at`, 16-byte aligned.
template <int DT>
__device__ __forceinline__ void store8(void* p, int64_t at, const float (&x)[8]) {
  if constexpr (DT == M5K_F32) {
    float4* d = reinterpret_cast<float4*>(static_cast<float*>(p) + at);
    d[0] = make_float4(x[0], x[1], x[2], x[3]);
    d[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == M5K_BF16) u[i] = f32x2_to_bf16x2(x[2 * i], x[2 * i + 1]);
      else u[i] = f32_to_f16_bits(x[2 * i]) | (f32_to_f16_bits(x[2 * i + 1]) << 16);
    }
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + at) = make_uint4(u[0], u[1], u[2], u[3]);
  }
}

// T threads, as many as the block's rows have chunks of 8 channels, in PASSES passes where that is more than 1024: the
// cosines and sines of a block of 64 tokens fill 64 KiB, and 16 waves share them.  TURNED: K and Q are turned.
template <int DT, int D, int MODE, int T, int PASSES, bool TURNED>
__global__ __launch_bounds__(T) void append_codes(const AppendArgs a) {
  constexpr int CH = D / 8, RPP = T / CH;  // chunks of a row, rows of a pass
  constexpr int ROWS = PASSES * RPP, PAIRS = D / 2, TURNS = T / PAIRS;  // TURNS: rows that get theirs at a time
  __shared__ double2 turns[TURNED ? ROWS * PAIRS : 1];
  float2* const turns32 = reinterpret_cast<float2*>(turns);  // of Q
  __shared__ double radians[TURNED ? PAIRS : 1];
  __shared__ float tops[2][T / 64];
  __shared__ int places[TURNED ? ROWS : 1];
  const int tid = threadIdx.x, c0 = tid % CH * 8, row = tid / CH;
  // Workgroups of K, then V, then Q; of each, the heads' groups of a slot side by side.
  const int kv = a.slots * a.groups.value, id = blockIdx.x, role = id < kv ? 0 : id < 2 * kv ? 1 : 2;
  const Divisor& groups = role == 2 ? a.q_groups : a.groups;
  const int slot = over(id - role * kv, groups), walk0 = (id - role * kv - slot * groups.value) * a.walk;
  const int head1 = min(walk0 + a.walk, role == 2 ? a.heads : a.kv_heads);
  const bool turn = TURNED && role != 1;
  const int pair = tid % PAIRS;
  if constexpr (TURNED) {
    if (turn && tid < a.pairs) radians[tid] = a.frequencies[tid];
  }

  if (role == 2) {
    // Rows of q by token; those behind the last sequence are 0.
    if constexpr (TURNED) {
      const int token0 = slot * ROWS;
      if (tid < ROWS && token0 + tid < a.tokens) {
        const int token = token0 + tid;
        int lo = 0, hi = a.sequences;
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (a.starts[mid] <= token) lo = mid;
          else hi = mid;
        }
        const int s = a.starts[lo], e = a.starts[lo + 1];
        places[tid] = token >= s && token < e ? a.context[lo] - (e - token) : INT32_MIN;
      }
      __syncthreads();
      for (int r = tid / PAIRS; r < ROWS && token0 + r < a.tokens && pair < a.pairs; r += TURNS) {
        float2& t = turns32[r * PAIRS + turn_at<D>(pair)];
        turn_of(places[r], radians[pair], static_cast<float>(a.magnitude), t.x, t.y);
      }
      __syncthreads();
#pragma unroll
      for (int pass = 0; pass < PASSES; ++pass) {
        const int r = pass * RPP + row, token = token0 + r;
        if (token >= a.tokens) break;
        const bool known = places[r] != INT32_MIN;
        const auto put = [&](int h, const float (&x)[8]) __attribute__((always_inline)) {
          float y[8];
          turned8<DT, D>(a.q, h * a.q_head + token * a.q_token, c0, turns32 + r * PAIRS, a.pairs, a.interleaved, x,
                         [&](int i, float own, float other, float2 u, bool turns_it) {
            const float z = turns_it ? own * u.x + other * u.y : own;
            y[i] = known ? z : 0.0f;
          });
          store8<DT>(a.q_out, (int64_t{h} * a.tokens + token) * D + c0, y);
        };
        int h = walk0;
        for (; h + Q_HEADS <= head1; h += Q_HEADS) {
          float x[Q_HEADS][8];
#pragma unroll
          for (int j = 0; j < Q_HEADS; ++j) load8<DT>(a.q, (h + j) * a.q_head + token * a.q_token + c0, x[j]);
#pragma unroll
          for (int j = 0; j < Q_HEADS; ++j) put(h + j, x[j]);
        }
        for (; h < head1; ++h) {
          float x[8];
          load8<DT>(a.q, h * a.q_head + token * a.q_token + c0, x);
          put(h, x);
        }
      }
    }
    return;
  }

  const Operand& op = a.op[role];
  const auto probes = [&](int lo, int left, int apart) {
    const int probe = (tid & 63) * apart;
    const bool below = probe < left && first_block_slot(a, lo + probe) <= slot;
    return __popcll(__builtin_amdgcn_ballot_w64(below));
  };
  const int b = __builtin_amdgcn_readfirstlane(attn::sequence_of_slot(a.sequences, probes));
  const int n = attn::tokens_of(a.starts, b, a.sequences, a.tokens), context = a.context[b];
  if (n == 0 || context <= 0) return;
  const int start = attn::start_of(a.starts, b, a.tokens), p_new = context - n;  // position of the first new token
  const int p0 = max(p_new, 0), tile = slot - first_block_slot(a, b);
  // The position of the block's first token; below 0 where it passes 31 bits, which unsigned products may.
  const uint32_t block = static_cast<uint32_t>(a.block.value);
  const int base = static_cast<int>(static_cast<uint32_t>(over(p0, a.block) + tile) * block);
  if (tile < 0 || base < 0 || base >= context) return;
  const int page_at = over(base, a.page_size);
  if (page_at >= a.table_width) return;
  const int page = a.table[b * a.table_width + page_at];
  if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.pages)) return;
  const int slot0 = base - page_at * a.page_size.value;
  const bool has_old = base < p_new;
  uint8_t* const exps = op.exps + page * op.exp_page + over(slot0, a.block);
  float x[PASSES][8], next[PASSES][8];  // of this head and the next
  auto load = [&](int h, float (&to)[PASSES][8]) __attribute__((always_inline)) {
#pragma unroll
    for (int pass = 0; pass < PASSES; ++pass) {
      const int r = pass * RPP + row, p = base + r;
      if (r < a.block.value && p >= p0 && p < context)
        load8<DT>(op.src, h * op.src_head + (start + (p - p_new)) * op.src_token + c0, to[pass]);
    }
  };
  load(walk0, x);
  int before = has_old ? exps[walk0 * op.exp_head] : 0;
  if constexpr (TURNED) {
    if (turn) {
      __syncthreads();
      for (int r = tid / PAIRS; r < a.block.value && pair < a.pairs; r += TURNS) {
        const int p = base + r;
        if (p >= p0 && p < context) turns[r * PAIRS + turn_at<D>(pair)] = turn64(p * radians[pair], a.magnitude);
      }
      __syncthreads();
    }
  }
  for (int h = walk0; h < head1; ++h) {
    uint8_t* codes = op.codes + page * op.page + h * op.head + slot0 * op.slot + c0;
    float top = 0.0f;
    int next_before = 0;
    if (h + 1 < head1) {
      load(h + 1, next);
      if (has_old) next_before = exps[(h + 1) * op.exp_head];
    }
#pragma unroll
    for (int pass = 0; pass < PASSES; ++pass) {
      const int r = pass * RPP + row, p = base + r;
      if (r >= a.block.value || p < p0 || p >= context) continue;
      if constexpr (TURNED) {
        if (turn) {
          float y[8];
          const int64_t at = h * op.src_head + (start + (p - p_new)) * op.src_token;
          turned8<DT, D>(op.src, at, c0, turns + r * PAIRS, a.pairs, a.interleaved, x[pass],
                          [&](int i, float own, float other, double2 u, bool turns_it) {
            y[i] = turns_it ? round_to_odd(__builtin_fma(static_cast<double>(own), u.x, other * u.y)) : own;
          });
#pragma unroll
          for (int i = 0; i < 8; ++i) x[pass][i] = y[i];
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        top = fmaxf(top, fabsf(x[pass][i]) < __builtin_inff() ? fabsf(x[pass][i]) : __builtin_inff());
    }
    top = wave_max(top);
    if ((tid & 63) == 0) tops[h & 1][tid >> 6] = top;
    __syncthreads();  // the other slot is written behind the next head's barrier at the earliest
#pragma unroll
    for (int w = 0; w < T / 64; ++w) top = fmaxf(top, tops[h & 1][w]);
    const int after = max(exponent_of<MODE>(top), before);
    const float unit = unit_of(after);
#pragma unroll
    for (int pass = 0; pass < PASSES; ++pass) {
      const int r = pass * RPP + row, p = base + r;
      if (r >= a.block.value || p >= context) continue;
      uint2* to = reinterpret_cast<uint2*>(codes + r * op.slot);
      float y[8];
      if (p >= p0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = after == 255 ? 0.0f : x[pass][i] * unit;
      } else {
        if (after == before || after == 255) continue;
        const uint2 w = *to;
        float lo[4], hi[4];
        decode4<MODE>(w.x, lo);
        decode4<MODE>(w.y, hi);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = __builtin_ldexpf(i < 4 ? lo[i & 3] : hi[i & 3], before - after);
      }
      *to = encode8<MODE>(y);
    }
    if (tid == 0) exps[h * op.exp_head] = static_cast<uint8_t>(after);
    before = next_before;
#pragma unroll
    for (int pass = 0; pass < PASSES; ++pass)
#pragma unroll
      for (int i = 0; i < 8; ++i) x[pass][i] = next[pass][i];
  }
}

// ---- read -----------------------------------------------------------------------------------------

struct ReadArgs {
  const uint8_t *codes[2], *exps[2];
  int64_t page[2], head[2], slot[2], exp_page[2], exp_head[2];
  void* out[2];
  const int32_t *table, *starts, *context;
  int64_t table_width;
  int tokens, kv_heads, sequences, pages, walk, groups;
  Divisor page_size, block;
};

// A thread has 8 channels of one token and walks over heads, READ_HEADS of them under way at once: 8 bytes in, 8 values
// out, neighbours side by side.  Memory bound: 32769 tokens of 8 heads of 128, E4M3 to BF16, 36 us, 5.6 TB/s; 19569
// tokens of 33 sequences, 16 heads of 64, INT8 to FP16, 24.5 us, 4.9 TB/s.  (16 channels, two stores that leave every
// other 16 bytes to each other, one head at a time: 48 and 31 us; 8 channels, one head at a time 37.6 and 29.2, two
// 37.1 and 28.0, eight 36.4 and 24.1.)
template <int DT, int D, int MODE>
__global__ __launch_bounds__(THREADS) void read_codes(const ReadArgs a) {
  constexpr int CH = D / 8;
  const int64_t unit = int64_t{blockIdx.x} * THREADS + threadIdx.x;
  const int token = static_cast<int>(unit / CH), c0 = static_cast<int>(unit % CH) * 8;
  if (token >= a.tokens) return;
  const int which = blockIdx.y >= a.groups, head0 = (blockIdx.y - which * a.groups) * a.walk;
  const int head1 = min(head0 + a.walk, a.kv_heads);
  int lo = 0, hi = a.sequences;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.starts[mid] <= token) lo = mid;
    else hi = mid;
  }
  const int s = a.starts[lo], e = a.starts[lo + 1];
  bool known = token >= s && token < e;
  const int position = known ? a.context[lo] - (e - token) : -1;
  known = known && position >= 0;
  const int page_at = known ? over(position, a.page_size) : 0;
  known = known && page_at < a.table_width;
  const int page = known ? a.table[lo * a.table_width + page_at] : -1;
  known = known && static_cast<uint32_t>(page) < static_cast<uint32_t>(a.pages);
  const int at = position - page_at * a.page_size.value, block = known ? over(at, a.block) : 0;
  const uint8_t* const codes = a.codes[which] + page * a.page[which] + at * a.slot[which] + c0;
  const uint8_t* const exps = a.exps[which] + page * a.exp_page[which] + block;
  for (int h0 = head0; h0 < head1; h0 += READ_HEADS) {
    uint2 w[READ_HEADS] = {};
    int exponent[READ_HEADS] = {};
    if (known) {
#pragma unroll
      for (int i = 0; i < READ_HEADS; ++i) {
        const int h = min(h0 + i, head1 - 1);
        w[i] = *reinterpret_cast<const uint2*>(codes + h * a.head[which]);
        exponent[i] = exps[h * a.exp_head[which]];
      }
    }
#pragma unroll
    for (int i = 0; i < READ_HEADS; ++i) {
      if (h0 + i >= head1) break;
      const float scale = scale_of(exponent[i]);
      float lo4[4], hi4[4], x[8];
      decode4<MODE>(w[i].x, lo4);
      decode4<MODE>(w[i].y, hi4);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = (j < 4 ? lo4[j & 3] : hi4[j & 3]) * scale;
      store8<DT>(a.out[which], (int64_t{h0 + i} * a.tokens + token) * D + c0, x);
    }
  }
}

// ---- launches -------------------------------------------------------------------------------------

template <int DT, int D, int MODE, int T, int PASSES, bool TURNED>
int append_threads(AppendArgs& a, hipStream_t st) {
  constexpr int ROWS = PASSES * T / (D / 8);  // of q a workgroup
  const int block = a.block.value;
  a.slots = block_slots(a.tokens, a.tokens / block, a.sequences);
  a.walk = append_walk(a.tokens, block, a.kv_heads, a.heads, T);
  a.groups = divisor((a.kv_heads + a.walk - 1) / a.walk);
  a.q_groups = divisor(a.heads ? (a.heads + a.walk - 1) / a.walk : 1);
  const int q_slots = a.heads ? (a.tokens + ROWS - 1) / ROWS : 0;
  const int64_t blocks = int64_t{2} * a.slots * a.groups.value + int64_t{q_slots} * a.q_groups.value;
  M5K_REQUIRE(fits_launch(blocks, T), "paged_append: too many rows for one launch");
  launch_kernel(append_codes<DT, D, MODE, T, PASSES, TURNED>, dim3(static_cast<uint32_t>(blocks)), dim3(T), st, a);
  return launch_status("paged_append");
}

template <int DT, int D, int MODE>
int append_block(AppendArgs& a, hipStream_t st) {
  const int threads = a.block.value * (D / 8);
  if (a.pairs) {
    if (threads <= 256) return append_threads<DT, D, MODE, 256, 1, true>(a, st);
    if (threads <= 512) return append_threads<DT, D, MODE, 512, 1, true>(a, st);
    if (threads <= 1024) return append_threads<DT, D, MODE, 1024, 1, true>(a, st);
    if constexpr (D == 128) return append_threads<DT, D, MODE, 1024, 2, true>(a, st);
  } else {
    if (threads <= 256) return append_threads<DT, D, MODE, 256, 1, false>(a, st);
    if (threads <= 512) return append_threads<DT, D, MODE, 256, 2, false>(a, st);
    if (threads <= 1024) return append_threads<DT, D, MODE, 256, 4, false>(a, st);
    if constexpr (D == 128) return append_threads<DT, D, MODE, 256, 8, false>(a, st);
  }
  return M5K_EINVAL;
}

template <int DT>
int append_typed(AppendArgs& a, int mode, int head_dim, hipStream_t st) {
  if (mode == M5K_QUANT_FP8)
    return head_dim == 64 ? append_block<DT, 64, M5K_QUANT_FP8>(a, st) : append_block<DT, 128, M5K_QUANT_FP8>(a, st);
  return head_dim == 64 ? append_block<DT, 64, M5K_QUANT_INT8>(a, st) : append_block<DT, 128, M5K_QUANT_INT8>(a, st);
}

template <int DT>
int read_typed(const ReadArgs& a, int mode, int head_dim, hipStream_t st) {
  const int64_t blocks = (int64_t{a.tokens} * (head_dim / 8) + THREADS - 1) / THREADS;
  M5K_REQUIRE(fits_launch(blocks, THREADS), "paged_read: too many tokens for one launch");
  const dim3 grid(static_cast<uint32_t>(blocks), static_cast<uint32_t>(2 * a.groups));
  auto kernel = mode == M5K_QUANT_FP8
                    ? (head_dim == 64 ? read_codes<DT, 64, M5K_QUANT_FP8> : read_codes<DT, 128, M5K_QUANT_FP8>)
                    : (head_dim == 64 ? read_codes<DT, 64, M5K_QUANT_INT8> : read_codes<DT, 128, M5K_QUANT_INT8>);
  launch_kernel(kernel, grid, dim3(THREADS), st, a);
  return launch_status("paged_read");
}

int check_cache(const char* what, int mode, int64_t head_dim, const void* k, const void* v, const void* ke,
                const void* ve, const int64_t (&strides)[6], int64_t block, int64_t pages, int64_t page_size,
                int64_t kv_heads, const int32_t* table, int64_t table_width, int64_t sequences, const int32_t* starts,
                const int32_t* context, int64_t tokens) {
  M5K_REQUIRE(k && v && ke && ve && table && starts && context, "%s: null pointer", what);
  M5K_REQUIRE(mode == M5K_QUANT_FP8 || mode == M5K_QUANT_INT8, "%s: codes must be FP8 or INT8", what);
  M5K_REQUIRE(head_dim == 64 || head_dim == 128, "%s: head_dim must be 64 or 128", what);
  M5K_REQUIRE(kv_heads > 0 && kv_heads <= 16384, "%s: bad number of heads", what);
  M5K_REQUIRE(pages > 0 && pages <= INT32_MAX && page_size > 0 && page_size <= (1 << 20) && table_width > 0 &&
                  table_width * page_size <= (1 << 30) && sequences > 0 && sequences <= (1 << 24),
              "%s: a sequence may have up to 2^30 keys in pages of up to 2^20", what);
  M5K_REQUIRE(block > 0 && block <= BLOCK_MAX && block % 16 == 0 && page_size % block == 0,
              "%s: a block must be 16 to 128 tokens, a multiple of 16, and divide the page", what);
  M5K_REQUIRE(tokens > 0 && tokens <= (1 << 28), "%s: bad number of tokens", what);
  bool rows = aligned16(k) && aligned16(v);
  for (int64_t s : strides) rows = rows && s % 16 == 0;
  M5K_REQUIRE(rows, "%s: rows of codes must be 16-byte aligned", what);
  return M5K_OK;
}

}  // namespace
}  // namespace m5k

extern "C" int m5k_paged_append_codes64(
    const void* k, int64_t k_head, int64_t k_token, const void* v, int64_t v_head, int64_t v_token, int dtype,
    int64_t tokens, int64_t kv_heads, int64_t head_dim, int mode, void* k_codes, int64_t kc_page, int64_t kc_head,
    int64_t kc_slot, uint8_t* k_exponents, int64_t ke_page, int64_t ke_head, void* v_codes, int64_t vc_page,
    int64_t vc_head, int64_t vc_slot, uint8_t* v_exponents, int64_t ve_page, int64_t ve_head, int64_t block,
    int64_t pages, int64_t page_size, const int32_t* page_table, int64_t table_width, int64_t sequences,
    const int32_t* query_starts, const int32_t* context_lengths, const void* q, int64_t heads, int64_t q_head,
    int64_t q_token, void* q_out, const double* frequencies, int64_t pairs, int interleaved, double magnitude,
    void* stream) {
  using namespace m5k;
  clear_error();
  M5K_REQUIRE(dtype == M5K_F32 || dtype == M5K_F16 || dtype == M5K_BF16,
              "paged_append: dtype must be f32, f16 or bf16");
  if (int rc = check_cache("paged_append", mode, head_dim, k_codes, v_codes, k_exponents, v_exponents,
                           {kc_page, kc_head, kc_slot, vc_page, vc_head, vc_slot}, block, pages, page_size, kv_heads,
                           page_table, table_width, sequences, query_starts, context_lengths, tokens))
    return rc;
  M5K_REQUIRE(k && v, "paged_append: null pointer");
  M5K_REQUIRE(pairs >= 0 && 2 * pairs <= head_dim && (pairs == 0 || frequencies),
              "paged_append: 2 * pairs must fit in head_dim");
  M5K_REQUIRE(!q || (q_out && heads > 0 && heads <= 16384 && pairs > 0),
              "paged_append: q needs q_out, heads and a rotation");
  const int64_t unit = dtype == M5K_F32 ? 4 : 8;
  M5K_REQUIRE(aligned16(k) && aligned16(v) && k_head % unit == 0 && k_token % unit == 0 && v_head % unit == 0 &&
                  v_token % unit == 0 && (!q || (aligned16(q) && q_head % unit == 0 && q_token % unit == 0)),
              "paged_append: rows must be 16-byte aligned");
  AppendArgs a = {};
  a.op[0] = Operand{k,       static_cast<uint8_t*>(k_codes), k_exponents, k_head, k_token, kc_page, kc_head, kc_slot,
                    ke_page, ke_head};
  a.op[1] = Operand{v,       static_cast<uint8_t*>(v_codes), v_exponents, v_head, v_token, vc_page, vc_head, vc_slot,
                    ve_page, ve_head};
  a.q = q;
  a.q_out = q_out;
  a.q_head = q_head;
  a.q_token = q_token;
  a.table = page_table;
  a.starts = query_starts;
  a.context = context_lengths;
  a.frequencies = frequencies;
  a.table_width = table_width;
  a.tokens = static_cast<int>(tokens);
  a.kv_heads = static_cast<int>(kv_heads);
  a.heads = q ? static_cast<int>(heads) : 0;
  a.pairs = static_cast<int>(pairs);
  a.interleaved = interleaved != 0;
  a.sequences = static_cast<int>(sequences);
  a.pages = static_cast<int>(pages);
  a.page_size = divisor(static_cast<int>(page_size));
  a.block = divisor(static_cast<int>(block));
  a.magnitude = magnitude;
  const int dim = static_cast<int>(head_dim);
  if (dtype == M5K_BF16) return append_typed<M5K_BF16>(a, mode, dim, as_stream(stream));
  if (dtype == M5K_F16) return append_typed<M5K_F16>(a, mode, dim, as_stream(stream));
  return append_typed<M5K_F32>(a, mode, dim, as_stream(stream));
}

extern "C" int m5k_paged_append_codes(
    const void* k, int64_t k_head, int64_t k_token, const void* v, int64_t v_head, int64_t v_token, int dtype,
    int64_t tokens, int64_t kv_heads, int64_t head_dim, int mode, void* k_codes, int64_t kc_page, int64_t kc_head,
    int64_t kc_slot, uint8_t* k_exponents, int64_t ke_page, int64_t ke_head, void* v_codes, int64_t vc_page,
    int64_t vc_head, int64_t vc_slot, uint8_t* v_exponents, int64_t ve_page, int64_t ve_head, int64_t block,
    int64_t pages, int64_t page_size, const int32_t* page_table, int64_t table_width, int64_t sequences,
    const int32_t* query_starts, const int32_t* context_lengths, const void* q, int64_t heads, int64_t q_head,
    int64_t q_token, void* q_out, const double* frequencies, int64_t pairs, int interleaved, float magnitude,
    void* stream) {
  return m5k_paged_append_codes64(k, k_head, k_token, v, v_head, v_token, dtype, tokens, kv_heads, head_dim, mode,
                                  k_codes, kc_page, kc_head, kc_slot, k_exponents, ke_page, ke_head, v_codes, vc_page,
                                  vc_head, vc_slot, v_exponents, ve_page, ve_head, block, pages, page_size, page_table,
                                  table_width, sequences, query_starts, context_lengths, q, heads, q_head, q_token,
                                  q_out, frequencies, pairs, interleaved, magnitude, stream);
}

extern "C" int m5k_paged_read(int mode, const void* k_codes, int64_t kc_page, int64_t kc_head, int64_t kc_slot,
                              const uint8_t* k_exponents, int64_t ke_page, int64_t ke_head, const void* v_codes,
                              int64_t vc_page, int64_t vc_head, int64_t vc_slot, const uint8_t* v_exponents,
                              int64_t ve_page, int64_t ve_head, int64_t block, int64_t pages, int64_t page_size,
                              int64_t kv_heads, int64_t head_dim, const int32_t* page_table, int64_t table_width,
                              int64_t sequences, const int32_t* query_starts, const int32_t* context_lengths,
                              int64_t tokens, void* k, void* v, int dtype, void* stream) {
  using namespace m5k;
  clear_error();
  M5K_REQUIRE(dtype == M5K_F32 || dtype == M5K_F16 || dtype == M5K_BF16, "paged_read: dtype must be f32, f16 or bf16");
  if (int rc = check_cache("paged_read", mode, head_dim, k_codes, v_codes, k_exponents, v_exponents,
                           {kc_page, kc_head, kc_slot, vc_page, vc_head, vc_slot}, block, pages, page_size, kv_heads,
                           page_table, table_width, sequences, query_starts, context_lengths, tokens))
    return rc;
  M5K_REQUIRE(k && v && aligned16(k) && aligned16(v), "paged_read: outputs must be 16-byte aligned");
  ReadArgs a = {};
  a.codes[0] = static_cast<const uint8_t*>(k_codes);
  a.codes[1] = static_cast<const uint8_t*>(v_codes);
  a.exps[0] = k_exponents;
  a.exps[1] = v_exponents;
  const int64_t strides[5][2] = {{kc_page, vc_page}, {kc_head, vc_head}, {kc_slot, vc_slot}, {ke_page, ve_page},
                                 {ke_head, ve_head}};
  for (int i = 0; i < 2; ++i) {
    a.page[i] = strides[0][i];
    a.head[i] = strides[1][i];
    a.slot[i] = strides[2][i];
    a.exp_page[i] = strides[3][i];
    a.exp_head[i] = strides[4][i];
  }
  a.out[0] = k;
  a.out[1] = v;
  a.table = page_table;
  a.starts = query_starts;
  a.context = context_lengths;
  a.table_width = table_width;
  a.tokens = static_cast<int>(tokens);
  a.kv_heads = static_cast<int>(kv_heads);
  a.sequences = static_cast<int>(sequences);
  a.pages = static_cast<int>(pages);
  a.page_size = divisor(static_cast<int>(page_size));
  a.block = divisor(static_cast<int>(block));
  static_assert(THREADS == 256, "read_walk counts with it");
  a.walk = read_walk(tokens, static_cast<int>(head_dim), a.kv_heads);
  a.groups = (a.kv_heads + a.walk - 1) / a.walk;
  const int dim = static_cast<int>(head_dim);
  if (dtype == M5K_BF16) return read_typed<M5K_BF16>(a, mode, dim, as_stream(stream));
  if (dtype == M5K_F16) return read_typed<M5K_F16>(a, mode, dim, as_stream(stream));
  return read_typed<M5K_F32>(a, mode, dim, as_stream(stream));
}
